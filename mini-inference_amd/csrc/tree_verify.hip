// Verification of drafted trees against a model's logits: the model's choice after every node, and the
// drafted path that agrees with it, at every node its first child that does.
//
// No reference counterpart (the reference decodes one token a step). For row r of the logits
//     target[r] = the lowest v with logits[r][v] = max (a NaN counts as the greatest value)
// and for sequence s, whose tree's node i is row cu_q[s] + i, the path starts at node 0 and goes on to the
// lowest node whose parent is the path's last node and whose token is that node's target, until there is
// none; the target of the last node is the token that follows. (Of siblings that carry one token the first is
// taken, whatever is drafted below the others.)
//
// Two launches. verify_max: a workgroup takes a piece of a row (rows are cut where there are few of them)
// and leaves its maximum as one 64-bit key, (value in an order-preserving integer form) << 32 |
// ~index, so that the greatest key is the greatest value at its lowest index whatever the order of
// comparison. A thread compares whole 16-byte chunks (a maximum of the chunk, one comparison with its
// best) and looks for the element in the best chunk alone, once. verify_walk: a workgroup per sequence
// folds its rows' keys and walks the tree, 64 nodes a step (a match of parent and token by ballot).
//
// Bound by the read of the logits: 64 trees of 9-16 nodes over 151936 fp32 logits, 469 MB, verify_max 87 us (5.4 TB/s,
// a large copy on the same card reads and writes 5.2) and verify_walk 6.6; one tree of 5 nodes over bf16 logits 3.8
// and 4.1, both latency. One launch for both would need every workgroup's last one to walk, behind a counter that a
// captured call has to clear.
#include "mip_common.h"

namespace mip {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxNodes = MIP_TREE_MAX_NODES;

// The order of floats as the order of unsigned integers: -0 and 0 alike, every NaN above infinity.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint64_t make_key(float x, uint32_t index) {
  return (static_cast<uint64_t>(order_key(x)) << 32) | static_cast<uint32_t>(~index);
}

__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t x) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t lo = __shfl_xor(static_cast<uint32_t>(x), d), hi = __shfl_xor(static_cast<uint32_t>(x >> 32), d);
    x = max_u64(x, (static_cast<uint64_t>(hi) << 32) | lo);
  }
  return x;
}

__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // NaN wins

// The values of a 16-byte chunk.
template <int DT> struct ChunkOf {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& w, float (&x)[N]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = lo16<DT>(u[i]);
      x[2 * i + 1] = hi16<DT>(u[i]);
    }
  }
};
template <> struct ChunkOf<MIP_F32> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& w, float (&x)[N]) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  }
};

template <int DT>
__global__ __launch_bounds__(kThreads) void verify_max_kernel(const char* logits, int64_t row_stride, int vocab,
                                                              int splits, uint64_t* keys) {
  using C = ChunkOf<DT>;
  using S = typename Elem<DT>::S;
  constexpr int N = C::N, kUnroll = 4;
  __shared__ uint64_t s_key[kThreads / kWave];
  const int64_t row = blockIdx.x / splits;
  const int part = static_cast<int>(blockIdx.x - row * splits);
  const S* x = reinterpret_cast<const S*>(logits) + row * row_stride;
  // Elements before the first 16-byte boundary, whole chunks, and what is left.
  const int head_raw = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(S));
  const int head = head_raw < vocab ? head_raw : vocab;
  const int chunks = (vocab - head) / N;
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  const int lo = static_cast<int>(static_cast<int64_t>(chunks) * part / splits);
  const int hi = static_cast<int>(static_cast<int64_t>(chunks) * (part + 1) / splits);

  float best = -INFINITY;
  int at = -1;
  auto take = [&](const uint4& w, int c) __attribute__((always_inline)) {
    float v[N];
    C::get(w, v);
    float m = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = maximum(m, v[i]);
    // Chunks come in rising order: a later one has to be greater (a NaN is, unless the best is one).
    if (at < 0 || m > best || (m != m && best == best)) {
      best = m;
      at = c;
    }
  };
  int c = lo + static_cast<int>(threadIdx.x);
  for (; c + (kUnroll - 1) * kThreads < hi; c += kUnroll * kThreads) {
    uint4 w[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) w[j] = body[c + j * kThreads];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) take(w[j], c + j * kThreads);
  }
  for (; c < hi; c += kThreads) take(body[c], c);

  uint64_t key = 0;  // below every element's key
  if (at >= 0) {
    float v[N];
    C::get(body[at], v);
#pragma unroll
    for (int i = 0; i < N; ++i) key = max_u64(key, make_key(v[i], static_cast<uint32_t>(head + at * N + i)));
  }
  if (part == 0) {  // fewer than two chunks' worth of elements beside the whole ones
    const int tail = head + chunks * N, rest = head + vocab - tail;
    for (int i = threadIdx.x; i < rest; i += kThreads) {
      const int e = i < head ? i : tail + i - head;
      key = max_u64(key, make_key(widen<DT>(x[e]), static_cast<uint32_t>(e)));
    }
  }
  key = wave_max_u64(key);
  if (threadIdx.x % kWave == 0) s_key[threadIdx.x / kWave] = key;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) key = max_u64(key, s_key[w]);
    keys[blockIdx.x] = key;
  }
}

struct WalkArgs {
  const uint64_t* keys;
  int splits, n_rows, num_seqs, max_q_len;
  const int64_t* tokens;
  const int32_t* parents;
  const int32_t* cu_q;
  int64_t* target;
  int32_t* path;
  int32_t* counts;
  int64_t* next;
};

__global__ __launch_bounds__(kThreads) void verify_walk_kernel(WalkArgs a) {
  __shared__ int32_t s_target[kMaxNodes];
  const int s = blockIdx.x, lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  // Workgroup num_seqs takes the rows of no sequence (those before the first and behind the last).
  const bool spare = s == a.num_seqs;
  const int r0 = a.cu_q[spare ? 0 : s], r1 = a.cu_q[spare ? a.num_seqs : s + 1];
  const int before = spare ? (r0 < a.n_rows ? r0 : a.n_rows) : 0;
  const int rows = spare ? before + a.n_rows - r1 : r1 - r0;
  for (int i = w; i < rows; i += kThreads / kWave) {
    const int r = spare ? (i < before ? i : r1 + i - before) : r0 + i;
    if (r < 0 || r >= a.n_rows) continue;
    uint64_t key = 0;
    for (int p = lane; p < a.splits; p += kWave) key = max_u64(key, a.keys[static_cast<int64_t>(r) * a.splits + p]);
    key = wave_max_u64(key);
    const int32_t t = static_cast<int32_t>(~static_cast<uint32_t>(key));
    if (lane == 0) a.target[r] = t;
    if (lane == 0 && !spare && i < kMaxNodes) s_target[i] = t;
  }
  if (spare) return;
  __syncthreads();
  if (w != 0) return;
  int n = rows < a.max_q_len ? rows : a.max_q_len;
  n = r0 >= 0 && r0 + n <= a.n_rows && n > 0 ? n : 0;
  int32_t* path = a.path + static_cast<int64_t>(s) * a.max_q_len;
  int count = 0, cur = 0, want = -1;
  if (n > 0) {
    // The first 64 nodes' parents and tokens stay in registers; later ones are read as the walk needs them.
    const int32_t parent0 = lane < n ? a.parents[r0 + lane] : -1;
    const int64_t token0 = lane < n ? a.tokens[r0 + lane] : -1;
    while (true) {
      if (lane == 0) path[count] = cur;
      ++count;
      want = s_target[cur];
      int next = -1;
      for (int base = cur & ~(kWave - 1); base < n && next < 0; base += kWave) {
        const int i = base + lane;
        const int32_t p = base == 0 ? parent0 : i < n ? a.parents[r0 + i] : -1;
        const int64_t t = base == 0 ? token0 : i < n ? a.tokens[r0 + i] : -1;
        const uint64_t hit = __ballot(i < n && i > cur && p == cur && t == want);  // a child comes behind its parent
        if (hit) next = base + __ffsll(static_cast<unsigned long long>(hit)) - 1;
      }
      if (next < 0) break;
      cur = next;
    }
  }
  for (int i = count + lane; i < a.max_q_len; i += kWave) path[i] = -1;
  if (lane == 0) {
    a.counts[s] = count;
    a.next[s] = want;
  }
}

// Pieces of a row: enough workgroups for the chip where rows are few, none with less than a chunk a
// thread. 4096: 16 workgroups a CU, so that uneven finishing costs little.
int verify_splits(int64_t rows, int32_t vocab, int32_t dtype) {
  const int64_t chunks = static_cast<int64_t>(vocab) / (dtype == MIP_F32 ? 4 : 8);
  const int64_t most = chunks / kThreads > 0 ? chunks / kThreads : 1;
  const int64_t want = rows > 0 ? (4096 + rows - 1) / rows : 1;
  return static_cast<int>(want < most ? want : most);
}

}  // namespace
}  // namespace mip

using namespace mip;

extern "C" size_t mip_tree_verify_workspace(int32_t n_rows, int32_t vocab, int32_t dtype) {
  if (n_rows <= 0 || vocab <= 0) return 0;
  return static_cast<size_t>(n_rows) * verify_splits(n_rows, vocab, dtype) * 8;
}

extern "C" int mip_tree_verify(int64_t* target, int32_t* path, int32_t* counts, int64_t* next_token, const void* logits,
                               int64_t row_stride, int32_t n_rows, int32_t vocab, const int64_t* tokens,
                               const int32_t* parents, const int32_t* cu_q, int32_t num_seqs, int32_t max_q_len,
                               void* workspace, size_t workspace_bytes, int32_t dtype, void* stream) {
  if (dtype != MIP_F32 && dtype != MIP_F16 && dtype != MIP_BF16) return MIP_EINVAL;
  if (n_rows < 0 || vocab <= 0 || num_seqs < 0 || max_q_len < 0 || row_stride < vocab) return MIP_EINVAL;
  if (max_q_len > kMaxNodes) return MIP_EUNSUPPORTED;
  if (n_rows == 0 && num_seqs == 0) return MIP_OK;
  if (!cu_q || (n_rows > 0 && (!target || !logits || !tokens || !parents || !workspace))) return MIP_EINVAL;
  if (num_seqs > 0 && (!counts || !next_token || (max_q_len > 0 && !path))) return MIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == MIP_F32 ? 3 : 1)) return MIP_EINVAL;
  if (workspace_bytes < mip_tree_verify_workspace(n_rows, vocab, dtype)) return MIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return MIP_EINVAL;
  const int splits = verify_splits(n_rows, vocab, dtype);
  const int64_t grid = static_cast<int64_t>(n_rows) * splits;
  if (grid >= (int64_t{1} << 24)) return MIP_EUNSUPPORTED;  // work-items of a launch stay below 2^32
  uint64_t* keys = static_cast<uint64_t*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const char* x = static_cast<const char*>(logits);
  if (grid > 0) {
    const dim3 g(static_cast<unsigned>(grid)), b(kThreads);
    switch (dtype) {
      case MIP_F32: hipLaunchKernelGGL(verify_max_kernel<MIP_F32>, g, b, 0, s, x, row_stride, vocab, splits, keys); break;
      case MIP_F16: hipLaunchKernelGGL(verify_max_kernel<MIP_F16>, g, b, 0, s, x, row_stride, vocab, splits, keys); break;
      default:      hipLaunchKernelGGL(verify_max_kernel<MIP_BF16>, g, b, 0, s, x, row_stride, vocab, splits, keys); break;
    }
  }
  const WalkArgs a{keys, splits, n_rows, num_seqs, max_q_len, tokens, parents, cu_q, target, path, counts, next_token};
  hipLaunchKernelGGL(verify_walk_kernel, dim3(num_seqs + 1), dim3(kThreads), 0, s, a);
  return status_from_hip(hipGetLastError());
}
