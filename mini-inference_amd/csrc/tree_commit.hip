// The accepted nodes of drafted trees, moved to the places that consecutive tokens have in the pool.
//
// No reference counterpart. Node i of a tree is stored at cache index ctx_start[s] + i. After
// verification path[s][0 .. counts[s]) are the accepted nodes in order; the cache of the accepted tokens
// has node path[s][d] at index ctx_start[s] + d. For every layer, K and V:
//     pool[layer][row(ctx + d)] = pool[layer][row(ctx + path[s][d])]      d < counts[s], bit for bit,
// with every source as it was before the call. A path rises (a parent comes before its children), so
// path[s][d] >= d: sources lie at or behind their destinations, and taking d in order reads each source
// before anything is written over it. An entry that breaks this (below d, or not above the one before
// it) or lies outside the table ends the path there.
//
// One thread owns one CHUNK-byte column of all a sequence's rows of one (layer, K|V, head) and moves it
// down entry by entry, kGroup loaded before they are stored: no thread reads what another writes, so no order between
// threads is needed. Bound by a serial chain: an entry ends the path by a branch on what was just loaded, so each entry
// waits for its path value, then its two table values, and with these for the row of the entry before. One sequence, 24
// layers of 2 heads of 64, 4.0 us on the device; 64 sequences, 28 layers of 4 heads of 128, 26 MB 12.0 us (2.2 TB/s).
#include "mip_common.h"

namespace mip {
namespace {

template <int CHUNK> struct MoveT;
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
template <> struct MoveT<16> { using T = u32x4_t; };  // (an array of uint4 would stay in scratch memory)
template <> struct MoveT<8>  { using T = u32x2_t; };
template <> struct MoveT<4>  { using T = uint32_t; };
template <> struct MoveT<2>  { using T = uint16_t; };

constexpr int kMoveThreads = 256;
constexpr int kGroup = 8;

struct CommitArgs {
  char* k;
  char* v;
  const int32_t* tables;
  int64_t bt_stride;
  const int32_t* ctx_start;
  const int32_t* path;
  int64_t path_stride;
  const int32_t* counts;
  int64_t ncb;
  int num_layers, hkv, row_bytes, block_size, log2_bs, max_blocks, max_path;
  uint32_t lanes;  // threads per sequence: layers * 2 * heads * chunks per row
};

template <int CHUNK>
__global__ __launch_bounds__(kMoveThreads) void tree_commit_kernel(CommitArgs a) {
  using V = typename MoveT<CHUNK>::T;
  const int s = blockIdx.y;
  int n = a.counts[s];
  n = n < a.max_path ? n : a.max_path;
  const uint32_t t = blockIdx.x * kMoveThreads + threadIdx.x;
  if (n <= 1 && a.path[s * a.path_stride] == 0) return;  // node 0 alone: in place already
  if (t >= a.lanes) return;
  const uint32_t cpr = static_cast<uint32_t>(a.row_bytes / CHUNK);
  const uint32_t c = t % cpr, u = t / cpr;
  const uint32_t h = u % static_cast<uint32_t>(a.hkv), ls = u / static_cast<uint32_t>(a.hkv);
  char* base = (ls & 1 ? a.v : a.k) + static_cast<int64_t>(ls >> 1) * a.ncb * a.hkv * a.block_size * a.row_bytes +
               static_cast<int64_t>(c) * CHUNK;
  const int32_t* table = a.tables + s * a.bt_stride;
  const int ctx = a.ctx_start[s];
  // Pool row of cache index p (-1 outside the table or the pool).
  auto row_of = [&](int p) -> int64_t {
    const int i = p >> a.log2_bs;
    if (p < 0 || i >= a.max_blocks) return -1;
    const int64_t blk = table[i];
    if (blk < 0 || blk >= a.ncb) return -1;
    return (blk * a.hkv + h) * a.block_size + (p & (a.block_size - 1));
  };
  int prev = -1;
  bool more = true;
  for (int d0 = 0; d0 < n && more; d0 += kGroup) {
    V val[kGroup];
    int64_t dst[kGroup];
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      dst[j] = -1;
      const int d = d0 + j;
      if (d >= n || !more) continue;
      const int i = a.path[s * a.path_stride + d];
      more = i >= d && i > prev;
      prev = i;
      if (!more || i == d) continue;
      const int64_t from = row_of(ctx + i), to = row_of(ctx + d);
      if (from < 0 || to < 0) {
        more = false;
        continue;
      }
      val[j] = *reinterpret_cast<const V*>(base + from * a.row_bytes);
      dst[j] = to;
    }
#pragma unroll
    for (int j = 0; j < kGroup; ++j)
      if (dst[j] >= 0) *reinterpret_cast<V*>(base + dst[j] * a.row_bytes) = val[j];
  }
}

template <int CHUNK>
void launch(const CommitArgs& a, int num_seqs, hipStream_t s) {
  hipLaunchKernelGGL(tree_commit_kernel<CHUNK>, dim3((a.lanes + kMoveThreads - 1) / kMoveThreads, num_seqs),
                     dim3(kMoveThreads), 0, s, a);
}

}  // namespace
}  // namespace mip

using namespace mip;

extern "C" int mip_tree_commit(void* k_pool, void* v_pool, int32_t num_layers, int64_t num_cache_blocks,
                               int32_t num_kv_heads, int32_t head_dim, int32_t block_size, const int32_t* block_tables,
                               int64_t bt_stride, int32_t max_blocks_per_seq, const int32_t* ctx_start,
                               const int32_t* path, int64_t path_stride, int32_t max_path, const int32_t* counts,
                               int32_t num_seqs, int32_t dtype, void* stream) {
  if (dtype != MIP_F32 && dtype != MIP_F16 && dtype != MIP_BF16) return MIP_EINVAL;
  if (num_layers <= 0 || num_cache_blocks <= 0 || num_kv_heads <= 0 || head_dim <= 0 || num_seqs < 0 || max_path < 0)
    return MIP_EINVAL;
  if (!is_pow2(block_size) || block_size > 4096 || max_blocks_per_seq <= 0 || bt_stride < max_blocks_per_seq ||
      path_stride < max_path)
    return MIP_EINVAL;
  if (num_seqs == 0 || max_path == 0) return MIP_OK;
  if (!k_pool || !v_pool || !block_tables || !ctx_start || !path || !counts) return MIP_EINVAL;
  const int64_t row_bytes = static_cast<int64_t>(head_dim) * (dtype == MIP_F32 ? 4 : 2);
  const uint64_t align_bits =
      static_cast<uint64_t>(row_bytes) | reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool);
  int chunk = 16;
  while (chunk > 2 && (align_bits & (chunk - 1))) chunk >>= 1;
  if (align_bits & 1) return MIP_EINVAL;
  const int64_t lanes = static_cast<int64_t>(num_layers) * 2 * num_kv_heads * (row_bytes / chunk);
  if (row_bytes >= (int64_t{1} << 31) || lanes >= (int64_t{1} << 31) || num_seqs > 65535) return MIP_EUNSUPPORTED;
  CommitArgs a{static_cast<char*>(k_pool), static_cast<char*>(v_pool), block_tables, bt_stride, ctx_start, path,
               path_stride, counts, num_cache_blocks, num_layers, num_kv_heads, static_cast<int>(row_bytes), block_size,
               ilog2_exact(block_size), max_blocks_per_seq, max_path, static_cast<uint32_t>(lanes)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (chunk) {
    case 16: launch<16>(a, num_seqs, s); break;
    case 8:  launch<8>(a, num_seqs, s); break;
    case 4:  launch<4>(a, num_seqs, s); break;
    default: launch<2>(a, num_seqs, s); break;
  }
  return status_from_hip(hipGetLastError());
}
