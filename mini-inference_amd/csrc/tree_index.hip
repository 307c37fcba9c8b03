// Where the nodes of drafted trees go and what they see: positions, pool slots and ancestor sets, from
// the trees' parents and the sequences' cached lengths and block tables.
//
// No reference counterpart (the reference decodes one token a step). Node i of sequence s is packed row
// r = cu_q[s] + i; parents[r] is its parent's number in the same tree. A parent comes before its
// children; a value that is negative or not below i makes node i a root, so that every path ends.
//     mask[r]      = the set of nodes on the path from i to its root, i among them, as bits
//     positions[r] = ctx_start[s] + (number of nodes on that path) - 1
//     slots[r]     = table[p / block_size] * block_size + p % block_size,  p = ctx_start[s] + i
// (a node is stored behind the cached tokens in its own place, whatever its depth; -1 where p lies past
// the table). Rows of no node, which pad a batch, get position 0, slot -1 and no bits, so that what takes
// them as a token appends and attends nothing.
//
// One wavefront per sequence, and one for the rows of none. Up to 64 nodes a lane holds one node's set in a register pair and the sets
// grow by pointer doubling: after round k a set holds the path's first 2^k nodes and `jump` is the node
// 2^k steps up, so a round is one exchange of sets between lanes and a path of 64 takes 6 rounds.
// Larger trees walk each path through the parents (held in LDS, up to kMaxNodes of them). Bound by the
// launch: 4 bytes read and 24 written per node (one tree of 5 nodes 1.6 us, 256 trees of 17-64 2.8 us on the device).
#include "mip_common.h"

namespace mip {
namespace {

constexpr int kMaxNodes = MIP_TREE_MAX_NODES;

struct IndexArgs {
  int64_t* positions;
  int64_t* slots;
  uint64_t* mask;
  const int32_t* parents;
  const int32_t* cu_q;
  const int32_t* ctx_start;
  const int32_t* tables;
  int64_t bt_stride;
  int n_rows, num_seqs, max_q_len, words, max_blocks, log2_bs;
};

__device__ __forceinline__ uint64_t shfl_u64(uint64_t x, int lane) {
  const uint32_t lo = __shfl(static_cast<uint32_t>(x), lane), hi = __shfl(static_cast<uint32_t>(x >> 32), lane);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

__device__ __forceinline__ int64_t slot_of(const IndexArgs& a, int s, int p) {
  const int i = p >> a.log2_bs;
  if (p < 0 || i >= a.max_blocks) return -1;
  return (static_cast<int64_t>(a.tables[s * a.bt_stride + i]) << a.log2_bs) + (p & ((1 << a.log2_bs) - 1));
}

// Rows [from, to) belong to no node.
__device__ __forceinline__ void blank_rows(const IndexArgs& a, int from, int to, int lane) {
  from = from > 0 ? from : 0;
  to = to < a.n_rows ? to : a.n_rows;
  for (int64_t r = from + lane; r < to; r += kWave) {
    a.positions[r] = 0;
    a.slots[r] = -1;
    for (int w = 0; w < a.words; ++w) a.mask[r * a.words + w] = 0;
  }
}

__global__ __launch_bounds__(kWave) void tree_index_kernel(IndexArgs a) {
  __shared__ int32_t s_parent[kMaxNodes];
  const int s = blockIdx.x, lane = threadIdx.x;
  if (s == a.num_seqs) {
    blank_rows(a, 0, a.cu_q[0], lane);
    blank_rows(a, a.cu_q[s], a.n_rows, lane);
    return;
  }
  const int r0 = a.cu_q[s], r1 = a.cu_q[s + 1], ctx = a.ctx_start[s];
  if (r0 < 0 || r1 > a.n_rows) return;
  int n = r1 - r0;
  if (n > a.max_q_len) {
    n = a.max_q_len;
    blank_rows(a, r0 + n, r1, lane);
  }
  if (n <= kWave) {
    const bool live = lane < n;
    int jump = live ? a.parents[r0 + lane] : -1;
    const int64_t slot = live ? slot_of(a, s, ctx + lane) : -1;
    if (jump < 0 || jump >= lane) jump = -1;
    uint64_t set = 1ull << lane;
    while (__any(jump >= 0)) {
      const int up = jump >= 0 ? jump : lane;
      const uint64_t more = shfl_u64(set, up);
      const int next = __shfl(jump, up);
      set |= more;
      jump = jump >= 0 ? next : -1;
    }
    if (!live) return;
    const int64_t r = r0 + lane;
    a.positions[r] = ctx + __popcll(set) - 1;
    a.slots[r] = slot;
    uint64_t* row = a.mask + r * a.words;
    row[0] = set;
    for (int w = 1; w < a.words; ++w) row[w] = 0;
    return;
  }
  for (int i = lane; i < n; i += kWave) {
    const int p = a.parents[r0 + i];
    s_parent[i] = p >= 0 && p < i ? p : -1;
  }
  __syncthreads();
  for (int i = lane; i < n; i += kWave) {
    const int64_t r = r0 + i;
    uint64_t* row = a.mask + r * a.words;
    // The path's node numbers fall, so each word is complete when the path leaves it.
    int at = i, depth = 0;
    for (int w = a.words - 1; w >= 0; --w) {
      uint64_t set = 0;
      while (at >= 64 * w) {  // at = -1 past the root
        set |= 1ull << (at & 63);
        at = s_parent[at];
        ++depth;
      }
      row[w] = set;
    }
    a.positions[r] = ctx + depth - 1;
    a.slots[r] = slot_of(a, s, ctx + i);
  }
}

}  // namespace
}  // namespace mip

using namespace mip;

extern "C" int mip_tree_index(int64_t* positions, int64_t* slot_mapping, uint64_t* mask, int32_t mask_words,
                              const int32_t* parents, int32_t n_rows, const int32_t* cu_q, const int32_t* ctx_start,
                              const int32_t* block_tables, int64_t bt_stride, int32_t num_seqs, int32_t max_q_len,
                              int32_t block_size, int32_t max_blocks_per_seq, void* stream) {
  if (n_rows < 0 || num_seqs < 0 || max_q_len < 0 || !is_pow2(block_size) || block_size > 4096) return MIP_EINVAL;
  if (max_blocks_per_seq <= 0 || bt_stride < max_blocks_per_seq) return MIP_EINVAL;
  if (max_q_len > kMaxNodes) return MIP_EUNSUPPORTED;
  if (n_rows == 0) return MIP_OK;
  if (mask_words < (max_q_len + 63) / 64 || mask_words > kMaxNodes / 64) return MIP_EINVAL;
  if (!positions || !slot_mapping || !parents || !cu_q || (mask_words > 0 && !mask)) return MIP_EINVAL;
  if (num_seqs > 0 && (!ctx_start || !block_tables)) return MIP_EINVAL;
  if (num_seqs >= 1 << 24) return MIP_EUNSUPPORTED;
  IndexArgs a{positions, slot_mapping, mask,       parents,    cu_q,               ctx_start,              block_tables, bt_stride,
              n_rows,    num_seqs,     max_q_len, mask_words, max_blocks_per_seq, ilog2_exact(block_size)};
  hipLaunchKernelGGL(tree_index_kernel, dim3(num_seqs + 1), dim3(kWave), 0, static_cast<hipStream_t>(stream), a);
  return status_from_hip(hipGetLastError());
}
