// Attention of drafted trees over the paged KV cache (gfx950): several sequences' nodes, packed, each over
// its sequence's cached keys and the nodes that its mask names.
//
// No reference counterpart (the reference decodes one token a step; its decode attention is
// engine/kv_cache.py:615-620). Row r = cu_q[s] + i is node i of sequence s, whose key is cache index
// c + i (c = ctx_start[s], n nodes); it sees key j < c, and key c + e where bit e of mask[r] is set, e < n:
//
//   out[r, h, :] = sum_j p_j V_s[j],  p = softmax over the seen keys of scale * q[r, h, :] . K_s[j]
//
// and zeros where it sees none.
//
// What bounds it: the keys and values are read once for all of a sequence's rows and heads of a group
// (n * group rows), so few rows are bound by the read of the cache and many by the softmax between the
// two products, as prefill is.
//
// Work split. A sequence's query rows are its (node, head of the kv head's group) pairs, packed
// node-major; a segment is (sequence, kv head, block of R rows) and has ceil((c + n) / KT) steps of KT
// keys. Segments of very different lengths share the chip, and one long sequence has to fill it, so the
// steps of all segments form one row and every workgroup takes an equal share of it; a cut that falls
// close to a segment's end moves there. A piece that is not a whole segment leaves its rows' maxima, sums
// and unnormalised outputs in a record (D + 2 floats a row) in the workspace, and a second kernel
// combines them. The shares follow from cu_q and ctx_start on the device: the grid depends on the integer
// arguments alone, so a captured call serves other lengths.
//
// A wavefront computes, for NC blocks of 16 rows and 32 keys at a time,
//   S^T[16 keys x 16 rows] = K . Q^T     v_mfma_f32_16x16x32, Q^T in registers
//   O^T[D x 16 rows]      += V^T . P^T   v_mfma_f32_16x16x32 over 32 keys
// with a base-2 online softmax whose maximum is raised only when a row's grows by more than 2^kRescaleLog2.
// V^T comes from transposing LDS reads; P is in the layout of S^T. Two shapes of a workgroup:
//   own keys     WR = 1, WK = 4: all wavefronts have the same rows and each 32 keys of a step of 128, which
//                it fetches by itself: direct global -> LDS loads into two tiles of its own, no barrier in the
//                loop. The four meet at the piece's end. For few rows, and for small calls.
//   shared keys  WR = 4, WK = 1: each wavefront has rows of its own; all threads stage a step of 32 keys
//                (two LDS stages, the next step's rows in registers meanwhile). For many rows.
// (Direct loads for the shared shape were slower: 64 x 33-64 nodes of 7 rows 58 -> 66 us, one of 61 nodes over
// 32000 keys 63 -> 104: four wavefronts wait at a barrier for loads that registers would have held back.)
//
// Roundings. Scores, sums and accumulators are fp32. Weights enter the product in V's type, as a 16-bit value and its
// remainder: 2^-22 of a weight is lost at most in fp16 (and 2^-32 of a row's largest), 2^-16 in bf16. (The value alone,
// one product instead of two: 64 x 33-64 nodes in fp16 49.7 us instead of 55.0, but weights off by 2^-11, which shows
// wherever values nearly cancel.) V enters as it is. (V staged as fp16 for one product instead of two
// loses what lies below 2^-24, a row of small values beside ordinary ones entirely.) A wavefront whose accumulators end
// up inf or NaN does its part of a piece again in a careful pass, which adds each value to the rows that see its key
// alone: a masked key must not reach a row as 0 * inf.
//
// Measured (graph replay, us a call, both kernels): 128 sequences of 4-8 nodes, 28q/4kv d128, 512-8192
// keys: 170, 725 MB at 4.3 TB/s; 64 x 33-64 nodes, 14q/2kv d64, 128-4096 keys: 55, 215 TFLOP/s; 61 nodes over
// 32000 keys, 28q/4kv d128: 70, 398 TFLOP/s; 32 x 8-24 nodes, 128-1024 keys: 20; 5 nodes over 37 keys: 4.0.
#include "paged_decode_common.h"

namespace mip {
namespace tree {
namespace {

using decode::f32x4_t;
using decode::fast_exp2;
using decode::kRescaleLog2;
using decode::MfmaOps;

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint4 u4(const u32x4_t& x) { return __builtin_bit_cast(uint4, x); }

constexpr int kMaxSeqs = 1024;  // sequences whose places fit in LDS; larger batches take several launches

struct TreeArgs {
  char* out;
  int64_t out_st, out_sh;  // elements
  const char* q;
  int64_t q_st, q_sh;      // elements
  const char* k;
  const char* v;
  int64_t ncb;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* cu_q;
  const int32_t* ctx_start;
  const uint64_t* mask;
  int64_t mask_st;         // words
  int mask_words;
  int hkv, group, bs, log2_bs, max_blocks;
  uint32_t group_inv;      // ceil(2^32 / group): r / group = high word of r * group_inv while r * group < 2^32
  int num_seqs, max_q_len;
  float scale_log2;
  int min_share;           // fewest steps a worker takes
  int slack;               // a cut this many steps or closer to a segment's end moves there
  float* ws_rec;           // two records a worker: m[R] | l[R] | accumulators
  int32_t* ws_start;       // first step of every sequence, then the steps of a share (null: no segment is split)
};

// Steps from a segment's end within which a cut moves there, which spares a record and its combination.
__device__ __forceinline__ int slack_of(const TreeArgs& a, int share) {
  return share / 8 > a.slack ? share / 8 : a.slack;
}

__device__ __forceinline__ float fmax2(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float fmax3(float a, float b, float c) { return fmax2(fmax2(a, b), c); }
__device__ __forceinline__ float max4(float x) {  // over the four 16-lane groups
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float y = fmax2(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return fmax2(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Transposing LDS read: in each 16-lane group, lane j supplies 4 consecutive 16-bit elements A[j][0..3];
// lane i receives A[4 k + i / 4][i % 4], k = 0..3.
typedef short v4i16_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 lds_tr16(const char* p) {
  typedef __attribute__((address_space(3))) v4i16_t lv4_t;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4_t*)(p)));
}

template <int D, int WR, int WK, int NC>
struct Shape {
  static constexpr int NW = WR * WK;               // wavefronts
  static constexpr int T = NW * kWave;             // threads
  static constexpr int R = 16 * NC * WR;           // query rows of a segment
  static constexpr int KT = 32 * WK;               // keys of a step
  static constexpr int RB = 2 * D;                 // bytes of a K / V row
  static constexpr int CPR = RB / 16;              // 16-byte chunks of a row
  static constexpr int KC = D / 32, MT = D / 16;
  static constexpr int TILE = KT * RB;             // bytes of a step's K (or V)
  static constexpr bool kPrivate = WR == 1;        // wavefronts share no keys: each fetches its own
  static constexpr int STAGE = 2 * TILE;           // shared: K | V of a step
  static constexpr int NLD = KT * CPR / T;         // shared: chunks a thread copies, each of K and V
  static constexpr int kRing = 2 * 64 * RB;        // private: a wavefront's two tiles of 32 K and 32 V rows
  static constexpr int kPark = NW * NC * MT * kWave * 16;  // every wavefront's sums, where the WK of a row meet
  static constexpr int kStages = kPrivate ? NW * kRing : 2 * STAGE;
  static constexpr int kLds = WK > 1 && kPark > kStages ? kPark : kStages;
  static constexpr int64_t kRec = 2 * R + static_cast<int64_t>(R) * D;  // floats of a record
  static_assert(NW == 4 && KT * CPR % T == 0 && MT % WK == 0, "a step splits evenly over four wavefronts");
};

// V row r keeps chunk c at c ^ vsw(r): even, so that each 32-byte segment of a transposing read stays whole,
// and the 8 rows that 32 lanes read start in distinct banks.
template <int D> __device__ __forceinline__ int vsw(int r) { return D >= 128 ? 2 * (r & 7) : 2 * ((r + (r >> 2)) & 3); }

struct Seq {
  int q0, n, ctx;
};

struct Piece {
  Seq q;
  int s, kvh, rb, last, step0, step1;  // last: the last key's index
};

// What a workgroup shares beside the stages.
struct Shared {
  int scan[4];
  int start[kMaxSeqs];  // first step of every sequence's segments
  int cu[kMaxSeqs + 1], ctx[kMaxSeqs];
  uint32_t ok[2];       // byte w: every key that wavefront w copied exists and lies in a block of the pool
};

// Node of query row r (group 1 has no 32-bit reciprocal).
__device__ __forceinline__ int node_of(const TreeArgs& a, int r) {
  return a.group_inv ? static_cast<int>(__umulhi(static_cast<uint32_t>(r), a.group_inv)) : r;
}

__device__ __forceinline__ Seq seq_of(const TreeArgs& a, int q0, int q1, int ctx) {
  Seq q;
  q.q0 = q0;
  q.n = q1 - q0;
  q.n = q.n < a.max_q_len ? q.n : a.max_q_len;
  q.n = q.n > 0 ? q.n : 0;
  q.ctx = ctx > 0 ? ctx : 0;
  return q;
}
__device__ __forceinline__ Seq seq_of(const TreeArgs& a, int s) {
  return seq_of(a, a.cu_q[s], a.cu_q[s + 1], a.ctx_start[s]);
}

// Keys of a sequence; those past the table are never read.
__device__ __forceinline__ int keys_of(const TreeArgs& a, const Seq& q) {
  const int cap = a.max_blocks * a.bs;
  return q.ctx < cap - q.n ? q.ctx + q.n : cap;
}

// The query rows of a wavefront, NC column blocks of 16 (a lane's row in each: lane % 16), with their running softmax.
template <int D, int NC>
struct Rows {
  static constexpr int KC = D / 32, MT = D / 16;
  u32x4_t q[NC][KC];  // Q^T operand; zeros in rows that are none
  int tok[NC];        // node (0 in rows that are none)
  bool live[NC];
  f32x4_t acc[NC][MT];
  f32x4_t l[NC];      // row sums by MFMA against a block of ones: every element holds the row's
  float m[NC];        // running maximum (log2 units)

  // Blocks first, first + step, ..: row `block * 16 + i16` each.
  __device__ __forceinline__ void load(const TreeArgs& a, const Piece& p, int first, int step, int i16, int grp) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int r = (first + c * step) * 16 + i16;
      const int t = node_of(a, r), g = r - t * a.group;
      live[c] = t < p.q.n;
      tok[c] = live[c] ? t : 0;
      const char* row = a.q + ((static_cast<int64_t>(p.q.q0) + tok[c]) * a.q_st +
                               static_cast<int64_t>(p.kvh * a.group + (live[c] ? g : 0)) * a.q_sh) * 2;
#pragma unroll
      for (int kc = 0; kc < KC; ++kc)
        q[c][kc] = live[c] ? *reinterpret_cast<const u32x4_t*>(row + (32 * kc + 8 * grp) * 2) : u32x4_t{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      m[c] = -INFINITY;
      l[c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[c][mt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  __device__ __forceinline__ bool finite() const {  // of the whole wavefront
    float big = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        big = fmax3(big, fmax2(fabsf(acc[c][mt][0]), fabsf(acc[c][mt][1])),
                    fmax2(fabsf(acc[c][mt][2]), fabsf(acc[c][mt][3])));
    // On the bits: the compiler takes a maximum of absolute values for a number and compares it as one.
    return __all(__float_as_uint(big) < 0x7f800000u);
  }
};

__device__ __forceinline__ uint32_t mask_window(const TreeArgs& a, const Piece& p, int tok, int key0) {
  return decode::tree_window(a.mask + (static_cast<int64_t>(p.q.q0) + tok) * a.mask_st, a.mask_words, key0 - p.q.ctx);
}

// Scores of 32 keys against a wavefront's rows, masked, and the rows' maxima brought up to date. k: the K operand of
// the two 16-key halves (lane: key 16 u + lane % 16, dims 32 kc + 8 (lane / 16) ..). real: bit k: key key0 + k
// exists and lies in the pool. sv[c][i]: row lane % 16 of block c against key 4 (lane / 16) + kKey[i].
constexpr int kKey[8] = {0, 1, 2, 3, 16, 17, 18, 19};
template <int DT, int D, int NC>
__device__ __forceinline__ void score_tile(const TreeArgs& a, const Piece& p, Rows<D, NC>& rows, const u32x4_t (&k)[2][D / 32],
                                           int key0, uint32_t real, int grp, float (&sv)[NC][8]) {
  constexpr int KC = D / 32, MT = D / 16;
  using Ops = MfmaOps<DT>;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    f32x4_t s0 = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      s0 = Ops::qk(u4(k[0][kc]), u4(rows.q[c][kc]), s0);
      s1 = Ops::qk(u4(k[1][kc]), u4(rows.q[c][kc]), s1);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sv[c][i] = i < 4 ? s0[i] : s1[i - 4];
  }
  if (real != 0xffffffffu || key0 + 31 >= p.q.ctx) {  // else: cached keys only, which everybody sees
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const uint32_t mine = (rows.live[c] ? mask_window(a, p, rows.tok[c], key0) & real : 0u) >> (4 * grp);
#pragma unroll
      for (int i = 0; i < 8; ++i) sv[c][i] = (mine >> kKey[i]) & 1u ? sv[c][i] : -INFINITY;
    }
  }
  // One wave-uniform test decides whether any row's maximum rises by more than kRescaleLog2; most tiles raise none.
  float mx[NC];
  bool need = false;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    mx[c] = fmax3(fmax3(sv[c][0], sv[c][1], sv[c][2]), fmax3(sv[c][3], sv[c][4], sv[c][5]), fmax2(sv[c][6], sv[c][7])) *
            a.scale_log2;
    need = need || mx[c] > rows.m[c] + kRescaleLog2;
  }
  if (__any(need)) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (__any(mx[c] > rows.m[c] + kRescaleLog2)) {
        const float mn = fmax2(rows.m[c], max4(mx[c]));
        const float alpha = rows.m[c] == -INFINITY ? 0.0f : fast_exp2(rows.m[c] - mn);
        rows.l[c] *= alpha;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) rows.acc[c][mt] *= alpha;
        rows.m[c] = mn;
      }
    }
  }
}

// The weights of block c from its scores: exp2(-inf - m) = 0 for a finite m; m stays -inf only while every score of the
// row is -inf, and then 0 stands for it. All weights carry a factor of 2^kLift: with it they reach 2^(kLift +
// kRescaleLog2) = 2^15, within fp16, and the smallest that fp16 holds is 2^-31 of a row's largest, so that what a
// long tail of small weights loses stays below the output's rounding (2^-32 each).
constexpr float kLift = 7.0f;
__device__ __forceinline__ void weights(const float (&sv)[8], float m, float scale_log2, float (&pr)[8]) {
  const float nm = m == -INFINITY ? 0.0f : kLift - m;
#pragma unroll
  for (int i = 0; i < 8; ++i) pr[i] = fast_exp2(fmaf(sv[i], scale_log2, nm));
}

template <class Ops> __device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(Ops::pack2(x[0], x[1]), Ops::pack2(x[2], x[3]), Ops::pack2(x[4], x[5]), Ops::pack2(x[6], x[7]));
}

// The weights' products with V^T and their sums. vt: lane (dim 16 mt + lane % 16): k index 8 grp + i stands for key
// 4 grp + i (i < 4) or 16 + 4 grp + i - 4, the keys of this lane's scores, so the weights stay where they are.
// They enter in V's type, with their rounding remainders as a second product.
template <int DT, int D, int NC>
__device__ __forceinline__ void value_tile(Rows<D, NC>& rows, const u32x4_t (&vt)[D / 16], const float (&sv)[NC][8],
                                           float scale_log2) {
  constexpr int MT = D / 16;
  using Ops = MfmaOps<DT>;
  constexpr uint32_t kOne2 = DT == MIP_BF16 ? 0x3f803f80u : 0x3c003c00u;
  const uint4 ones = make_uint4(kOne2, kOne2, kOne2, kOne2);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float pr[8];
    weights(sv[c], rows.m[c], scale_log2, pr);
    const uint4 ph = pack8<Ops>(pr);
    rows.l[c] = Ops::qk(ones, ph, rows.l[c]);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) rows.acc[c][mt] = Ops::qk(u4(vt[mt]), ph, rows.acc[c][mt]);
    const uint32_t h[4] = {ph.x, ph.y, ph.z, ph.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) pr[i] -= i & 1 ? Ops::hi(h[i / 2]) : Ops::lo(h[i / 2]);
    const uint4 pl = pack8<Ops>(pr);
    rows.l[c] = Ops::qk(ones, pl, rows.l[c]);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) rows.acc[c][mt] = Ops::qk(u4(vt[mt]), pl, rows.acc[c][mt]);
  }
}

// A wavefront's keys of a piece (32 at wk * 32 of every step of KT), for sums that ended as inf or NaN: the same
// softmax, each value added to the rows that see its key alone (0 * inf of a masked key must not reach a row), in fp32
// with the weights as they are, scaled by 2^-40: with weights of up to 2^kRescaleLog2 a sum could pass the largest
// fp32 although its mean does not. Rare, so plain: one tile at a time, no LDS.
// One column block, so that few registers are needed beside the other blocks' sums.
template <int DT, int D, int KT>
__device__ __forceinline__ void careful_block(const TreeArgs& a, const Piece& p, Rows<D, 1>& rows, int wk, int lane) {
  constexpr int KC = D / 32, MT = D / 16;
  constexpr float kBias = 40.0f;
  const int i16 = lane & 15, grp = lane >> 4;
  const int32_t* table = a.bt + static_cast<int64_t>(p.s) * a.bt_stride;
  rows.clear();
  auto row_of = [&](int key, bool& ok) {
    const int b = table[key >> a.log2_bs];
    ok = b >= 0 && b < a.ncb;
    return static_cast<uint64_t>(ok ? static_cast<uint32_t>(b) : 0u) * static_cast<uint32_t>(a.hkv * a.bs) +
           static_cast<uint32_t>(p.kvh * a.bs + (key & (a.bs - 1)));
  };
#pragma unroll 1
  for (int t = p.step0; t < p.step1; ++t) {
    const int key0 = t * KT + wk * 32;
    if (key0 > p.last) break;
    bool ok;
    const int mine = key0 + (lane & 31);
    row_of(mine < p.last ? mine : p.last, ok);
    const uint32_t real = static_cast<uint32_t>(__ballot(ok && mine <= p.last));
    float sv[1][8];
    {
      u32x4_t k[2][KC];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int key = key0 + 16 * u + i16;
        const char* row = a.k + row_of(key < p.last ? key : p.last, ok) * (2 * D) + 16 * grp;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) k[u][kc] = *reinterpret_cast<const u32x4_t*>(row + 64 * kc);
      }
      score_tile<DT, D, 1>(a, p, rows, k, key0, real, grp, sv);
    }
    const uint32_t win = rows.live[0] ? mask_window(a, p, rows.tok[0], key0) & real : 0u;
    float pr[8];
    weights(sv[0], rows.m[0] + kBias, a.scale_log2, pr);
#pragma unroll 1
    for (int kk = 0; kk < 32; ++kk) {
      const int e = (kk & 3) + (kk >= 16 ? 4 : 0);
      float pk = pr[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) pk = e == i ? pr[i] : pk;
      pk = __shfl(pk, ((kk & 15) >> 2) * 16 + i16);
      if (!((real >> kk) & 1u)) continue;
      const uint16_t* v = reinterpret_cast<const uint16_t*>(a.v + row_of(key0 + kk, ok) * (2 * D)) + 4 * grp;
      if (!((win >> kk) & 1u)) continue;
      rows.l[0] += pk;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) rows.acc[0][mt][i] += pk * widen<DT>(v[16 * mt + i]);
    }
  }
  rows.m[0] += kBias;  // what the sums are relative to
}

template <int DT, int D, int NC, int KT>
__device__ __forceinline__ void careful_pass(const TreeArgs& a, const Piece& p, Rows<D, NC>& rows, int first, int step, int wk,
                                             int lane) {
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    Rows<D, 1> one;
    one.load(a, p, first + c * step, 0, lane & 15, lane >> 4);
    careful_block<DT, D, KT>(a, p, one, wk, lane);
    rows.m[c] = one.m[0];
    rows.l[c] = one.l[0];
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt) rows.acc[c][mt] = one.acc[0][mt];
  }
}

// Direct global -> LDS loads: 64 lanes x 16 bytes to l + 16 lane. K/V rows of a private pass are read once a call: the
// nontemporal policy.
typedef __attribute__((address_space(1))) void gvoid_t;
typedef __attribute__((address_space(3))) void lvoid_t;
typedef __attribute__((address_space(3))) char lchar_t;
__device__ __forceinline__ void dma16(const char* g, lchar_t* l) {
  __builtin_amdgcn_global_load_lds((gvoid_t*)g, (lvoid_t*)l, 16, 0, 2);
}
template <int N> __device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt field is 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));  // no wait on the other counters
}

// LDS reads of a ring tile. They are asm because the compiler cannot tell which tile a direct load fills and would
// drain every load before each read; each block waits for its own reads.
template <int D> struct RingRead;
template <> struct RingRead<64> {
  static __device__ __forceinline__ void k(u32x4_t (&k)[2][2], const uint32_t (&at)[2]) {
    asm volatile(
        "ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:2048\n\t"
        "ds_read_b128 %3, %5 offset:2048\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[1][0]), "=&v"(k[1][1])
        : "v"(at[0]), "v"(at[1])
        : "memory");
  }
};
template <> struct RingRead<128> {
  static __device__ __forceinline__ void k(u32x4_t (&k)[2][4], const uint32_t (&at)[4]) {
    asm volatile(
        "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
        "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %9 offset:4096\n\tds_read_b128 %6, %10 offset:4096\n\t"
        "ds_read_b128 %7, %11 offset:4096\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[0][2]), "=&v"(k[0][3]), "=&v"(k[1][0]), "=&v"(k[1][1]),
          "=&v"(k[1][2]), "=&v"(k[1][3])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
        : "memory");
  }
};
// V^T of four 16-dim tiles: rows 4 grp .. and 16 + 4 grp .. (HALF bytes on), transposed.
template <int HALF>
__device__ __forceinline__ void ring_v4(u32x2_t (&lo)[4], u32x2_t (&hi)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %9\n\tds_read_b64_tr_b16 %2, %10\n\t"
      "ds_read_b64_tr_b16 %3, %11\n\tds_read_b64_tr_b16 %4, %8 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %10 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3])
      : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "i"(HALF)
      : "memory");
}

// A wavefront's keys of a piece, fetched by itself: 32 of every step of 128. Direct loads fill its two LDS tiles of
// K and V rows in turn, the next tile's while this one is computed, so loads in flight cost no registers and
// wavefronts never wait for each other. Row r keeps its 16-byte chunk c at c ^ (r % CPR) (K) or c ^ vsw(r) (V), by the
// choice of the chunk that each lane fetches.
template <int DT, int D, int NC>
__device__ __forceinline__ void private_pass(const TreeArgs& a, const Piece& p, Rows<D, NC>& rows, lchar_t* ring, int wk,
                                             int lane) {
  constexpr int KC = D / 32, MT = D / 16, RB = 2 * D, CPR = RB / 16, RPD = kWave / CPR, ND = 32 / RPD;
  constexpr int TILE = 64 * RB, V_OFF = 32 * RB;
  const int i16 = lane & 15, grp = lane >> 4;
  const int32_t* table = a.bt + static_cast<int64_t>(p.s) * a.bt_stride;
  const int last = p.last, ncb = static_cast<int>(a.ncb);
  const uint32_t per_block = static_cast<uint32_t>(a.hkv * a.bs), head = static_cast<uint32_t>(p.kvh * a.bs);
  rows.clear();
  // Tiles of this wavefront: steps whose first key of its 32 exists.
  const int mine = last < wk * 32 ? 0 : (last - wk * 32) / 128 + 1;
  const int t1 = p.step1 < mine ? p.step1 : mine;
  if (p.step0 >= t1) return;

  const bool wide = a.bs >= 16;  // each half of a tile lies in one block, found by a scalar load
  int id0 = 0, id1 = 0;          // of the tile that is fetched next
  auto lookup = [&](int t) __attribute__((always_inline)) {
    if (!wide) return;
    const int key0 = t * 128 + wk * 32, key1 = key0 + 16 < last ? key0 + 16 : last;
    id0 = load_uniform_i32(table + (key0 >> a.log2_bs));
    id1 = load_uniform_i32(table + (key1 >> a.log2_bs));
  };
  // Start the loads of tile t into `to`; returns which of its keys exist and lie in the pool. Keys past the last one
  // stand for it, block ids outside the pool for block 0.
  auto fetch = [&](int t, lchar_t* to) __attribute__((always_inline)) -> uint32_t {
    const int key0 = t * 128 + wk * 32;
    uint32_t real = last - key0 >= 31 ? 0xffffffffu : (2u << (last - key0)) - 1u;
    const bool ok0 = id0 >= 0 && id0 < ncb, ok1 = id1 >= 0 && id1 < ncb;
    if (wide)
      real &= (ok0 ? 0xffffu : 0u) | (ok1 ? 0xffff0000u : 0u);
    else {
      const int key = key0 + (lane & 31), b = table[(key < last ? key : last) >> a.log2_bs];
      real &= static_cast<uint32_t>(__ballot(b >= 0 && b < ncb));
    }
#pragma unroll
    for (int j = 0; j < ND; ++j) {
      const int r = j * RPD + lane / CPR, c = lane % CPR;
      const int key = key0 + r < last ? key0 + r : last;
      int blk;
      if (wide) {
        blk = j * RPD < 16 ? (ok0 ? id0 : 0) : (ok1 ? id1 : 0);
      } else {
        blk = table[key >> a.log2_bs];
        blk = blk >= 0 && blk < ncb ? blk : 0;
      }
      const uint64_t row = static_cast<uint64_t>(static_cast<uint32_t>(blk)) * per_block +
                           (head + static_cast<uint32_t>(key & (a.bs - 1)));
      dma16(a.k + row * RB + ((c ^ (r & (CPR - 1))) * 16), to + j * 1024);
      dma16(a.v + row * RB + ((c ^ vsw<D>(r)) * 16), to + V_OFF + j * 1024);
    }
    return real;
  };

  uint32_t k_at[KC], v_at[MT];
  const int vrow = 4 * grp + (i16 >> 2);  // rows vrow and vrow + 16 share vsw
#pragma unroll
  for (int kc = 0; kc < KC; ++kc)
    k_at[kc] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ring)) + i16 * RB + (((4 * kc + grp) ^ (i16 & (CPR - 1))) * 16);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
    v_at[mt] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ring)) + V_OFF + vrow * RB + (i16 & 3) * 8 +
               (((2 * mt) ^ vsw<D>(vrow)) * 16);
  lookup(p.step0);
  uint32_t real = fetch(p.step0, ring), next = 0;
  if (p.step0 + 1 < t1) lookup(p.step0 + 1);
  uint32_t flip = 0;  // byte offset of the tile in use
  for (int t = p.step0; t < t1; ++t) {
    if (t + 1 < t1) {
      next = fetch(t + 1, ring + (flip ^ TILE));
      if (t + 2 < t1) lookup(t + 2);
      wait_vmcnt<2 * ND>();
    } else {
      wait_vmcnt<0>();
    }
    u32x4_t k[2][KC];
    uint32_t at[KC];
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) at[kc] = k_at[kc] + flip;
    RingRead<D>::k(k, at);
    float sv[NC][8];
    score_tile<DT, D, NC>(a, p, rows, k, t * 128 + wk * 32, real, grp, sv);
    u32x4_t vt[MT];
#pragma unroll
    for (int q = 0; q < MT / 4; ++q) {
      u32x2_t lo[4], hi[4];
      ring_v4<16 * RB>(lo, hi, v_at[4 * q] + flip, v_at[4 * q + 1] + flip, v_at[4 * q + 2] + flip, v_at[4 * q + 3] + flip);
#pragma unroll
      for (int i = 0; i < 4; ++i) vt[4 * q + i] = u32x4_t{lo[i][0], lo[i][1], hi[i][0], hi[i][1]};
    }
    value_tile<DT, D, NC>(rows, vt, sv, a.scale_log2);
    real = next;
    flip ^= TILE;
  }
}

// A workgroup's keys of a piece, staged by all its threads for all its wavefronts: two LDS stages of a step, the
// next step's rows in registers meanwhile. WR x WK wavefronts: WK take different 32 keys of a step.
template <int DT, int D, int WR, int WK, int NCK, int NC>
__device__ __forceinline__ void shared_pass(const TreeArgs& a, const Piece& p, Rows<D, NC>& rows, char* smem, Shared& sh,
                                            int w, int lane) {
  using P = Shape<D, WR, WK, NCK>;
  constexpr int KC = P::KC, MT = P::MT, RB = P::RB, CPR = P::CPR, NLD = P::NLD;
  const int tid = w * kWave + lane, wk = w % WK, i16 = lane & 15, grp = lane >> 4;
  const int32_t* table = a.bt + static_cast<int64_t>(p.s) * a.bt_stride;
  const int last = p.last;
  rows.clear();
  // A wavefront's chunks of one copy are RW consecutive rows of one block (blocks have RW rows at least), 1 KB: block
  // and address are scalar, a lane's part of the address is a constant but in the segment's last step, where keys past
  // the last one stand for it (addresses by lane: 69.3 -> 67.4 us for one tree of 61 nodes over 32000 keys).
  constexpr int RW = kWave / CPR, RJ = P::T / CPR;
  u32x4_t kbuf[NLD], vbuf[NLD];
  bool okbuf = true;
  int bid[NLD];  // of the step that is fetched next
  uint32_t mine[NLD];
#pragma unroll
  for (int j = 0; j < NLD; ++j) mine[j] = lane * 16;
  const int ncb = static_cast<int>(a.ncb), inside = a.bs - 1, w0 = w * RW;
  const uint32_t per_block = static_cast<uint32_t>(a.hkv * a.bs), head = static_cast<uint32_t>(p.kvh * a.bs);
  auto lookup = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NLD; ++j) {
      const int key = t * P::KT + j * RJ + w0;
      bid[j] = load_uniform_i32(table + ((key < last ? key : last) >> a.log2_bs));
    }
  };
  auto fetch = [&](int t) __attribute__((always_inline)) {
    okbuf = true;
    const bool whole = t * P::KT + P::KT - 1 <= last;
    if (!whole) {
#pragma unroll
      for (int j = 0; j < NLD; ++j) {
        const int key = t * P::KT + j * RJ + w0, from = key < last ? key : last;
        const int mid = key + lane / CPR < last ? key + lane / CPR : last;  // at `from` or behind it, in the same block
        mine[j] = static_cast<uint32_t>(mid - from) * RB + lane % CPR * 16;
      }
      okbuf = false;
    }
#pragma unroll
    for (int j = 0; j < NLD; ++j) {
      const int key = t * P::KT + j * RJ + w0, from = key < last ? key : last;
      const bool bok = bid[j] >= 0 && bid[j] < ncb;
      const uint64_t row = static_cast<uint64_t>(bok ? static_cast<uint32_t>(bid[j]) : 0u) * per_block +
                           (head + static_cast<uint32_t>(from & inside));
      kbuf[j] = *reinterpret_cast<const u32x4_t*>(a.k + row * RB + mine[j]);
      vbuf[j] = *reinterpret_cast<const u32x4_t*>(a.v + row * RB + mine[j]);
      okbuf = okbuf && bok;
    }
  };
  auto stash = [&](int stage) __attribute__((always_inline)) {
    char* st = smem + stage * P::STAGE;
#pragma unroll
    for (int j = 0; j < NLD; ++j) {
      const int idx = tid + j * P::T, r = idx / CPR, c = idx % CPR;
      *reinterpret_cast<u32x4_t*>(st + r * RB + ((c ^ (r & (CPR - 1))) * 16)) = kbuf[j];
      *reinterpret_cast<u32x4_t*>(st + P::TILE + r * RB + ((c ^ vsw<D>(r)) * 16)) = vbuf[j];
    }
    if (lane == 0) reinterpret_cast<uint8_t*>(&sh.ok[stage])[w] = okbuf ? 1 : 0;
  };
  lookup(p.step0);
  fetch(p.step0);
  if (p.step0 + 1 < p.step1) lookup(p.step0 + 1);
  stash(0);
  __syncthreads();
  for (int t = p.step0; t < p.step1; ++t) {
    const int stage = (t - p.step0) & 1;
    if (t + 1 < p.step1) {
      fetch(t + 1);
      if (t + 2 < p.step1) lookup(t + 2);
    }
    const char* st = smem + stage * P::STAGE + wk * 32 * RB;
    const int key0 = t * P::KT + wk * 32;
    if (key0 <= last) {
      u32x4_t k[2][KC];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          const int r = 16 * u + i16, ch = 4 * kc + grp;
          k[u][kc] = *reinterpret_cast<const u32x4_t*>(st + r * RB + ((ch ^ (r & (CPR - 1))) * 16));
        }
      }
      u32x4_t vt[MT];
      const int vrow = 4 * grp + (i16 >> 2), vs = vsw<D>(vrow);  // rows vrow and vrow + 16 share vsw
      const char* vr = st + P::TILE + vrow * RB + (i16 & 3) * 8;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int so = ((2 * mt) ^ vs) * 16;
        const uint2 lo = lds_tr16(vr + so), hi = lds_tr16(vr + 16 * RB + so);
        vt[mt] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
      }
      uint32_t real = 0xffffffffu;
      if (__builtin_amdgcn_readfirstlane(sh.ok[stage]) != 0x01010101u) {  // the tile's keys one by one
        const int key = key0 + (lane & 31);
        const int b = table[(key < last ? key : last) >> a.log2_bs];
        real = static_cast<uint32_t>(__ballot(key <= last && b >= 0 && b < a.ncb));
      }
      float sv[NC][8];
      score_tile<DT, D, NC>(a, p, rows, k, key0, real, grp, sv);
      value_tile<DT, D, NC>(rows, vt, sv, a.scale_log2);
    }
    if (t + 1 < p.step1) stash(stage ^ 1);
    __syncthreads();
  }
}

// Output rows of a column block, or its part of a record (accumulators as the lanes hold them, [block][mt][lane]).
template <int DT, int D, int R, int N>
__device__ __forceinline__ void put_block(const TreeArgs& a, const Piece& p, float* rec, int cb, int mt0, bool live, int tok,
                                          float m, float l, const f32x4_t (&acc)[N], int lane) {
  using Ops = MfmaOps<DT>;
  using S = typename Elem<DT>::S;
  const int i16 = lane & 15, grp = lane >> 4;
  if (!__any(live)) return;
  if (rec) {
    f32x4_t* out = reinterpret_cast<f32x4_t*>(rec + 2 * R) + (cb * (D / 16) + mt0) * kWave + lane;
#pragma unroll
    for (int x = 0; x < N; ++x) out[x * kWave] = acc[x];
    if (mt0 == 0 && grp == 0) {
      rec[cb * 16 + i16] = m;
      rec[R + cb * 16 + i16] = l;
    }
    return;
  }
  if (!live) return;
  const float inv = l == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(l);  // to 2^-23; 0: no key seen, sums of 0
  const int r = p.rb * R + cb * 16 + i16;
  S* row = reinterpret_cast<S*>(a.out) + (static_cast<int64_t>(p.q.q0) + tok) * a.out_st +
           static_cast<int64_t>(p.kvh * a.group + r - tok * a.group) * a.out_sh;
#pragma unroll
  for (int x = 0; x < N; ++x) {
    const uint32_t w0 = Ops::pack2(acc[x][0] * inv, acc[x][1] * inv), w1 = Ops::pack2(acc[x][2] * inv, acc[x][3] * inv);
    *reinterpret_cast<uint2*>(row + 16 * (mt0 + x) + 4 * grp) = make_uint2(w0, w1);
  }
}

// One piece: rows of block p.rb against steps [p.step0, p.step1). rec: null where that is the whole segment. NC: column
// blocks of a wavefront here, at most the kernel's.
template <int DT, int D, int WR, int WK, int NCK, int NC>
__device__ __forceinline__ void run_piece(const TreeArgs& a, const Piece& p, float* rec, char* smem, Shared& sh,
                                          float (*sh_ml)[4][16 * NCK]) {
  using P = Shape<D, WR, WK, NCK>;
  constexpr int MT = P::MT;
  const int lane = threadIdx.x & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wr = w / WK, wk = w % WK, i16 = lane & 15, grp = lane >> 4;
  Rows<D, NC> rows;
  const int first = p.rb * (P::R / 16) + wr;
  rows.load(a, p, first, WR, i16, grp);
  if constexpr (P::kPrivate) {
    private_pass<DT, D, NC>(a, p, rows, (lchar_t*)(smem + w * P::kRing), wk, lane);
  } else {
    shared_pass<DT, D, WR, WK, NCK, NC>(a, p, rows, smem, sh, w, lane);
  }
  // A wavefront whose accumulators hold inf or NaN does its part again.
  if (!rows.finite()) careful_pass<DT, D, NC, P::KT>(a, p, rows, first, WR, wk, lane);
  if constexpr (WK == 1) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      put_block<DT, D, P::R, MT>(a, p, rec, c * WR + wr, 0, rows.live[c], rows.tok[c], rows.m[c], rows.l[c][0], rows.acc[c],
                                 lane);
  } else {
    // The WK wavefronts of a row meet: each scales its sums to the common maximum, and each takes MT / WK of
    // the dims of every column block.
    constexpr int PER = MT / WK;
    if (grp == 0) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        sh_ml[0][w][c * 16 + i16] = rows.m[c];
        sh_ml[1][w][c * 16 + i16] = rows.l[c][0];
      }
    }
    __syncthreads();  // also: every wavefront is done with its stage
    f32x4_t* park = reinterpret_cast<f32x4_t*>(smem);
    float m[NC], l[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      m[c] = -INFINITY;
      l[c] = 0.0f;
#pragma unroll
      for (int o = 0; o < WK; ++o) m[c] = fmax2(m[c], sh_ml[0][wr * WK + o][c * 16 + i16]);
#pragma unroll
      for (int o = 0; o < WK; ++o) {
        const float mo = sh_ml[0][wr * WK + o][c * 16 + i16];
        // A wavefront without keys has sums of 0 and a maximum of -inf (and so may all).
        l[c] += sh_ml[1][wr * WK + o][c * 16 + i16] * (mo == -INFINITY ? 0.0f : fast_exp2(mo - m[c]));
      }
      const float f = rows.m[c] == -INFINITY ? 0.0f : fast_exp2(rows.m[c] - m[c]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) park[((w * NC + c) * MT + mt) * kWave + lane] = rows.acc[c][mt] * f;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      f32x4_t sum[PER];
#pragma unroll
      for (int x = 0; x < PER; ++x) {
        sum[x] = park[((wr * WK * NC + c) * MT + wk * PER + x) * kWave + lane];
#pragma unroll
        for (int o = 1; o < WK; ++o) sum[x] += park[(((wr * WK + o) * NC + c) * MT + wk * PER + x) * kWave + lane];
      }
      put_block<DT, D, P::R, PER>(a, p, rec, c * WR + wr, wk * PER, rows.live[c], rows.tok[c], m[c], l[c], sum, lane);
    }
    __syncthreads();  // the next piece fetches over the parked sums
  }
}

__device__ __forceinline__ int segments_of(const TreeArgs& a, const Seq& q, int rows) {
  return (q.n * a.group + rows - 1) / rows * a.hkv;
}

template <int DT, int D, int WR, int WK, int NC, int OCC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void paged_tree_kernel(TreeArgs a) {
  using P = Shape<D, WR, WK, NC>;
  __shared__ __attribute__((aligned(16))) char smem[P::kLds];
  __shared__ Shared sh;
  __shared__ float sh_ml[2][4][16 * NC];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = tid / kWave;
  const int S = a.num_seqs;
  auto steps_of = [&](const Seq& q) { return (keys_of(a, q) + P::KT - 1) / P::KT; };

  // ---- the place of every sequence's steps in the call's one row of steps.
  int total = 0;
  for (int s0 = 0; s0 < S; s0 += P::T) {
    const int s = s0 + tid;
    int n = 0;
    if (s < S) {
      const int q0 = a.cu_q[s], q1 = a.cu_q[s + 1], ctx = a.ctx_start[s];
      const Seq q = seq_of(a, q0, q1, ctx);
      sh.cu[s] = q0;
      if (s == S - 1) sh.cu[S] = q1;
      sh.ctx[s] = ctx;
      n = segments_of(a, q, P::R) * steps_of(q);
    }
    const int incl = decode::wave_inclusive_scan(n, lane);
    if (lane == kWave - 1) sh.scan[w] = incl;
    __syncthreads();
    int before = total;
#pragma unroll
    for (int i = 0; i < P::NW; ++i) {
      before += i < w ? sh.scan[i] : 0;
      total += sh.scan[i];
    }
    if (s < S) sh.start[s] = before + incl - n;
    __syncthreads();
  }

  // ---- equal shares: worker i takes steps [i * share, i * share + share). The workers of an XCD are neighbours, so
  // that row blocks of the same keys meet in its L2.
  int share = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  share = share > a.min_share ? share : a.min_share;
  const int workers = (total + share - 1) / share, per_xcd = (workers + 7) / 8;
  const int worker = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (a.ws_start && blockIdx.x == 0) {  // for the second kernel
    for (int s = tid; s < S; s += P::T) a.ws_start[s] = sh.start[s];
    if (tid == 0) a.ws_start[S] = share;
  }
  if (static_cast<int>(blockIdx.x >> 3) >= per_xcd || worker >= workers) return;
  const int slack = slack_of(a, share);
  auto known = [&](int s) {
    Seq q = seq_of(a, sh.cu[s], sh.cu[s + 1], sh.ctx[s]);
    return Seq{__builtin_amdgcn_readfirstlane(q.q0), __builtin_amdgcn_readfirstlane(q.n),
               __builtin_amdgcn_readfirstlane(q.ctx)};
  };
  auto cut = [&](int at, int& s) {
    if (at >= total) return total;
    int lo = 0, hi = S - 1;  // the last sequence that starts at or before `at`
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sh.start[mid] <= at) lo = mid; else hi = mid - 1;
    }
    s = __builtin_amdgcn_readfirstlane(lo);
    const int nt = steps_of(known(s)), into = (at - __builtin_amdgcn_readfirstlane(sh.start[s])) % nt;
    return into < slack ? at - into : nt - into < slack ? at + nt - into : at;
  };
  int s = 0, dummy;
  int at = cut(worker * share, s);
  const int end = cut(worker * share + share, dummy);
  for (; at < end; ++s) {
    Piece p;
    p.s = __builtin_amdgcn_readfirstlane(s);
    p.q = known(p.s);
    p.last = keys_of(a, p.q) - 1;
    const int nt = steps_of(p.q), nrb = (p.q.n * a.group + P::R - 1) / P::R, segs = nrb * a.hkv;
    const int first = __builtin_amdgcn_readfirstlane(sh.start[s]);
    while (at < end && at < first + segs * nt) {
      const int seg = (at - first) / nt, seg0 = first + seg * nt;
      p.kvh = seg / nrb;
      p.rb = seg - p.kvh * nrb;
      p.step0 = at - seg0;
      p.step1 = end - seg0 < nt ? end - seg0 : nt;
      float* rec = nullptr;
      // A worker's first piece, if it begins inside its segment, has record 0, its last, if it ends inside, 1.
      if (p.step0 > 0 || p.step1 < nt)
        rec = a.ws_rec + (static_cast<int64_t>(worker) * 2 + (p.step0 > 0 ? 0 : 1)) * P::kRec;
      // Column blocks that each wavefront has of the segment's, so that none is spent on rows that are none.
      const int left = (p.q.n * a.group + 15) / 16 - p.rb * (P::R / 16);
      const int nc = ((left < P::R / 16 ? left : P::R / 16) + WR - 1) / WR;
      if (NC >= 4 && nc == 4) run_piece<DT, D, WR, WK, NC, NC < 4 ? NC : 4>(a, p, rec, smem, sh, sh_ml);
      else if (NC >= 3 && nc == 3) run_piece<DT, D, WR, WK, NC, NC < 3 ? NC : 3>(a, p, rec, smem, sh, sh_ml);
      else if (NC >= 2 && nc == 2) run_piece<DT, D, WR, WK, NC, NC < 2 ? NC : 2>(a, p, rec, smem, sh, sh_ml);
      else run_piece<DT, D, WR, WK, NC, 1>(a, p, rec, smem, sh, sh_ml);
      at = seg0 + p.step1;
    }
  }
}

// Combine the pieces of a split segment x = (sequence, (kv head, row block)). BY_PIECE: workgroup (x, cb, z) takes two
// dim tiles (z) of column block cb, each wavefront a quarter of the pieces (few segments, cut into many pieces each:
// more workgroups and shorter chains). Else every wavefront of workgroup (x, y) a whole column block of its own, 4 y + w
// (64 x 33-64 nodes of 7 rows, d64, 33 MB of records: 10.7 us, 13.8 with a quarter of a block's dims a wavefront).
template <int DT, int D, int R, bool BY_PIECE>
__global__ __launch_bounds__(256) void paged_tree_merge(TreeArgs a, int segs_per_seq, int keys_per_step) {
  constexpr int MT = D / 16, PER = BY_PIECE ? 2 : MT;
  const int lane = threadIdx.x & (kWave - 1), i16 = lane & 15, w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int s = blockIdx.x / segs_per_seq, seg = blockIdx.x - s * segs_per_seq;
  const int cb = BY_PIECE ? blockIdx.y : blockIdx.y * 4 + w;
  if (cb >= R / 16) return;  // shapes of fewer than four column blocks (whole wavefronts; BY_PIECE has none such)
  Piece p;
  p.s = s;
  p.q = seq_of(a, s);
  const int first = a.ws_start[s], share = a.ws_start[a.num_seqs];
  const int nt = (keys_of(a, p.q) + keys_per_step - 1) / keys_per_step;
  const int nrb = (p.q.n * a.group + R - 1) / R, segs = nrb * a.hkv;
  if (seg >= segs) return;
  // The cuts inside the segment: the multiples of `share` that did not move to one of its ends. Worker w0 has the
  // first piece, w0 + 1 .. w1 have the others.
  const int begin = first + seg * nt, near = slack_of(a, share);
  const int w0 = (begin + near - 1) / share, w1 = (begin + nt - near) / share;
  if (w0 >= w1) return;
  p.kvh = seg / nrb;
  p.rb = seg - p.kvh * nrb;
  if (p.rb * R + cb * 16 >= p.q.n * a.group) return;
  const int mt0 = BY_PIECE ? 2 * blockIdx.z : 0;
  constexpr int64_t kRec = 2 * R + static_cast<int64_t>(R) * D;
  // The segment's first piece ends inside it (record 1 of its worker); the others begin inside it (record 0).
  auto record = [&](int x) { return a.ws_rec + (static_cast<int64_t>(x) * 2 + (x == w0 ? 1 : 0)) * kRec; };
  const int from = BY_PIECE ? w0 + (w1 - w0 + 1) * w / 4 : w0, to = BY_PIECE ? w0 + (w1 - w0 + 1) * (w + 1) / 4 : w1 + 1;
  float m = -INFINITY, l = 0.0f;
#pragma unroll 8
  for (int x = from; x < to; ++x) m = fmax2(m, record(x)[cb * 16 + i16]);
  f32x4_t acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int x = from; x < to; ++x) {
    const float* rec = record(x);
    const float mp = rec[cb * 16 + i16];
    const float f = mp == -INFINITY ? 0.0f : fast_exp2(mp - m);
    l += f * rec[R + cb * 16 + i16];
    const f32x4_t* racc = reinterpret_cast<const f32x4_t*>(rec + 2 * R) + (cb * MT + mt0) * kWave + lane;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] += racc[i * kWave] * f;
  }
  if constexpr (BY_PIECE) {
    __shared__ float s_ml[2][4][16];
    __shared__ f32x4_t s_acc[4][PER][kWave];
    if (lane < 16) {
      s_ml[0][w][i16] = m;
      s_ml[1][w][i16] = l;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) s_acc[w][i][lane] = acc[i];
    __syncthreads();
    if (w > 0) return;
    m = fmax2(fmax2(s_ml[0][0][i16], s_ml[0][1][i16]), fmax2(s_ml[0][2][i16], s_ml[0][3][i16]));
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      const float mo = s_ml[0][o][i16], f = mo == -INFINITY ? 0.0f : fast_exp2(mo - m);
      l += f * s_ml[1][o][i16];
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] += s_acc[o][i][lane] * f;
    }
  }
  const int r = p.rb * R + cb * 16 + i16, tok = node_of(a, r);
  put_block<DT, D, R, PER>(a, p, nullptr, cb, mt0, tok < p.q.n, tok, m, l, acc, lane);
}

// ------------------------------------------------------------------ one query row at a time
//
// Every type, head size (powers of two from 8 to 256), group and alignment of elements: a workgroup of 4
// wavefronts per (node, query head). A lane holds 16 bytes of a row, LPR lanes a row, so a wavefront
// takes 64 / LPR keys at once and every key's row lanes keep a softmax state of their own (a score is summed
// over its LPR lanes alone); the states meet at the end. A key that the row does not see contributes
// nothing at all, whatever its bytes are.
// Bound by latency at the sizes that it is for (5 nodes over 37 keys, 14 heads of 64: 4.0 us a call).
// Long contexts of few rows are cut into parts of `tokens` keys (blockIdx.z), which leave their states in
// ml [x][head][part][2] and acc [x][head][part][D], x = s * max_q_len + i of node i of sequence s.
struct PartArgs {
  int hq, tokens, parts;
  float* ml;
  float* acc;
};

template <int DT, int D>
__global__ __launch_bounds__(256) void paged_tree_row_kernel(TreeArgs a, PartArgs pt) {
  using S = typename Elem<DT>::S;
  constexpr int ES = Elem<DT>::kBytes, N = 16 / ES, LPR = D / N > 0 ? D / N : 1, RPP = kWave / LPR;
  static_assert(D % N == 0 && LPR <= kWave, "a row is whole 16-byte chunks, at most 64");
  constexpr int kStates = 4 * RPP;
  __shared__ float s_m[kStates], s_l[kStates];
  __shared__ float s_acc[kStates][D];
  const int64_t x = blockIdx.x;  // (sequence, node)
  const int s = static_cast<int>(x / a.max_q_len), i = static_cast<int>(x - static_cast<int64_t>(s) * a.max_q_len);
  const Seq p = seq_of(a, s);
  if (i >= p.n) return;
  const int all = keys_of(a, p), np = (all + pt.tokens - 1) / pt.tokens, part = blockIdx.z;
  if (part >= np) return;
  const int first = part * pt.tokens, keys = first + pt.tokens < all ? first + pt.tokens : all;
  const int h = blockIdx.y, kvh = h / a.group;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = tid / kWave;
  const int row = lane / LPR, c = lane % LPR;
  const int64_t r = static_cast<int64_t>(p.q0) + i;
  const S* q = reinterpret_cast<const S*>(a.q) + r * a.q_st + static_cast<int64_t>(h) * a.q_sh + c * N;
  const uint64_t* mask = a.mask + r * a.mask_st;
  const int32_t* table = a.bt + static_cast<int64_t>(s) * a.bt_stride;
  float qf[N], acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    qf[e] = widen<DT>(q[e]);
    acc[e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  // A step: U keys for every row of lanes, their block ids read one step ahead and all of their K and V
  // requested before any is used.
  constexpr int U = RPP >= 16 ? 1 : RPP >= 8 ? 2 : 4, STEP = 4 * RPP * U;
  int ids[U];
  bool in[U];
  auto lookup = [&](int base) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = base + (u * 4 + w) * RPP + row, e0 = key - p.ctx;
      in[u] = key < keys;
      ids[u] = in[u] ? table[key >> a.log2_bs] : -1;
      if (in[u] && e0 >= 0) in[u] = (e0 >> 6) < a.mask_words && ((mask[e0 >> 6] >> (e0 & 63)) & 1u);
    }
  };
  lookup(first);
  for (int base = first; base < keys; base += STEP) {
    u32x4_t kw[U], vw[U];
    bool seen[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = base + (u * 4 + w) * RPP + row;
      const bool ok = ids[u] >= 0 && ids[u] < a.ncb;
      seen[u] = ok && in[u];
      const int64_t at =
          (((static_cast<int64_t>(ok ? ids[u] : 0) * a.hkv + kvh) * a.bs + (key & (a.bs - 1))) * D + c * N) * ES;
      kw[u] = *reinterpret_cast<const u32x4_t*>(a.k + at);
      vw[u] = *reinterpret_cast<const u32x4_t*>(a.v + at);
    }
    if (base + STEP < keys) lookup(base + STEP);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      S kr[N], vr[N];
      __builtin_memcpy(kr, &kw[u], 16);
      __builtin_memcpy(vr, &vw[u], 16);
      float dot = 0.0f;
#pragma unroll
      for (int e = 0; e < N; ++e) dot = fmaf(qf[e], widen<DT>(kr[e]), dot);
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) dot += __shfl_xor(dot, o);
      const float sc = dot * a.scale_log2;  // -inf also where a finite product's score is below fp32: it weighs nothing
      if (!seen[u] || sc == -INFINITY) continue;
      const float mn = fmax2(m, sc);
      const float alpha = fast_exp2(m - mn), pk = fast_exp2(sc - mn);  // m = -inf before any key: alpha 0
      l = l * alpha + pk;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = fmaf(pk, widen<DT>(vr[e]), acc[e] * alpha);
      m = mn;
    }
  }
  const int state = w * RPP + row;
#pragma unroll
  for (int e = 0; e < N; ++e) s_acc[state][c * N + e] = acc[e];
  if (c == 0) {
    s_m[state] = m;
    s_l[state] = l;
  }
  __syncthreads();
  for (int d = tid; d < D; d += 256) {
    float top = -INFINITY;
    for (int k = 0; k < kStates; ++k) top = fmax2(top, s_m[k]);
    float A = 0.0f, Ls = 0.0f;
    for (int k = 0; k < kStates; ++k) {
      const float f = s_m[k] == -INFINITY ? 0.0f : fast_exp2(s_m[k] - top);
      A = fmaf(f, s_acc[k][d], A);
      Ls = fmaf(f, s_l[k], Ls);
    }
    if (np == 1) {
      reinterpret_cast<S*>(a.out)[r * a.out_st + static_cast<int64_t>(h) * a.out_sh + d] =
          from_f32<DT>(Ls == 0.0f ? 0.0f : A / Ls);
    } else {
      const int64_t slot = (x * pt.hq + h) * pt.parts + part;
      pt.acc[slot * D + d] = A;
      if (d == 0) {
        pt.ml[2 * slot] = top;
        pt.ml[2 * slot + 1] = Ls;
      }
    }
  }
}

// Combine the parts of every (node, query head) that has more than one: a wavefront each.
template <int DT>
__global__ __launch_bounds__(kWave) void paged_tree_parts_kernel(TreeArgs a, PartArgs pt, int dim) {
  using S = typename Elem<DT>::S;
  const int64_t x = blockIdx.x;  // (sequence, node)
  const int s = static_cast<int>(x / a.max_q_len), i = static_cast<int>(x - static_cast<int64_t>(s) * a.max_q_len);
  const Seq p = seq_of(a, s);
  const int h = blockIdx.y, np = (keys_of(a, p) + pt.tokens - 1) / pt.tokens;
  if (i >= p.n || np < 2) return;
  const int64_t r = static_cast<int64_t>(p.q0) + i, slot = (x * pt.hq + h) * pt.parts;
  float m = -INFINITY;
  for (int k = 0; k < np; ++k) m = fmax2(m, pt.ml[2 * (slot + k)]);
  for (int d = threadIdx.x; d < dim; d += kWave) {
    float A = 0.0f, l = 0.0f;
#pragma unroll 4
    for (int k = 0; k < np; ++k) {
      const float mk = pt.ml[2 * (slot + k)], f = mk == -INFINITY ? 0.0f : fast_exp2(mk - m);
      A = fmaf(f, pt.acc[(slot + k) * dim + d], A);
      l = fmaf(f, pt.ml[2 * (slot + k) + 1], l);
    }
    reinterpret_cast<S*>(a.out)[r * a.out_st + static_cast<int64_t>(h) * a.out_sh + d] =
        from_f32<DT>(l == 0.0f ? 0.0f : A / l);
  }
}

// ------------------------------------------------------------------ host side

using KernelFn = void (*)(TreeArgs);
using MergeFn = void (*)(TreeArgs, int, int);
using KernelRowFn = void (*)(TreeArgs, PartArgs);

struct Config {
  KernelFn fn = nullptr;
  MergeFn merge = nullptr, merge_by_piece = nullptr;
  int rows = 0, keys = 0, occ = 0;  // R, KT, workgroups per CU
  int64_t rec_floats = 0;
};

template <int DT, int D, int WR, int WK, int NC, int OCC>
Config config_of() {
  using P = Shape<D, WR, WK, NC>;
  return {paged_tree_kernel<DT, D, WR, WK, NC, OCC>, paged_tree_merge<DT, D, P::R, false>,
          paged_tree_merge<DT, D, P::R, true>, P::R, P::KT, OCC, P::kRec};
}

// The workgroup's shape by the most rows a segment's kv head can have, and the products of the call (sequences x kv
// heads x rows x keys). Wavefronts with the same 16, 32 or 64 rows and keys of their own need no staging together and
// cut a segment finely; wavefronts with rows of their own that share keys read each key a quarter as often. The
// second takes blocks of 8 tokens or more and pays for more rows than 64 once the call is large (graph replay, us, own keys /
// shared, bf16, fp16 the same within 4 %; sequences x half of to all of the nodes, of 7 rows each, over half of to all of
// the keys; d64, 2 kv heads: 16 x 24 over 1024 keys 19.0/22.3, 64 x 48 over 256 21.8/27.7, 64 x 24 over 1024 (22M)
// 30.3/29.7, 64 x 32 over 1024 (29M) 34.6/32.1, 64 x 48 over 1024 40.7/38.0, 64 x 64 over 4096 111/95.4; d128, 4 kv
// heads: 4 x 24 over 4096 29.4/28.8, 1 x 16 over 32768 (15M) 33.2/30.6, 16 x 48 over 1024 (22M) 49.9/39.6, 16 x 64 over
// 4096 139/93.3). The keys are the table's width: a call of short contexts with a wide table is taken for a large one.
// d64 with shared keys: 32 rows a wavefront and three workgroups a CU against 64 and two, 64 x 64 over 512 35.5/38.9,
// 256 x 64 over 512 71.9/81.8, 64 x 64 over 4096 95.0/100.
template <int DT>
Config pick(int d, int64_t rows, int64_t products, int bs) {
  if (d == 64) {
    if (rows <= 16) return config_of<DT, 64, 1, 4, 1, 2>();
    if (rows <= 32) return config_of<DT, 64, 1, 4, 2, 2>();
    if (rows <= 64 || products <= 28 << 20 || bs < 8) return config_of<DT, 64, 1, 4, 4, 2>();
    return config_of<DT, 64, 4, 1, 2, 3>();
  }
  if (rows <= 16) return config_of<DT, 128, 1, 4, 1, 1>();
  if (rows <= 32) return config_of<DT, 128, 1, 4, 2, 1>();
  if (rows <= 64 || products <= 16 << 20 || bs < 8) return config_of<DT, 128, 1, 4, 4, 1>();
  return config_of<DT, 128, 4, 1, 2, 2>();
}

constexpr unsigned kMergeByPiece = 512;  // column blocks up to which pieces are combined by piece
constexpr int kMinShareKeys = 64;  // fewest keys a worker takes

int compute_units() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 256;
  return cus;
}

struct Plan {
  Config cfg;
  bool ok = false;      // the matrix-core kernel takes this shape
  int grid = 0, segs_per_seq = 0, min_share = 0, slack = 1;
  int64_t start_off = 0, bytes = 0;  // bytes 0: no segment can be split
};

Plan plan_of(int num_seqs, int max_q_len, int hq, int hkv, int d, int bs, int max_blocks, int dtype) {
  Plan p;
  const int group = hq / hkv;
  const int64_t rows = static_cast<int64_t>(max_q_len) * group, cap = static_cast<int64_t>(max_blocks) * bs;
  if ((dtype != MIP_F16 && dtype != MIP_BF16) || (d != 64 && d != 128)) return p;
  const int64_t products = static_cast<int64_t>(num_seqs) * hkv * rows * cap;
  p.cfg = dtype == MIP_F16 ? pick<MIP_F16>(d, rows, products, bs) : pick<MIP_BF16>(d, rows, products, bs);
  const int64_t segs = hkv * ((rows + p.cfg.rows - 1) / p.cfg.rows), steps = (cap + p.cfg.keys - 1) / p.cfg.keys;
  if ((rows + 256) * group >= (int64_t{1} << 31) || segs * steps >= (int64_t{1} << 30) || segs * num_seqs * steps >= (int64_t{1} << 30) ||
      segs * num_seqs >= (int64_t{1} << 24))
    return p;
  p.ok = true;
  p.segs_per_seq = static_cast<int>(segs);
  p.min_share = (kMinShareKeys + p.cfg.keys - 1) / p.cfg.keys;
  const int64_t most = (segs * num_seqs * steps + p.min_share - 1) / p.min_share, slots = compute_units() * p.cfg.occ;
  p.grid = static_cast<int>((most < slots ? most : slots) + 7) / 8 * 8;
  // Where there are enough segments for the chip, cuts keep away from their ends, and segments of up to 640 keys stay
  // whole, at which no second kernel is launched (graph replay, us, cut anywhere / 256 keys away / 384; sequences x
  // nodes over half of to all of the keys, 14q/2kv d64, 512 keys: 32 x 24 20.6/19.5/16.2, 64 x 12 21.3/19.6/16.8, 128 x 12
  // 28.2/23.4/18.3; 1024: 32 x 12 20.3/18.9/22.5, 32 x 24 24.9/22.1/25.3, 64 x 5 18.9/18.0/21.0, 64 x 24 30.9/29.9/28.4;
  // 2048: 32 x 12 25.3/22.7/23.6, 64 x 12 31.2/29.9/30.4; 28q/4kv d128, 512 keys, cut / 256 away / whole: 32 x 5
  // 22.9/20.1/16.6, 32 x 12 29.6/25.1/20.1; 1024: 8 x 12 22.5/20.3). Where there are few, they are cut anywhere (64
  // nodes over 250 keys 13.6, whole 18.8; 4 x 64 over 512 16.2/23.9).
  const int64_t all = segs * num_seqs;
  if (p.cfg.keys >= 128 ? 4 * all >= p.grid : all >= 2 * p.grid) p.slack = (cap <= 640 ? 384 : 256) / p.cfg.keys;
  if (steps >= 2 * p.slack) {  // else no cut stays inside a segment
    p.start_off = (static_cast<int64_t>(p.grid) * 2 * p.cfg.rec_floats * 4 + 255) / 256 * 256;
    p.bytes = p.start_off + (num_seqs + 1) * 4;
  }
  return p;
}

// Where the row kernel beats the matrix-core kernel in 16 bits: a workgroup for each (node, head) reads the keys
// again, so it wins while they are few and so are the rows (graph replay, us, row / matrix cores; sequences x nodes,
// 14q/2kv d64: 1 x 5 over 60 keys 4.4/7.2, 500 8.9/10.3, 1000 14.6/11.0; 1 x 64 120 6.9/13.0, 500 13.5/14.4;
// 32 x 5 16 6.4/8.0, 120 8.8/8.1; 8 x 24 60 9.1/13.9, 250 16.6/15.7; 28q/4kv d128: 1 x 5 250 8.6/12.5, 500 14.6/12.8;
// 8 x 5 120 9.0/9.8, 250 14.4/13.6; 32 x 5 16 13.7/9.9).
// In fp32 the tiles are the smaller ones and win earlier (1 x 5 over 60 keys 5.3/6.4, 8 x 7 over 16-256 9.0/8.5).
bool row_kernel_pays(int num_seqs, int max_q_len, int hq, int d, int64_t cap, int dtype) {
  const int64_t work = static_cast<int64_t>(num_seqs) * max_q_len * hq * cap * d;
  return dtype == MIP_F32 ? cap * d <= 8192 && work <= (int64_t{1} << 22) : cap * d <= 49152 && work <= (int64_t{1} << 24);
}

// Parts of the other kernels' calls, at least kPartTokens keys each, where their workgroups leave half of the chip idle
// (fp32, graph replay, us, whole / parts: 14 tiles of workgroups over 1000 keys 22.3/11.5, 2 over 2000 37.9/10.6, 32 over
// 500 14.1/11.0; parts of 224 over 500 16.1/20.9).
constexpr int kPartTokens = 256;
struct Parts {
  int tokens = 1, parts = 1;
  int64_t acc_off = 0, bytes = 0;  // bytes 0: one part
};

Parts parts_of(int num_seqs, int max_q_len, int hq, int hkv, int d, int64_t cap, bool tiles) {
  Parts p;
  const int64_t rows = static_cast<int64_t>(num_seqs) * max_q_len, per_kv = static_cast<int64_t>(max_q_len) * (hq / hkv);
  const int64_t groups = tiles ? (per_kv + 15) / 16 * hkv * num_seqs : rows * hq;
  const int64_t want = groups < 256 ? 256 / groups : 1, most = (cap + kPartTokens - 1) / kPartTokens;
  const int64_t parts = want < most ? want : most;
  p.tokens = static_cast<int>(((cap + parts - 1) / parts + 63) / 64 * 64);
  p.parts = static_cast<int>((cap + p.tokens - 1) / p.tokens);
  if (p.parts > 1) {
    p.acc_off = (rows * hq * p.parts * 8 + 255) / 256 * 256;
    p.bytes = p.acc_off + rows * hq * p.parts * d * 4;
  }
  return p;
}

// fp32 on the matrix cores: head_dim 64 / 128, where its grid and its 32-bit pool rows suffice.
bool f32_fits(int dtype, int d, int num_seqs, int64_t rows, int64_t pool_rows) {
  return dtype == MIP_F32 && (d == 64 || d == 128) && (rows + 15) / 16 * num_seqs < (int64_t{1} << 24) &&
         pool_rows < (int64_t{1} << 31);
}

template <int DT>
KernelRowFn row_kernel(int d) {
  switch (d) {
    case 8:   return paged_tree_row_kernel<DT, 8>;
    case 16:  return paged_tree_row_kernel<DT, 16>;
    case 32:  return paged_tree_row_kernel<DT, 32>;
    case 64:  return paged_tree_row_kernel<DT, 64>;
    case 128: return paged_tree_row_kernel<DT, 128>;
    case 256: return paged_tree_row_kernel<DT, 256>;
    default:  return nullptr;
  }
}

}  // namespace
}  // namespace tree
}  // namespace mip

using namespace mip;

extern "C" size_t mip_paged_tree_workspace(int32_t num_seqs, int32_t max_q_len, int32_t num_heads, int32_t num_kv_heads,
                                           int32_t head_dim, int32_t block_size, int32_t max_blocks_per_seq,
                                           int32_t dtype) {
  if (num_seqs <= 0 || max_q_len <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads ||
      head_dim <= 0 || block_size <= 0 || max_blocks_per_seq <= 0 ||
      static_cast<int64_t>(max_blocks_per_seq) * block_size >= (int64_t{1} << 30))
    return 0;
  if (num_seqs > tree::kMaxSeqs) {  // several launches, one after the other
    const size_t full = mip_paged_tree_workspace(tree::kMaxSeqs, max_q_len, num_heads, num_kv_heads, head_dim, block_size,
                                                 max_blocks_per_seq, dtype);
    const size_t rest = mip_paged_tree_workspace(num_seqs % tree::kMaxSeqs, max_q_len, num_heads, num_kv_heads, head_dim,
                                                 block_size, max_blocks_per_seq, dtype);
    return full > rest ? full : rest;
  }
  const int64_t cap = static_cast<int64_t>(max_blocks_per_seq) * block_size;
  // The larger of what the kernels need that may take the call (its alignment is not known here).
  const int64_t main =
      tree::plan_of(num_seqs, max_q_len, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, dtype).bytes;
  int64_t need = main;
  for (const bool tiles : {false, dtype == MIP_F32}) {
    const int64_t rest = tree::parts_of(num_seqs, max_q_len, num_heads, num_kv_heads, head_dim, cap, tiles).bytes;
    need = rest > need ? rest : need;
  }
  return static_cast<size_t>(need);
}

extern "C" int mip_paged_tree(void* out, int64_t out_stride_tok, int64_t out_stride_head, const void* q,
                              int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache, const void* v_cache,
                              int64_t num_cache_blocks, const int32_t* block_tables, int64_t bt_stride,
                              const int32_t* cu_q, const int32_t* ctx_start, const uint64_t* mask, int64_t mask_stride,
                              int32_t mask_words, int32_t num_seqs, int32_t max_q_len, int32_t num_heads,
                              int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t max_blocks_per_seq,
                              float scale, void* workspace, size_t workspace_bytes, int32_t dtype, void* stream) {
  if (dtype != MIP_F32 && dtype != MIP_F16 && dtype != MIP_BF16) return MIP_EINVAL;
  if (num_seqs < 0 || max_q_len < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads) return MIP_EINVAL;
  if (head_dim <= 0 || num_cache_blocks <= 0 || max_blocks_per_seq <= 0 || bt_stride < max_blocks_per_seq) return MIP_EINVAL;
  if (!is_pow2(block_size) || block_size > 4096 || num_cache_blocks > INT32_MAX || !(scale > 0.0f && scale <= 0x1p127f))
    return MIP_EINVAL;
  if (num_seqs == 0 || max_q_len == 0) return MIP_OK;
  if (!out || !q || !k_cache || !v_cache || !block_tables || !cu_q || !ctx_start || !mask) return MIP_EINVAL;
  if (mask_words < (max_q_len + 63) / 64 || mask_stride < mask_words) return MIP_EINVAL;
  const int64_t cap = static_cast<int64_t>(max_blocks_per_seq) * block_size;
  if (cap >= (int64_t{1} << 30) || static_cast<int64_t>(num_kv_heads) * block_size >= (int64_t{1} << 31)) return MIP_EINVAL;
  const int64_t es = dtype == MIP_F32 ? 4 : 2;
  const uint64_t q_bits = reinterpret_cast<uintptr_t>(q) | static_cast<uint64_t>(q_stride_tok * es) |
                          static_cast<uint64_t>(q_stride_head * es);
  const uint64_t out_bits = reinterpret_cast<uintptr_t>(out) | static_cast<uint64_t>(out_stride_tok * es) |
                            static_cast<uint64_t>(out_stride_head * es);
  if (((q_bits | out_bits) & (es - 1)) || ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15))
    return MIP_EINVAL;
  if (num_seqs > tree::kMaxSeqs) {
    const size_t need = mip_paged_tree_workspace(num_seqs, max_q_len, num_heads, num_kv_heads, head_dim, block_size,
                                                 max_blocks_per_seq, dtype);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
      return MIP_EINVAL;
    for (int32_t s0 = 0; s0 < num_seqs; s0 += tree::kMaxSeqs) {
      const int32_t some = num_seqs - s0 < tree::kMaxSeqs ? num_seqs - s0 : tree::kMaxSeqs;
      const int rc = mip_paged_tree(out, out_stride_tok, out_stride_head, q, q_stride_tok, q_stride_head, k_cache, v_cache,
                                    num_cache_blocks, block_tables + s0 * bt_stride, bt_stride, cu_q + s0, ctx_start + s0,
                                    mask, mask_stride, mask_words, some, max_q_len, num_heads, num_kv_heads, head_dim,
                                    block_size, max_blocks_per_seq, scale, workspace, workspace_bytes, dtype, stream);
      if (rc != MIP_OK) return rc;
    }
    return MIP_OK;
  }

  tree::TreeArgs a{};
  a.out = static_cast<char*>(out);
  a.out_st = out_stride_tok;
  a.out_sh = out_stride_head;
  a.q = static_cast<const char*>(q);
  a.q_st = q_stride_tok;
  a.q_sh = q_stride_head;
  a.k = static_cast<const char*>(k_cache);
  a.v = static_cast<const char*>(v_cache);
  a.ncb = num_cache_blocks;
  a.bt = block_tables;
  a.bt_stride = bt_stride;
  a.cu_q = cu_q;
  a.ctx_start = ctx_start;
  a.mask = mask;
  a.mask_st = mask_stride;
  a.mask_words = mask_words;
  a.hkv = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.group_inv = a.group > 1 ? static_cast<uint32_t>(((uint64_t{1} << 32) + a.group - 1) / a.group) : 0;
  a.bs = block_size;
  a.log2_bs = ilog2_exact(block_size);
  a.max_blocks = max_blocks_per_seq;
  a.num_seqs = num_seqs;
  a.max_q_len = max_q_len;
  a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = static_cast<hipStream_t>(stream);

  // q rows are read 16 bytes and output rows written 8 bytes at a time by the matrix-core kernel.
  const tree::Plan p = (q_bits & 15) || (out_bits & 7)
                           ? tree::Plan{}
                           : tree::plan_of(num_seqs, max_q_len, num_heads, num_kv_heads, head_dim, block_size,
                                           max_blocks_per_seq, dtype);
  if (p.ok && !tree::row_kernel_pays(num_seqs, max_q_len, num_heads, head_dim, cap, dtype)) {
    if (p.bytes > 0) {
      if (!workspace || workspace_bytes < static_cast<size_t>(p.bytes) || (reinterpret_cast<uintptr_t>(workspace) & 255))
        return MIP_EINVAL;
      a.ws_rec = static_cast<float*>(workspace);
      a.ws_start = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + p.start_off);
    }
    a.min_share = p.min_share;
    a.slack = p.slack;
    hipLaunchKernelGGL(p.cfg.fn, dim3(p.grid), dim3(256), 0, s, a);
    if (p.bytes > 0) {
      const unsigned segs = static_cast<unsigned>(p.segs_per_seq * num_seqs), blocks = p.cfg.rows / 16;
      // Few workgroups by column block: each segment has many pieces.
      if (segs * blocks <= tree::kMergeByPiece)
        hipLaunchKernelGGL(p.cfg.merge_by_piece, dim3(segs, blocks, head_dim / 32), dim3(256), 0, s, a, p.segs_per_seq,
                           p.cfg.keys);
      else
        hipLaunchKernelGGL(p.cfg.merge, dim3(segs, (blocks + 3) / 4), dim3(256), 0, s, a, p.segs_per_seq, p.cfg.keys);
    }
    return status_from_hip(hipGetLastError());
  }
  const int64_t rows = static_cast<int64_t>(num_seqs) * max_q_len;
  if (rows >= (int64_t{1} << 24) || num_heads > 65535) return MIP_EUNSUPPORTED;
  const bool tiles = tree::f32_fits(dtype, head_dim, num_seqs, static_cast<int64_t>(max_q_len) * a.group,
                                    num_cache_blocks * num_kv_heads * block_size) &&
                     !tree::row_kernel_pays(num_seqs, max_q_len, num_heads, head_dim, cap, dtype);
  const tree::KernelRowFn fn = dtype == MIP_F32   ? tree::row_kernel<MIP_F32>(head_dim)
                               : dtype == MIP_F16 ? tree::row_kernel<MIP_F16>(head_dim)
                                                  : tree::row_kernel<MIP_BF16>(head_dim);
  if (!fn) return MIP_EUNSUPPORTED;
  const tree::Parts parts = tree::parts_of(num_seqs, max_q_len, num_heads, num_kv_heads, head_dim, cap, tiles);
  tree::PartArgs pt{num_heads, parts.tokens, parts.parts, nullptr, nullptr};
  if (parts.bytes > 0) {
    if (!workspace || workspace_bytes < static_cast<size_t>(parts.bytes) || (reinterpret_cast<uintptr_t>(workspace) & 255))
      return MIP_EINVAL;
    pt.ml = static_cast<float*>(workspace);
    pt.acc = reinterpret_cast<float*>(static_cast<char*>(workspace) + parts.acc_off);
  }
  if (tiles) {
    decode::DecodeArgs da{};
    da.out = a.out;
    da.out_sb = out_stride_tok;
    da.out_sh = out_stride_head;
    da.q = a.q;
    da.q_sb = q_stride_tok;
    da.q_sh = q_stride_head;
    da.k = a.k;
    da.v = a.v;
    da.ncb = num_cache_blocks;
    da.bt = block_tables;
    da.bt_stride = bt_stride;
    da.hq = num_heads;
    da.hkv = num_kv_heads;
    da.bs = block_size;
    da.log2_bs = a.log2_bs;
    da.max_blocks = max_blocks_per_seq;
    da.group = a.group;
    da.part_tokens = parts.tokens;
    da.nparts = parts.parts;
    da.scale_log2 = a.scale_log2;
    da.ws_ml = pt.ml;
    da.ws_acc = pt.acc;
    da.cu_q = cu_q;
    da.ctx_start = ctx_start;
    da.max_q_len = max_q_len;
    const int st = decode::f32_tree_launch(da, decode::TreeMask{mask, mask_stride, mask_words}, num_seqs, head_dim, s);
    if (st) return st;
  } else {
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(rows), num_heads, parts.parts), dim3(256), 0, s, a, pt);
  }
  if (parts.parts > 1) {
    const dim3 grid(static_cast<unsigned>(rows), num_heads);
    switch (dtype) {
      case MIP_F32: hipLaunchKernelGGL(tree::paged_tree_parts_kernel<MIP_F32>, grid, dim3(kWave), 0, s, a, pt, head_dim); break;
      case MIP_F16: hipLaunchKernelGGL(tree::paged_tree_parts_kernel<MIP_F16>, grid, dim3(kWave), 0, s, a, pt, head_dim); break;
      default:      hipLaunchKernelGGL(tree::paged_tree_parts_kernel<MIP_BF16>, grid, dim3(kWave), 0, s, a, pt, head_dim);
    }
  }
  return status_from_hip(hipGetLastError());
}
