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
// keys. Segments of very different lengths share the chip, and one long sequence has to fill it, so
// segments of more than L steps are cut into pieces of at most L (about as many steps as a workgroup's
// equal share); a piece leaves its rows' maxima, sums and unnormalised outputs in the workspace and a
// second kernel combines them. L and each piece's place follow from cu_q and ctx_start on the device:
// the grid depends on the integer arguments alone.
//
// A workgroup is WR x WK wavefronts: WR take different rows (NC blocks of 16 each) of the same keys, WK
// take different 32 keys of a step for the same rows and meet at the piece's end. Few rows use WK = 4 (no
// wavefront idles), many WR = 4 (each key staged once serves 256 rows). All threads copy the step's K and
// V rows into LDS (two stages; the next step's rows travel in registers meanwhile); a wavefront then
// computes
//   S^T[16 keys x 16 rows] = K . Q^T     v_mfma_f32_16x16x32, Q^T in registers
//   O^T[D x 16 rows]      += V^T . P^T   v_mfma_f32_16x16x32 over 32 keys
// with a base-2 online softmax. V^T comes from transposing LDS reads; P is in the layout of S^T.
//
// Roundings. Scores, sums and accumulators are fp32. The weights enter the V product as fp16 (2^-11
// relative; the sums are taken of the rounded weights, so the error of a lone key cancels), bf16 V is
// staged as fp16 (exact below 65536). A piece whose accumulators end up inf or NaN runs again with V
// as it is, weights in two parts (their sum holds them to 2^-16 and better), and every inf or NaN of V
// applied to the rows that see its key alone: a masked key must not reach a row as 0 * inf.
#include "paged_decode_common.h"

namespace mip {
namespace tree {
namespace {

using decode::f32x4_t;
using decode::fast_exp2;
using decode::kRescaleLog2;
using decode::MfmaOps;

constexpr int kMaxSeqs = 1024;  // sequences whose places fit in LDS

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
  int num_seqs, max_q_len;
  float scale_log2;
  // Split segments: record g (m[R] | l[R] | acc) at ws_rec + g * rec_floats, its segment's descriptor
  // at ws_desc + g * kDesc, written by the segment's first piece and invalid (pieces 0) elsewhere.
  float* ws_rec;
  int32_t* ws_desc;
  int64_t rec_floats;
  int target, min_steps, max_recs;
};

constexpr int kDesc = 4;  // words: pieces, sequence, kv head, row block

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

// Eight bf16 values -> fp16: exact from 2^-17 to 65280 in magnitude, inf from 65536 on; smaller ones land
// on fp16's subnormal grid (a change of at most 2^-25).
__device__ __forceinline__ uint4 bf16x8_to_f16x8(const uint4& v) {
  auto cv = [](uint32_t x) __attribute__((always_inline)) {
    return MfmaOps<MIP_F16>::pack2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  };
  return make_uint4(cv(v.x), cv(v.y), cv(v.z), cv(v.w));
}

// A pair of 16-bit values with inf and NaN replaced by 0; `wild` is set if there was one.
template <int DT> __device__ __forceinline__ uint32_t finite2(uint32_t x, bool& wild) {
  constexpr uint32_t kExp = DT == MIP_BF16 ? 0x7f80u : 0x7c00u;
  if ((x & kExp) == kExp) {
    x &= 0xffff0000u;
    wild = true;
  }
  if (((x >> 16) & kExp) == kExp) {
    x &= 0xffffu;
    wild = true;
  }
  return x;
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
  static constexpr int STAGE = 2 * TILE;
  static constexpr int NLD = KT * CPR / T;         // chunks a thread copies, each of K and V
  static constexpr int64_t kRec = 2 * R + static_cast<int64_t>(R) * D;  // floats of a record
  static_assert(NLD >= 1 && NLD * T == KT * CPR, "a step splits evenly over the threads");
  // The meeting of the WK wavefronts of a row reuses the stages.
  static_assert(WK == 1 || WR * (WK - 1) * NC * MT * kWave * 16 <= 2 * STAGE, "accumulators must fit");
  // V row r keeps chunk c at c ^ vsw(r): even, so that each 32-byte segment of a transposing read stays
  // whole, and the 8 rows that 32 lanes read start in distinct banks.
  static __device__ __forceinline__ int vsw(int r) { return CPR >= 16 ? 2 * (r & 7) : 2 * ((r + (r >> 2)) & 3); }
};

struct Piece {
  int s, kvh, rb, q0, n, ctx, keys, step0, step1;
};

// What a workgroup shares beside the stages.
template <int T, int NW, int ML>
struct Shared {
  int scan[2][NW];
  int pieces[kMaxSeqs + 1], recs[kMaxSeqs + 1];  // exclusive prefixes over the sequences
  uint32_t ok[2];      // byte w: every key that wavefront w copied lies in a block of the pool
  uint32_t wild[2];    // careful pass: byte w: wavefront w copied an inf or NaN value
  uint32_t tag;        // of the piece that has to run again
  float ml[2][ML];     // maxima and sums of the WK - 1 other wavefronts of each row
};

__device__ __forceinline__ Piece seq_shape(const TreeArgs& a, int s, int cap) {
  Piece p;
  p.s = s;
  p.q0 = a.cu_q[s];
  p.n = a.cu_q[s + 1] - p.q0;
  p.n = p.n < a.max_q_len ? p.n : a.max_q_len;
  p.n = p.n > 0 ? p.n : 0;
  p.ctx = a.ctx_start[s];
  p.ctx = p.ctx > 0 ? p.ctx : 0;
  p.keys = p.ctx < cap - p.n ? p.ctx + p.n : cap;  // keys past the table are never read
  return p;
}

// One piece: rows of block p.rb against steps [p.step0, p.step1). Returns true (and writes nothing) if it has
// to run again with CAREFUL. rec < 0: the piece is its whole segment and writes the output.
template <int DT, int D, int WR, int WK, int NC, bool CAREFUL, class Sh>
__device__ __forceinline__ bool run_piece(const TreeArgs& a, const Piece& p, int64_t rec, uint32_t tag, char* smem,
                                          Sh& sh) {
  using P = Shape<D, WR, WK, NC>;
  constexpr bool VF16 = DT == MIP_BF16 && !CAREFUL;
  using Ops = MfmaOps<DT>;
  using OpsV = MfmaOps<VF16 ? MIP_F16 : DT>;
  constexpr int RB = P::RB, CPR = P::CPR, KC = P::KC, MT = P::MT, NLD = P::NLD;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wr = w / WK, wk = w - wr * WK;
  const int i16 = lane & 15, grp = lane >> 4;
  const int G = a.group, last = p.keys - 1;
  const int32_t* table = a.bt + static_cast<int64_t>(p.s) * a.bt_stride;

  // ---- this lane's query row in each column block.
  bool live[NC];
  int tok[NC];
  uint4 qreg[NC][KC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int r = p.rb * P::R + (wr * NC + c) * 16 + i16;
    const int t = r / G, g = r - t * G;
    live[c] = t < p.n;
    tok[c] = live[c] ? t : 0;
    const char* qrow = a.q + ((static_cast<int64_t>(p.q0) + tok[c]) * a.q_st +
                              static_cast<int64_t>(p.kvh * G + (live[c] ? g : 0)) * a.q_sh) * 2;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc)
      qreg[c][kc] = live[c] ? *reinterpret_cast<const uint4*>(qrow + (32 * kc + 8 * grp) * 2) : make_uint4(0, 0, 0, 0);
  }

  // ---- loader: block ids one step ahead of the rows, rows one step ahead of their use.
  uint4 kbuf[NLD], vbuf[NLD];
  bool okbuf[NLD];
  int bid[NLD];
  auto lookup = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NLD; ++j) {
      const int key = t * P::KT + (tid + j * P::T) / CPR;
      bid[j] = table[(key < last ? key : last) >> a.log2_bs];
    }
  };
  auto fetch = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NLD; ++j) {
      const int idx = tid + j * P::T;
      const int r = idx / CPR, c = idx % CPR;
      const int key = t * P::KT + r;
      const int kk = key < last ? key : last;  // keys past the last one stand for it
      const bool bok = bid[j] >= 0 && bid[j] < a.ncb;
      const uint64_t row = static_cast<uint64_t>(bok ? static_cast<uint32_t>(bid[j]) : 0u) *
                               static_cast<uint32_t>(a.hkv * a.bs) +
                           static_cast<uint32_t>(p.kvh * a.bs + (kk & (a.bs - 1)));
      kbuf[j] = *reinterpret_cast<const uint4*>(a.k + row * RB + c * 16);
      vbuf[j] = *reinterpret_cast<const uint4*>(a.v + row * RB + c * 16);
      okbuf[j] = bok;
    }
  };
  auto stash = [&](int stage) __attribute__((always_inline)) {
    char* st = smem + stage * P::STAGE;
    bool ok = true, wild = false;
#pragma unroll
    for (int j = 0; j < NLD; ++j) {
      const int idx = tid + j * P::T;
      const int r = idx / CPR, c = idx % CPR;
      uint4 vv = vbuf[j];
      if constexpr (VF16) vv = bf16x8_to_f16x8(vv);
      if constexpr (CAREFUL)
        vv = make_uint4(finite2<DT>(vv.x, wild), finite2<DT>(vv.y, wild), finite2<DT>(vv.z, wild), finite2<DT>(vv.w, wild));
      *reinterpret_cast<uint4*>(st + r * RB + ((c ^ (r & (CPR - 1))) * 16)) = kbuf[j];
      *reinterpret_cast<uint4*>(st + P::TILE + r * RB + ((c ^ P::vsw(r)) * 16)) = vv;
      ok = ok && okbuf[j];
    }
    ok = __all(ok);
    if (lane == 0) reinterpret_cast<uint8_t*>(&sh.ok[stage])[w] = ok ? 1 : 0;
    if constexpr (CAREFUL) {
      wild = __any(wild);
      if (lane == 0) reinterpret_cast<uint8_t*>(&sh.wild[stage])[w] = wild ? 1 : 0;
    }
  };
  constexpr uint32_t kAllOk = P::NW == 4 ? 0x01010101u : P::NW == 2 ? 0x0101u : 0x01u;
  static_assert(P::NW == 4 || P::NW == 2 || P::NW == 1, "one byte per wavefront");

  f32x4_t acc[NC][MT];
  f32x4_t lacc[NC];  // row sums by MFMA against a block of ones: every element holds row i16's
  float m[NC], mth[NC], nm[NC];  // running maximum, the raw score that raises it, -m (0 while m = -inf)
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m[c] = -INFINITY;
    mth[c] = -INFINITY;
    nm[c] = 0.0f;
    lacc[c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[c][mt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

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
      uint4 kreg[2][KC];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          const int r = 16 * u + i16, ch = 4 * kc + grp;
          kreg[u][kc] = *reinterpret_cast<const uint4*>(st + r * RB + ((ch ^ (r & (CPR - 1))) * 16));
        }
      }
      // The PV product's k index 8 grp + i stands for key 4 grp + i (i < 4) or 16 + 4 grp + i - 4: the keys
      // of this lane's two S^T halves.
      uint4 vt[MT];
      const int vrow = 4 * grp + (i16 >> 2), vs = P::vsw(vrow);  // rows vrow and vrow + 16 share vsw
      const char* vb = st + P::TILE + vrow * RB + (i16 & 3) * 8;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int so = ((2 * mt) ^ vs) * 16;
        const uint2 lo = lds_tr16(vb + so);
        const uint2 hi = lds_tr16(vb + 16 * RB + so);
        vt[mt] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
      constexpr int kr[8] = {0, 1, 2, 3, 16, 17, 18, 19};  // this lane's keys: 4 grp + kr[i]
      float sv[NC][8];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        f32x4_t s0 = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          s0 = Ops::qk(kreg[0][kc], qreg[c][kc], s0);
          s1 = Ops::qk(kreg[1][kc], qreg[c][kc], s1);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sv[c][i] = i < 4 ? s0[i] : s1[i - 4];
      }
      const bool allok = __builtin_amdgcn_readfirstlane(sh.ok[stage]) == kAllOk;
      uint32_t win[NC];  // bit k: this lane's row sees key key0 + k
      const bool open = allok && key0 + 31 < p.ctx && key0 + 31 <= last;  // cached keys only: everybody sees them
      if (!open) {
        const int e0 = key0 - p.ctx;  // tree number of the first key (below 0: cached)
        uint32_t real = last - key0 >= 31 ? 0xffffffffu : (2u << (last - key0)) - 1u;
        if (!allok) {  // blocks outside the pool: the tile's keys one by one
          const int key = key0 + (lane & 31);
          const int b = table[(key < last ? key : last) >> a.log2_bs];
          real &= static_cast<uint32_t>(__ballot(b >= 0 && b < a.ncb));
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          uint32_t see = 0xffffffffu;
          if (e0 > -32) {
            const uint64_t* row = a.mask + (static_cast<int64_t>(p.q0) + tok[c]) * a.mask_st;
            if (e0 < 0) {
              see = static_cast<uint32_t>(row[0] << -e0) | ((1u << -e0) - 1u);
            } else {
              const int word = e0 >> 6, off = e0 & 63;
              uint64_t x = word < a.mask_words ? row[word] >> off : 0;
              if (off > 32 && word + 1 < a.mask_words) x |= row[word + 1] << (64 - off);
              see = static_cast<uint32_t>(x);
            }
          }
          win[c] = live[c] ? see & real : 0u;
          const uint32_t mine = win[c] >> (4 * grp);
#pragma unroll
          for (int i = 0; i < 8; ++i) sv[c][i] = (mine >> kr[i]) & 1u ? sv[c][i] : -INFINITY;
        }
      } else {
#pragma unroll
        for (int c = 0; c < NC; ++c) win[c] = 0xffffffffu;
      }
      float mx[NC];
      bool need = false;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        mx[c] = fmax3(fmax3(sv[c][0], sv[c][1], sv[c][2]), fmax3(sv[c][3], sv[c][4], sv[c][5]),
                      fmax2(sv[c][6], sv[c][7]));
        need = need || mx[c] > mth[c];
      }
      if (__any(need)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (__any(mx[c] > mth[c])) {
            const float mn = fmax2(m[c], max4(mx[c]) * a.scale_log2);
            const float alpha = (m[c] == -INFINITY) ? 0.0f : fast_exp2(m[c] - mn);
            lacc[c] *= alpha;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[c][mt] *= alpha;
            m[c] = mn;
            mth[c] = (mn + kRescaleLog2) / a.scale_log2;
            nm[c] = mn == -INFINITY ? 0.0f : -mn;
          }
        }
      }
      const bool wild = CAREFUL && __builtin_amdgcn_readfirstlane(sh.wild[stage]) != 0;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float pr[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pr[i] = fast_exp2(fmaf(sv[c][i], a.scale_log2, nm[c]));
        uint4 ph;
        ph.x = OpsV::pack2(pr[0], pr[1]);
        ph.y = OpsV::pack2(pr[2], pr[3]);
        ph.z = OpsV::pack2(pr[4], pr[5]);
        ph.w = OpsV::pack2(pr[6], pr[7]);
        constexpr uint32_t kOne2 = DT == MIP_BF16 && !VF16 ? 0x3f803f80u : 0x3c003c00u;
        const uint4 ones = make_uint4(kOne2, kOne2, kOne2, kOne2);
        lacc[c] = OpsV::qk(ones, ph, lacc[c]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[c][mt] = OpsV::qk(vt[mt], ph, acc[c][mt]);
        if constexpr (CAREFUL) {
          uint4 pl;
          pl.x = Ops::pack2(pr[0] - Ops::lo(ph.x), pr[1] - Ops::hi(ph.x));
          pl.y = Ops::pack2(pr[2] - Ops::lo(ph.y), pr[3] - Ops::hi(ph.y));
          pl.z = Ops::pack2(pr[4] - Ops::lo(ph.z), pr[5] - Ops::hi(ph.z));
          pl.w = Ops::pack2(pr[6] - Ops::lo(ph.w), pr[7] - Ops::hi(ph.w));
          lacc[c] = Ops::qk(ones, pl, lacc[c]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) acc[c][mt] = Ops::qk(vt[mt], pl, acc[c][mt]);
          if (wild) {
            // Values that are inf or NaN were staged as 0: each joins the rows that see its key.
#pragma unroll 1
            for (int kk = 0; kk < 32 && key0 + kk <= last; ++kk) {
              const int e = (kk & 3) + (kk >= 16 ? 4 : 0);
              float pk = pr[0];
#pragma unroll
              for (int i = 1; i < 8; ++i) pk = e == i ? pr[i] : pk;
              pk = __shfl(pk, ((kk & 15) >> 2) * 16 + i16);
              const int b = table[(key0 + kk) >> a.log2_bs];
              if (b < 0 || b >= a.ncb) continue;
              const uint64_t row = static_cast<uint64_t>(b) * static_cast<uint32_t>(a.hkv * a.bs) +
                                   static_cast<uint32_t>(p.kvh * a.bs + ((key0 + kk) & (a.bs - 1)));
              const uint16_t* vr = reinterpret_cast<const uint16_t*>(a.v + row * RB);
              const bool seen = (win[c] >> kk) & 1u;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float x = widen<DT>(vr[16 * mt + 4 * grp + i]);
                  if (seen && !(fabsf(x) < INFINITY)) acc[c][mt][i] += pk * x;
                }
            }
          }
        }
      }
    }
    if (t + 1 < p.step1) stash(stage ^ 1);
    __syncthreads();
  }

  // ---- a fast pass that met inf or NaN runs again. Every thread reads the flag before any writes it again.
  if constexpr (!CAREFUL) {
    float big = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        big = fmax3(big, fmax2(fabsf(acc[c][mt][0]), fabsf(acc[c][mt][1])),
                    fmax2(fabsf(acc[c][mt][2]), fabsf(acc[c][mt][3])));
    if (__any(!(big < INFINITY)) && lane == 0) sh.tag = tag;
    __syncthreads();
    const bool again = __builtin_amdgcn_readfirstlane(sh.tag) == tag;
    __syncthreads();
    if (again) return true;
  }

  // ---- the wavefronts of one row block meet: wavefront wk = 0 takes the others' sums.
  if constexpr (WK > 1) {
    f32x4_t* park = reinterpret_cast<f32x4_t*>(smem);
    if (wk > 0) {
      const int at = wr * (WK - 1) + wk - 1;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) park[((at * NC + c) * MT + mt) * kWave + lane] = acc[c][mt];
        if (grp == 0) {
          sh.ml[0][(at * NC + c) * 16 + i16] = m[c];
          sh.ml[1][(at * NC + c) * 16 + i16] = lacc[c][0];
        }
      }
    }
    __syncthreads();
    if (wk == 0) {
#pragma unroll
      for (int o = 0; o < WK - 1; ++o) {
        const int at = wr * (WK - 1) + o;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float mo = sh.ml[0][(at * NC + c) * 16 + i16], lo = sh.ml[1][(at * NC + c) * 16 + i16];
          const float mn = fmax2(m[c], mo);
          // A part without keys has sums of 0 (its maximum is -inf, and so may both be).
          const float fa = m[c] == -INFINITY ? 0.0f : fast_exp2(m[c] - mn);
          const float fb = mo == -INFINITY ? 0.0f : fast_exp2(mo - mn);
          m[c] = mn;
          lacc[c][0] = lacc[c][0] * fa + lo * fb;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const f32x4_t x = park[((at * NC + c) * MT + mt) * kWave + lane];
            acc[c][mt] = acc[c][mt] * fa + x * fb;
          }
        }
      }
    }
  }

  if (wk == 0) {
    if (rec >= 0) {
      // Record: accumulators as the lanes hold them, [column block][mt][lane].
      float* base = a.ws_rec + rec * a.rec_floats;
      f32x4_t* racc = reinterpret_cast<f32x4_t*>(base + 2 * P::R);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int cb = wr * NC + c;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) racc[(cb * MT + mt) * kWave + lane] = acc[c][mt];
        if (grp == 0) {
          base[cb * 16 + i16] = m[c];
          base[P::R + cb * 16 + i16] = lacc[c][0];
        }
      }
    } else {
      using S = typename Elem<DT>::S;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (!live[c]) continue;
        const float lt = lacc[c][0];
        const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;  // 0: no key seen, sums of 0
        const int r = p.rb * P::R + (wr * NC + c) * 16 + i16;
        S* orow = reinterpret_cast<S*>(a.out) + (static_cast<int64_t>(p.q0) + tok[c]) * a.out_st +
                  static_cast<int64_t>(p.kvh * G + r - tok[c] * G) * a.out_sh;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint32_t w0 = Ops::pack2(acc[c][mt][0] * inv, acc[c][mt][1] * inv);
          const uint32_t w1 = Ops::pack2(acc[c][mt][2] * inv, acc[c][mt][3] * inv);
          *reinterpret_cast<uint2*>(orow + 16 * mt + 4 * grp) = make_uint2(w0, w1);
        }
      }
    }
  }
  if constexpr (WK > 1) __syncthreads();  // the next piece stages over the parked sums
  return false;
}

template <int DT, int D, int WR, int WK, int NC>
__global__ __launch_bounds__(WR * WK * kWave) __attribute__((amdgpu_waves_per_eu(WR * WK / 2, WR * WK / 2)))
void paged_tree_kernel(TreeArgs a) {
  using P = Shape<D, WR, WK, NC>;
  constexpr int T = P::T, NW = P::NW, ML = WK > 1 ? WR * (WK - 1) * NC * 16 : 1;
  __shared__ __attribute__((aligned(16))) char smem[2 * P::STAGE];
  __shared__ Shared<T, NW, ML> sh;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = tid / kWave;
  const int S = a.num_seqs, cap = a.max_blocks * a.bs;

  // ---- steps of all segments, then the piece length L, then every sequence's first piece and record.
  auto segments = [&](const Piece& p) { return (p.n * a.group + P::R - 1) / P::R * a.hkv; };
  auto steps = [&](const Piece& p) { return (p.keys + P::KT - 1) / P::KT; };
  int sum = 0;
  for (int s = tid; s < S; s += T) {
    const Piece p = seq_shape(a, s, cap);
    sum += segments(p) * steps(p);
  }
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) sh.scan[0][w] = sum;
  if (tid == 0) {
    sh.tag = 0;
    sh.ok[0] = sh.ok[1] = sh.wild[0] = sh.wild[1] = 0;
  }
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) total += sh.scan[0][i];
  __syncthreads();
  int L = (total + a.target - 1) / a.target;
  L = L > a.min_steps ? L : a.min_steps;
  int base_p = 0, base_r = 0;
  for (int s0 = 0; s0 < S; s0 += T) {
    const int s = s0 + tid;
    int np = 0, nr = 0;
    if (s < S) {
      const Piece p = seq_shape(a, s, cap);
      const int cuts = (steps(p) + L - 1) / L, segs = segments(p);
      np = segs * cuts;
      nr = cuts > 1 ? np : 0;
    }
    const int ip = decode::wave_inclusive_scan(np, lane), ir = decode::wave_inclusive_scan(nr, lane);
    if (lane == kWave - 1) {
      sh.scan[0][w] = ip;
      sh.scan[1][w] = ir;
    }
    __syncthreads();
    int before_p = base_p, before_r = base_r;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if (i < w) {
        before_p += sh.scan[0][i];
        before_r += sh.scan[1][i];
      }
      base_p += sh.scan[0][i];
      base_r += sh.scan[1][i];
    }
    if (s < S) {
      sh.pieces[s] = before_p + ip - np;
      sh.recs[s] = before_r + ir - nr;
    }
    __syncthreads();
  }
  // Descriptors of records that no piece of this call has.
  if (blockIdx.x == 0)
    for (int i = base_r + tid; i < a.max_recs; i += T) a.ws_desc[i * kDesc] = 0;

  // ---- pieces, each XCD a contiguous range of them (row blocks of the same keys are neighbours and meet in
  // its L2).
  const int per_xcd = (base_p + 7) / 8, xcd = blockIdx.x & 7;
  const int stride = static_cast<int>(gridDim.x) / 8;
  for (int i = blockIdx.x >> 3; i < per_xcd; i += stride) {
    const int it = xcd * per_xcd + i;
    if (it >= base_p) break;
    int lo = 0, hi = S - 1;  // the last sequence with pieces[s] <= it (those before it without pieces are passed by)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sh.pieces[mid] <= it) lo = mid; else hi = mid - 1;
    }
    const int s = __builtin_amdgcn_readfirstlane(lo);
    Piece p = seq_shape(a, s, cap);
    const int nt = steps(p), cuts = (nt + L - 1) / L, nrb = (p.n * a.group + P::R - 1) / P::R;
    const int at = __builtin_amdgcn_readfirstlane(it - sh.pieces[s]);  // ((kv head, piece), row block)
    p.rb = at % nrb;
    const int kj = at / nrb;
    p.kvh = kj / cuts;
    const int j = kj - p.kvh * cuts;
    p.step0 = static_cast<int>(static_cast<int64_t>(nt) * j / cuts);
    p.step1 = static_cast<int>(static_cast<int64_t>(nt) * (j + 1) / cuts);
    int64_t rec = -1;
    if (cuts > 1) {
      const int first = __builtin_amdgcn_readfirstlane(sh.recs[s]) + (p.kvh * nrb + p.rb) * cuts;
      rec = first + j;
      if (tid == 0) {
        int32_t* d = a.ws_desc + rec * kDesc;
        d[0] = j == 0 ? cuts : 0;
        d[1] = s;
        d[2] = p.kvh;
        d[3] = p.rb;
      }
    }
    if (run_piece<DT, D, WR, WK, NC, false>(a, p, rec, it + 1u, smem, sh))
      run_piece<DT, D, WR, WK, NC, true>(a, p, rec, it + 1u, smem, sh);
  }
}

// Combine the pieces of every split segment. Workgroup (g, y): column block y of the segment whose first
// record is g.
template <int DT, int D, int R>
__global__ __launch_bounds__(256) void paged_tree_merge(TreeArgs a) {
  using Ops = MfmaOps<DT>;
  using S = typename Elem<DT>::S;
  constexpr int MT = D / 16, PER = MT / 4;  // dim tiles; of each wavefront
  const int g = blockIdx.x, cb = blockIdx.y;
  const int32_t* d = a.ws_desc + g * kDesc;
  const int pieces = d[0];
  if (pieces == 0) return;
  const int s = d[1], kvh = d[2], rb = d[3];
  const int q0 = a.cu_q[s];
  int n = a.cu_q[s + 1] - q0;
  n = n < a.max_q_len ? n : a.max_q_len;
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave, i16 = lane & 15, grp = lane >> 4;
  const int r = rb * R + cb * 16 + i16, t = r / a.group, h = kvh * a.group + r - t * a.group;
  if (rb * R + cb * 16 >= n * a.group) return;
  const float* first = a.ws_rec + static_cast<int64_t>(g) * a.rec_floats;
  float m = -INFINITY;
  for (int p = 0; p < pieces; ++p) m = fmaxf(m, first[p * a.rec_floats + cb * 16 + i16]);
  float l = 0.0f;
  f32x4_t acc[PER];
#pragma unroll
  for (int x = 0; x < PER; ++x) acc[x] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int p = 0; p < pieces; ++p) {
    const float* rec = first + p * a.rec_floats;
    const float mp = rec[cb * 16 + i16];
    const float f = mp == -INFINITY ? 0.0f : fast_exp2(mp - m);
    l += f * rec[R + cb * 16 + i16];
    const f32x4_t* racc = reinterpret_cast<const f32x4_t*>(rec + 2 * R) + (cb * MT + w * PER) * kWave + lane;
#pragma unroll
    for (int x = 0; x < PER; ++x) acc[x] += racc[x * kWave] * f;
  }
  if (t >= n) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  S* orow = reinterpret_cast<S*>(a.out) + (static_cast<int64_t>(q0) + t) * a.out_st + static_cast<int64_t>(h) * a.out_sh;
#pragma unroll
  for (int x = 0; x < PER; ++x) {
    const uint32_t w0 = Ops::pack2(acc[x][0] * inv, acc[x][1] * inv), w1 = Ops::pack2(acc[x][2] * inv, acc[x][3] * inv);
    *reinterpret_cast<uint2*>(orow + 16 * (w * PER + x) + 4 * grp) = make_uint2(w0, w1);
  }
}

// ------------------------------------------------------------------ one query row at a time
//
// Every type, head size (powers of two from 8 to 256), group and alignment of elements: a workgroup of 4
// wavefronts per (node, query head). A lane holds 16 bytes of a row, LPR lanes a row, so a wavefront
// takes 64 / LPR keys at once and every key's row lanes keep a softmax state of their own (a score is summed
// over its LPR lanes alone); the states meet at the end. A key that the row does not see contributes
// nothing at all, whatever its bytes are.
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_tree_row_kernel(TreeArgs a, int hq) {
  using S = typename Elem<DT>::S;
  constexpr int ES = Elem<DT>::kBytes, N = 16 / ES, LPR = D / N > 0 ? D / N : 1, RPP = kWave / LPR;
  static_assert(D % N == 0 && LPR <= kWave, "a row is whole 16-byte chunks, at most 64");
  constexpr int kStates = 4 * RPP;
  __shared__ float s_m[kStates], s_l[kStates];
  __shared__ float s_acc[kStates][D];
  const int64_t x = blockIdx.x;  // (sequence, node)
  const int s = static_cast<int>(x / a.max_q_len), i = static_cast<int>(x - static_cast<int64_t>(s) * a.max_q_len);
  const Piece p = seq_shape(a, s, a.max_blocks * a.bs);
  if (i >= p.n) return;
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
  auto values = [&](const char* pool, int64_t at, float (&v)[N]) {
    const uint4 u = *reinterpret_cast<const uint4*>(pool + at);
    S raw[N];
    __builtin_memcpy(raw, &u, 16);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = widen<DT>(raw[e]);
  };
  for (int base = 0; base < p.keys; base += 4 * RPP) {
    const int key = base + w * RPP + row, e0 = key - p.ctx;
    bool seen = key < p.keys;
    if (seen && e0 >= 0) seen = (e0 >> 6) < a.mask_words && ((mask[e0 >> 6] >> (e0 & 63)) & 1u);
    const int blk = seen ? table[key >> a.log2_bs] : -1;
    seen = blk >= 0 && blk < a.ncb;
    const int64_t at = (((static_cast<int64_t>(seen ? blk : 0) * a.hkv + kvh) * a.bs + (key & (a.bs - 1))) * D + c * N) * ES;
    float kf[N];
    values(a.k, at, kf);
    float dot = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) dot = fmaf(qf[e], kf[e], dot);
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) dot += __shfl_xor(dot, o);
    if (seen && dot != -INFINITY) {
      float vf[N];
      values(a.v, at, vf);
      const float sc = dot * a.scale_log2;
      const float mn = fmax2(m, sc);
      const float alpha = fast_exp2(m - mn), pk = fast_exp2(sc - mn);  // m = -inf before any key: alpha 0
      l = l * alpha + pk;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = fmaf(pk, vf[e], acc[e] * alpha);
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
    reinterpret_cast<S*>(a.out)[r * a.out_st + static_cast<int64_t>(h) * a.out_sh + d] =
        from_f32<DT>(Ls == 0.0f ? 0.0f : A / Ls);
  }
}

// ------------------------------------------------------------------ host side

using KernelFn = void (*)(TreeArgs);

struct Config {
  KernelFn fn = nullptr, merge = nullptr;
  int rows = 0, keys = 0, threads = 0;  // R, KT
  int64_t rec_floats = 0;
};

template <int DT, int D, int WR, int WK, int NC>
Config config_of() {
  using P = Shape<D, WR, WK, NC>;
  return {paged_tree_kernel<DT, D, WR, WK, NC>, paged_tree_merge<DT, D, P::R>, P::R, P::KT, P::T, P::kRec};
}

// The workgroup's shape by the most rows a sequence can have.
template <int DT>
Config pick(int d, int64_t rows) {
  if (d == 64) {
    if (rows <= 16) return config_of<DT, 64, 1, 4, 1>();
    if (rows <= 32) return config_of<DT, 64, 1, 4, 2>();
    if (rows <= 64) return config_of<DT, 64, 1, 4, 4>();
    if (rows <= 128) return config_of<DT, 64, 2, 2, 4>();
    return config_of<DT, 64, 4, 1, 4>();
  }
  if (rows <= 16) return config_of<DT, 128, 1, 2, 1>();
  if (rows <= 32) return config_of<DT, 128, 1, 2, 2>();
  if (rows <= 64) return config_of<DT, 128, 2, 2, 2>();
  return config_of<DT, 128, 4, 1, 2>();
}

constexpr int kWgPerCu = 2;
constexpr int kMinSteps = 2;

int compute_units() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 256;
  return cus;
}

struct Plan {
  Config cfg;
  bool ok = false;      // the matrix-core kernel takes this shape
  int target = 0, grid = 0, max_recs = 0, rec_grid = 0;
  int64_t desc_off = 0, bytes = 0;
};

Plan plan_of(int num_seqs, int max_q_len, int hq, int hkv, int d, int bs, int max_blocks, int dtype) {
  Plan p;
  const int group = hq / hkv;
  const int64_t rows = static_cast<int64_t>(max_q_len) * group, cap = static_cast<int64_t>(max_blocks) * bs;
  if ((dtype != MIP_F16 && dtype != MIP_BF16) || (d != 64 && d != 128) || num_seqs > kMaxSeqs) return p;
  p.cfg = dtype == MIP_F16 ? pick<MIP_F16>(d, rows) : pick<MIP_BF16>(d, rows);
  const int64_t segs = static_cast<int64_t>(num_seqs) * hkv * ((rows + p.cfg.rows - 1) / p.cfg.rows);
  const int64_t steps = (cap + p.cfg.keys - 1) / p.cfg.keys;
  if (segs * steps >= (int64_t{1} << 30)) return p;
  p.ok = true;
  const int slots = (compute_units() * kWgPerCu + 7) / 8 * 8;
  p.target = slots;
  // Pieces: at most one per kMinSteps steps beside the last, and at most target + segments in all. A split segment has
  // more than L >= total / target steps and at most steps / L + 1 pieces: at most 2 target records.
  const int64_t cuts = (steps + kMinSteps - 1) / kMinSteps;
  const int64_t pieces = segs * cuts < slots + segs ? segs * cuts : slots + segs;
  p.grid = static_cast<int>((pieces < slots ? pieces : slots) + 7) / 8 * 8;
  const int64_t recs = cuts > 1 ? (segs * cuts < 2 * slots ? segs * cuts : 2 * slots) : 0;
  p.max_recs = static_cast<int>(recs);
  p.desc_off = (recs * p.cfg.rec_floats * 4 + 255) / 256 * 256;
  p.bytes = recs > 0 ? p.desc_off + recs * kDesc * 4 : 0;
  return p;
}

template <int DT>
bool launch_row_d(const TreeArgs& a, int d, int hq, dim3 grid, hipStream_t s) {
  switch (d) {
    case 8:   hipLaunchKernelGGL((paged_tree_row_kernel<DT, 8>), grid, dim3(256), 0, s, a, hq); return true;
    case 16:  hipLaunchKernelGGL((paged_tree_row_kernel<DT, 16>), grid, dim3(256), 0, s, a, hq); return true;
    case 32:  hipLaunchKernelGGL((paged_tree_row_kernel<DT, 32>), grid, dim3(256), 0, s, a, hq); return true;
    case 64:  hipLaunchKernelGGL((paged_tree_row_kernel<DT, 64>), grid, dim3(256), 0, s, a, hq); return true;
    case 128: hipLaunchKernelGGL((paged_tree_row_kernel<DT, 128>), grid, dim3(256), 0, s, a, hq); return true;
    case 256: hipLaunchKernelGGL((paged_tree_row_kernel<DT, 256>), grid, dim3(256), 0, s, a, hq); return true;
    default:  return false;
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
  return static_cast<size_t>(
      tree::plan_of(num_seqs, max_q_len, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, dtype).bytes);
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
  if (!is_pow2(block_size) || block_size > 4096 || num_cache_blocks > INT32_MAX || !(scale > 0.0f)) return MIP_EINVAL;
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
  if (p.ok) {
    if (p.bytes > 0) {
      if (!workspace || workspace_bytes < static_cast<size_t>(p.bytes) || (reinterpret_cast<uintptr_t>(workspace) & 255))
        return MIP_EINVAL;
      a.ws_rec = static_cast<float*>(workspace);
      a.ws_desc = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + p.desc_off);
    }
    a.rec_floats = p.cfg.rec_floats;
    a.target = p.target;
    a.min_steps = tree::kMinSteps;
    a.max_recs = p.max_recs;
    hipLaunchKernelGGL(p.cfg.fn, dim3(p.grid), dim3(p.cfg.threads), 0, s, a);
    if (p.max_recs > 0)
      hipLaunchKernelGGL(p.cfg.merge, dim3(p.max_recs, p.cfg.rows / 16), dim3(256), 0, s, a);
    return status_from_hip(hipGetLastError());
  }
  const int64_t rows = static_cast<int64_t>(num_seqs) * max_q_len;
  if (rows >= (int64_t{1} << 24) || num_heads > 65535) return MIP_EUNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(rows), num_heads);
  bool found;
  switch (dtype) {
    case MIP_F32: found = tree::launch_row_d<MIP_F32>(a, head_dim, num_heads, grid, s); break;
    case MIP_F16: found = tree::launch_row_d<MIP_F16>(a, head_dim, num_heads, grid, s); break;
    default:      found = tree::launch_row_d<MIP_BF16>(a, head_dim, num_heads, grid, s); break;
  }
  return found ? status_from_hip(hipGetLastError()) : MIP_EUNSUPPORTED;
}
