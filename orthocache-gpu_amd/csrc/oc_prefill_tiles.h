#pragma once
// The tile step of the flash-attention kernels over whole prompts (prefill,
// query blocks, changed scores): a workgroup of eight waves stages the K and V
// of one 64-token tile in LDS, and each wave computes S^T = K q^T for its 16
// queries, updates the online softmax, and adds V^T P^T.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "oc_kernels.h"
#include "orthocache_hip.h"

namespace oc {
namespace {

constexpr int kPfWaves = 8;
constexpr int kPfRows = 16 * kPfWaves;  // query positions per workgroup
constexpr int kPfThreads = kPfWaves * kWave;
constexpr int kPfPvGroup = 4;  // p.V column pairs whose V reads are in flight together
// work items of a call that splits its longest causal windows (beyond: no split)
constexpr int kPfMaxItems = 512;
// -(1e-10) * ln(1e-10): what one zero probability adds to the entropy of a
// softmax row whose probabilities are clamped to >= 1e-10 before the log
constexpr float kZeroPTerm = 2.302585093e-9f;

struct PrefillArgs {
  const char* q;
  const char* k;
  const char* v;
  char* out;
  int64_t q_sb, q_sh, q_ss;  // byte strides (batch, head, position)
  int64_t k_sb, k_sh, k_ss;
  int64_t v_sb, v_sh, v_ss;
  int64_t o_sb, o_sh, o_ss;
  int32_t B, Hq, Hkv, G, Sq, Skv, T;  // T: full tiles the mask covers
  const uint8_t* mask;                // (B, Hkv, >= T) evict flags or null
  int64_t m_sb, m_sh;
  float scale;
  float* entropy;  // (B, Hq, Sq) or null
  int32_t qblocks;
  int32_t o_vec;  // out rows 8-byte aligned
  int32_t rev;    // query blocks dispatched longest first; those after them shortest first
  // split windows (nitems > 0): work item e is query block items[e] >> 2,
  // part items[e] & 3 (0: its whole window; 1, 2: the first and second half
  // of its tiles).  Blocks >= q0 are split: (block, head) pair k of them keeps
  // the two halves' per-lane states at part + (2 k + half) * 512 * (4 + D/4)
  // floats and its ticket at ctr[k * ctr_stride].
  int32_t nitems, q0, ctr_stride;
  float* part;
  int32_t* ctr;
  uint16_t items[kPfMaxItems];
};

// Online-softmax state in the transposed layout: lane 16r + x works on
// query x (scores of tokens 16tb + 4r + i, i = 0..3, in c[tb][i]); m is
// shared by the query's four lanes x, x + 16, x + 32, x + 48, and l, e are
// their partial sums.  Scores are kept in base-2 units (s2 = s * log2 e), so
// that each probability is one exp2.  m is the reference that the sums and
// accumulators are relative to: at least the running max less kPfSlack.
struct PfState {
  float m;  // base-2 units
  float l;
  float e;  // sum of 2^(s2 - m) * s2 (entropy), base-2 units
  int n;    // attended tokens of the query (entropy)
};

// The accumulators are rescaled only when a query's max has passed its
// reference by more than this many powers of two; until then its
// probabilities are at most 2^kPfSlack, of the same relative precision.  (With
// the reference always the running max, some query of the wave's 16 moved it
// in most tiles of a window, at 32 multiplications a lane each time.)  This, the
// scale inside the fma and the tile walk without memory reads took the 32-head
// 4096-token layer of 128 columns from 217 to 202 us in bfloat16 and 177 to 163
// in float16, and with half the tiles evicted from 152 to 125 and 127 to 103;
// the kernel is bound by the vector instructions between its matrix products
// (69% of the SIMD cycles before).
constexpr float kPfSlack = 8.f;

// Causal online-softmax update of one tile's raw scores c (transposed
// layout); token tok0 + j is visible to the lane's query when tok0 + j <
// nvis.  full (wave-uniform): every token of the tile is visible to every
// query of the wave (no mask needed).  scale2 = softmax scale * log2 e.
// c becomes 2^(s2 - m).  A full tile's scores stay unscaled: their max is
// scaled once (scale2 > 0), and the scale goes into the exponent's fma.
template <int D, bool ENT>
__device__ __forceinline__ void pf_softmax(PfState& st, f32x4 (&acc)[D / 16], f32x4 (&c)[4], float scale2, int nvis,
                                           int tok0, bool full, int lane) {
  (void)lane;  // lane / 16 (the row group r) is formed from the thread index below
  float mt = -__builtin_inff();
  float s = 1.f;  // c's units: s2 = c * s
  if (full && scale2 > 0.f) {
#pragma unroll
    for (int tb = 0; tb < 4; ++tb)
#pragma unroll
      for (int i = 0; i < 4; ++i) mt = fmaxf(mt, c[tb][i]);
    mt *= scale2;
    s = scale2;
  } else {
    // 4 r formed here from the thread index (lane = threadIdx.x mod 64; the
    // empty asm keeps the compiler from keeping it in a register across the
    // tile loop, where the bfloat16 entropy kernels would spill it)
    int tx = threadIdx.x;
    asm volatile("" : "+v"(tx));
    const int r4 = (tx >> 2) & 12;
#pragma unroll
    for (int tb = 0; tb < 4; ++tb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = full || tok0 + 16 * tb + r4 + i < nvis ? c[tb][i] * scale2 : -__builtin_inff();
        c[tb][i] = v;
        mt = fmaxf(mt, v);
      }
  }
  mt = fmaxf(mt, xpair<16>(mt));
  mt = fmaxf(mt, xpair<32>(mt));
  const bool move = mt > st.m + kPfSlack;
  if (__builtin_amdgcn_ballot_w64(move)) {
    const float mn = move ? mt : st.m;
    const float alpha = __builtin_amdgcn_exp2f(st.m - mn);  // 1 for the queries that stay
    st.m = mn;
    st.l *= alpha;
    if constexpr (ENT) st.e *= alpha;
#pragma unroll
    for (int nc = 0; nc < D / 16; ++nc) acc[nc] *= alpha;
  }
  float ls = 0.f, es = 0.f;
#pragma unroll
  for (int tb = 0; tb < 4; ++tb)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = c[tb][i];
      const float pp = __builtin_amdgcn_exp2f(__builtin_fmaf(v, s, -st.m));
      ls += pp;
      if constexpr (ENT) es = pp > 0.f ? __builtin_fmaf(pp, v, es) : es;
      c[tb][i] = pp;
    }
  st.l += ls;
  if constexpr (ENT) {
    st.e = __builtin_fmaf(es, s, st.e);
    st.n += min(max(nvis - tok0, 0), 64);
  }
}

// q of the wave's 16 rows as MFMA A operands.  16-bit: lane 16kg + x holds
// elements 32dc + 8kg .. +8 of row x for instruction dc.  float32 (16x16x4
// instructions): lane 16kg + x holds column kg*D/4 + dc of row x for
// instruction dc.  Rows past q_len read as zero.
template <int DT, int D>
struct PfQ {
  static constexpr bool F32 = DT == OC_F32;
  uint32_t w[F32 ? D / 4 : D / 8];
};

template <int DT, int D>
__device__ __forceinline__ void pf_load_q(const PrefillArgs& a, const char* qh, int pos0, int lane, PfQ<DT, D>& q) {
  const int x = lane & 15;
  const int kg = lane >> 4;
  const bool ok = pos0 + x < a.Sq;
  const char* rowp = qh + (int64_t)(pos0 + x) * a.q_ss;
  if constexpr (DT == OC_F32) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      uint4 u = {0u, 0u, 0u, 0u};
      if (ok) u = *reinterpret_cast<const uint4*>(rowp + 4 * (kg * (D / 4) + 4 * j));
      q.w[4 * j] = u.x;
      q.w[4 * j + 1] = u.y;
      q.w[4 * j + 2] = u.z;
      q.w[4 * j + 3] = u.w;
    }
  } else {
#pragma unroll
    for (int dc = 0; dc < D / 32; ++dc) {
      uint4 u = {0u, 0u, 0u, 0u};
      if (ok) u = *reinterpret_cast<const uint4*>(rowp + 2 * (32 * dc + 8 * kg));
      q.w[4 * dc] = u.x;
      q.w[4 * dc + 1] = u.y;
      q.w[4 * dc + 2] = u.z;
      q.w[4 * dc + 3] = u.w;
    }
  }
}

// The workgroup's shared K/V tiles: K and V of one 64-token tile, row-major
// [token][D], in STAGES LDS stages.  The 512 threads stage the next tile, in
// 16-byte chunks, while the waves compute the current one: straight into the
// other stage where there are two, else (float32 at head_dim 128) through
// registers, stored once that compute is done.  K's chunks
// are XOR-swizzled per row (chunk c of row r sits at c ^ swz(r)) so that the
// 16 rows one B-operand read touches fall in distinct LDS banks.
template <int DT, int D>
struct PfTile {
  static constexpr int ES = DT == OC_F32 ? 4 : 2;
  static constexpr int ROW = D * ES;                      // bytes per token row
  static constexpr int LPT = ROW / 16;                    // 16-byte chunks per row
  static constexpr int RB = ROW >= 256 ? 1 : 256 / ROW;   // rows per 256-byte bank line
  static constexpr int KV = 64 * ROW;                     // bytes of one K (or V) tile
  static constexpr int NL = KV / (kPfThreads * 16);       // chunks per thread per matrix
  static constexpr int STAGES = 2 * KV <= 32768 ? 2 : 1;
  static constexpr int LDS = STAGES * 2 * KV;
  __device__ static int swz(int r) { return (r / RB) % LPT; }
  // 16-bit V: the 32-byte column pair p of LDS row r is stored at pair
  // p ^ vswz(r).  A transposing read takes one pair of the 16 rows
  // 8g + i (+ 4h), g, i < 4; vswz gives those rows distinct pairs (each
  // bank slot used twice) instead of one pair 16 times over.
  static constexpr int PAIRS = ROW / 32;
  __device__ static int vswz(int r) {
    return PAIRS >= 8 ? (r & 3) + 4 * ((r >> 3) & 1) : ((r & 3) >> 1) + 2 * ((r >> 3) & 1);
  }
};

template <int DT, int D>
struct PfStage {
  uint4 k[PfTile<DT, D>::NL];
  uint4 v[PfTile<DT, D>::NL];
};

// a wave-uniform pointer as scalar registers
__device__ __forceinline__ const char* pf_uniform(const char* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return reinterpret_cast<const char*>(((uint64_t)hi << 32) | lo);
}

// global -> registers: chunk g = tid + 512 j of the tile is row g / LPT,
// chunk g % LPT; rows at or past kv_len read as zero (buffer range check)
template <int DT, int D>
__device__ __forceinline__ void pf_fetch(const PrefillArgs& a, const char* kh, const char* vh, int t, int tid,
                                         PfStage<DT, D>& st) {
  using L = PfTile<DT, D>;
  // every value of the resources is wave-uniform; saying so keeps the
  // compiler from wrapping each load in a readfirstlane loop
  t = __builtin_amdgcn_readfirstlane(t);
  const int nvalid = min(a.Skv - t * 64, 64);
  const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
      (void*)pf_uniform(kh + (int64_t)t * 64 * a.k_ss), (short)0,
      __builtin_amdgcn_readfirstlane(nvalid * (int)a.k_ss), 0x00020000);
  const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
      (void*)pf_uniform(vh + (int64_t)t * 64 * a.v_ss), (short)0,
      __builtin_amdgcn_readfirstlane(nvalid * (int)a.v_ss), 0x00020000);
#pragma unroll
  for (int j = 0; j < L::NL; ++j) {
    const int g = tid + kPfThreads * j;
    const int r = g / L::LPT, c = g % L::LPT;
    const auto uk = __builtin_amdgcn_raw_buffer_load_b128(rk, r * (int)a.k_ss + 16 * c, 0, 0);
    const auto uv = __builtin_amdgcn_raw_buffer_load_b128(rv, r * (int)a.v_ss + 16 * c, 0, 0);
    st.k[j] = uint4{uk[0], uk[1], uk[2], uk[3]};
    st.v[j] = uint4{uv[0], uv[1], uv[2], uv[3]};
  }
}

// 16 bytes per lane from a buffer straight to LDS: lane i's bytes land at
// dst + 16 i (dst wave-uniform)
__device__ __forceinline__ void pf_load_lds16(__amdgpu_buffer_rsrc_t r, char* dst, int voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, voff, 0, 0, 0);
}

// Token kept in LDS row r of a 16-bit V stage: within each 32-token block,
// token 16a + 4g + b sits in row 8g + 4a + b, so that the transposing read
// of rows 8g .. 8g + 7 hands lane group g the tokens 4g + b and 16 + 4g + b
// -- the tokens whose scores the lane holds (pf_pv).
__device__ __forceinline__ int pf_vtok(int r) {
  return (r & ~31) + 16 * ((r >> 2) & 1) + 4 * ((r >> 3) & 3) + (r & 3);
}

// global -> an LDS stage directly (two-stage tiles): each wave's load
// instruction fills a contiguous 1 KiB of the stage, slot g = tid + 512 j
// (row g / LPT, chunk g % LPT), so the lane filling a slot loads the chunk
// that the layout keeps there: K chunk c ^ swz(row); 16-bit V the token
// pf_vtok(row), chunk c ^ 2 vswz(row).  Rows at or past kv_len read as zero
// (buffer range check).  Default cache policy: the G query heads' workgroups
// of a kv head read the same tiles.
template <int DT, int D>
__device__ __forceinline__ void pf_fetch_lds(const PrefillArgs& a, const char* kh, const char* vh, int t, int tid,
                                             char* sk, char* sv) {
  using L = PfTile<DT, D>;
  t = __builtin_amdgcn_readfirstlane(t);
  const int nvalid = min(a.Skv - t * 64, 64);
  const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
      (void*)pf_uniform(kh + (int64_t)t * 64 * a.k_ss), (short)0,
      __builtin_amdgcn_readfirstlane(nvalid * (int)a.k_ss), 0x00020000);
  const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
      (void*)pf_uniform(vh + (int64_t)t * 64 * a.v_ss), (short)0,
      __builtin_amdgcn_readfirstlane(nvalid * (int)a.v_ss), 0x00020000);
  const int wbase = __builtin_amdgcn_readfirstlane(tid & ~63);  // the wave's first slot
#pragma unroll
  for (int j = 0; j < L::NL; ++j) {
    const int g = tid + kPfThreads * j;
    const int r = g / L::LPT, c = g % L::LPT;
    const int slot0 = 16 * (wbase + kPfThreads * j);
    pf_load_lds16(rk, sk + slot0, r * (int)a.k_ss + 16 * (c ^ L::swz(r)));
    int vt = r, vc = c;
    if constexpr (DT != OC_F32) {
      vt = pf_vtok(r);
      vc = c ^ (2 * L::vswz(r));
    }
    pf_load_lds16(rv, sv + slot0, vt * (int)a.v_ss + 16 * vc);
  }
}

// registers -> the LDS stage (single-stage tiles: float32 at head_dim 128;
// 16-bit tiles always have two stages and load straight into LDS): K
// swizzled, V in token order
template <int DT, int D>
__device__ __forceinline__ void pf_stash(const PfStage<DT, D>& st, int tid, char* sk, char* sv) {
  using L = PfTile<DT, D>;
  static_assert(DT == OC_F32, "only float32 tiles are staged through registers");
#pragma unroll
  for (int j = 0; j < L::NL; ++j) {
    const int g = tid + kPfThreads * j;
    const int r = g / L::LPT, c = g % L::LPT;
    *reinterpret_cast<uint4*>(sk + r * L::ROW + 16 * (c ^ L::swz(r))) = st.k[j];
    *reinterpret_cast<uint4*>(sv + r * L::ROW + 16 * c) = st.v[j];
  }
}

// S^T = K.q^T of one tile from the LDS stage: c[tb][i] is the score of
// token 16tb + 4r + i for query x in lane 16r + x.  K is the A operand:
// 16-bit instruction dc takes row 16tb + x, logical chunk 4dc + kg; float32
// reads 4 columns kg*D/4 + 4j .. for instructions 4j .. 4j + 3; q (the B
// operand) is in the same registers as before.
template <int DT, int D>
__device__ __forceinline__ void pf_logits(const PfQ<DT, D>& q, const char* sk, int lane, f32x4 (&c)[4]) {
  using L = PfTile<DT, D>;
  const int x = lane & 15;
  const int kg = lane >> 4;
#pragma unroll
  for (int tb = 0; tb < 4; ++tb) {
    c[tb] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int r = 16 * tb + x;
    const char* rowp = sk + r * L::ROW;
    const int sw = L::swz(r);
    if constexpr (DT == OC_F32) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const uint4 u = *reinterpret_cast<const uint4*>(rowp + 16 * ((kg * (D / 16) + j) ^ sw));
        const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          c[tb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(uw[e]), __uint_as_float(q.w[4 * j + e]),
                                                       c[tb], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int dc = 0; dc < D / 32; ++dc) {
        const uint4 u = *reinterpret_cast<const uint4*>(rowp + 16 * ((4 * dc + kg) ^ sw));
        const uint32_t aq[4] = {q.w[4 * dc], q.w[4 * dc + 1], q.w[4 * dc + 2], q.w[4 * dc + 3]};
        const uint32_t bk[4] = {u.x, u.y, u.z, u.w};
        c[tb] = mfma_qk<DT>(bk, aq, c[tb]);
      }
    }
  }
}

// O^T += V^T P^T on the matrix cores (transposed layout): acc[nc][i] is
// output column 16nc + 4r + i of query x in lane 16r + x.  16-bit: per
// 32-token block j, A = V^T read with ds_read_b64_tr_b16 from the permuted
// rows (lane group g gets tokens 32j + 4g + b and 32j + 16 + 4g + b), B =
// the lane's own eight probabilities c[2j][b], c[2j + 1][b].  HILO sends a
// 16-bit high part plus the 16-bit rounding of the remainder (two
// instructions); without it they are rounded once, which the causal kernel
// does for float16 (relative error at most 2^-11; below 2^-14, where float16 is
// subnormal, an absolute 2^-25): in bfloat16 one rounding (2^-8) moves short
// causal rows past the output tolerance.
// float32: 16x16x4 steps over (tb, i), A = V[16tb + 4r + i][16nc + x], B =
// c[tb][i], exact.
// PK: pairs by one instruction (the same rounding).
template <int DT, int D, bool HILO = DT == OC_BF16, bool PK = false>
__device__ __forceinline__ void pf_pv(f32x4 (&acc)[D / 16], const f32x4 (&c)[4], const char* svb, int lane) {
  const int x = lane & 15;
  const int kg = lane >> 4;
  if constexpr (DT == OC_F32) {
    const float* sv = reinterpret_cast<const float*>(svb);
#pragma unroll
    for (int tb = 0; tb < 4; ++tb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* vr = sv + (16 * tb + 4 * kg + i) * D + x;
#pragma unroll
        for (int nc = 0; nc < D / 16; ++nc)
          acc[nc] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[16 * nc], c[tb][i], acc[nc], 0, 0, 0);
      }
  } else {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    const uint16_t* sv = reinterpret_cast<const uint16_t*>(svb);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float pv[8];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        pv[b] = c[2 * j][b];
        pv[4 + b] = c[2 * j + 1][b];
      }
      uint32_t bhi[4], blo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (PK) {
          static_assert(!HILO, "pairs are rounded once");
          typedef float f32x2 __attribute__((ext_vector_type(2)));
          typedef std::conditional_t<DT == OC_BF16, __bf16, _Float16> T;
          typedef T pair __attribute__((ext_vector_type(2)));
          bhi[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{pv[2 * e], pv[2 * e + 1]}), pair));
        } else if constexpr (DT == OC_BF16) {
          const __bf16 h0 = (__bf16)pv[2 * e], h1 = (__bf16)pv[2 * e + 1];
          bhi[e] = (uint32_t)__builtin_bit_cast(uint16_t, h0) | ((uint32_t)__builtin_bit_cast(uint16_t, h1) << 16);
          if constexpr (HILO) {
            const __bf16 l0 = (__bf16)(pv[2 * e] - (float)h0), l1 = (__bf16)(pv[2 * e + 1] - (float)h1);
            blo[e] = (uint32_t)__builtin_bit_cast(uint16_t, l0) | ((uint32_t)__builtin_bit_cast(uint16_t, l1) << 16);
          }
        } else {
          const _Float16 h0 = (_Float16)pv[2 * e], h1 = (_Float16)pv[2 * e + 1];
          bhi[e] = (uint32_t)__builtin_bit_cast(uint16_t, h0) | ((uint32_t)__builtin_bit_cast(uint16_t, h1) << 16);
          if constexpr (HILO) {
            const _Float16 l0 = (_Float16)(pv[2 * e] - (float)h0), l1 = (_Float16)(pv[2 * e + 1] - (float)h1);
            blo[e] = (uint32_t)__builtin_bit_cast(uint16_t, l0) | ((uint32_t)__builtin_bit_cast(uint16_t, l1) << 16);
          }
        }
      }
      // lane x of group kg reads rows 32j + 8kg + 4h + x/4 (h = 0, 1), column
      // pair nc stored at nc ^ vswz(row) (the same for h = 0, 1 and every j)
      const int vrow = 32 * j + 8 * kg + (x >> 2);
      const int vt = PfTile<DT, D>::vswz(vrow);
      const uint16_t* rowp = sv + vrow * D + 4 * (x & 3);
      // the transposing reads of GS column pairs are issued before their
      // products, so that their latencies overlap
#pragma unroll
      for (int n0 = 0; n0 < D / 16; n0 += kPfPvGroup) {
        uint32_t av[kPfPvGroup][4];
#pragma unroll
        for (int g = 0; g < kPfPvGroup; ++g) {
          const int nc = n0 + g;
          const s16x4 b0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(rowp + 16 * (nc ^ vt)));
          const s16x4 b1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(rowp + 4 * D + 16 * (nc ^ vt)));
          typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
          const u32x2 w0 = __builtin_bit_cast(u32x2, b0), w1 = __builtin_bit_cast(u32x2, b1);
          av[g][0] = w0[0];
          av[g][1] = w0[1];
          av[g][2] = w1[0];
          av[g][3] = w1[1];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < kPfPvGroup; ++g) {
          acc[n0 + g] = mfma_qk<DT>(av[g], bhi, acc[n0 + g]);
          if constexpr (HILO) acc[n0 + g] = mfma_qk<DT>(av[g], blo, acc[n0 + g]);
        }
      }
    }
  }
}

// two values rounded to the 16-bit type DT
template <int DT>
__device__ __forceinline__ uint32_t pf_pack(float lo, float hi) {
  if constexpr (DT == OC_BF16) return bf16_bits(lo) | (bf16_bits(hi) << 16);
  else return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16);
}

}  // namespace
}  // namespace oc
