// Attention of whole prompts with changed scores (declared in
// include/orthocache_paged.h): capped by a tanh, biased by distance, in a
// window, behind a prefix, between documents.
//
// The tile step is the prefill kernel's (oc_prefill_tiles.h): a workgroup of
// eight waves, 16 queries each, walks the 64-token tiles that any of its 128
// queries sees, through a bit word of 64 tiles at a time.  A tile that every
// query of a wave sees whole takes no mask; only the tiles at the borders of
// the causal triangle, the window, the prefix and the documents do.
//
// What is not seen must have no effect, NaN and infinities among it.  A masked
// score is replaced, so K needs nothing; V does, since 0 * NaN is NaN: the
// threads that stage a border tile look at the 16-byte pieces they staged, and
// a tile that holds a value which is not finite takes a slower p.V
// (prompt_pv_any).
//
// P is rounded once to the 16-bit type (half a step, as large as the output's
// own rounding; two parts as in the prefill kernel would double its products).
// Bound by the vector instructions, busy for 80% of the cycles, beside matrix
// cores busy for 35%.  Measured, 32 / 8 heads of 128, 4096 tokens, bf16 / f16:
// 166 / 177 us without changes, 190 / 199 capped, 187 / 192 biased, 206 / 213
// both, 64 with documents of 600, 88 / 90 in a window of 1024.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "oc_kernels.h"
#include "oc_paged.h"
#include "oc_prefill_tiles.h"
#include "oc_status.h"
#include "orthocache_hip.h"
#include "orthocache_paged.h"

namespace oc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
// the reference that a row's sums are relative to before its first score: below every finite score
constexpr float kNoScore = -3e38f;

// What a head's scores go through: z = s (c - slope |i - j|) in base-2 units,
// with c the raw score, or its tanh in the same units near zero (cap_scores),
// and s = pre.  Where pre is negative or next to nothing, c is multiplied by it,
// and s is 1.
constexpr float kSmallest = 1e-6f;
struct Change {
  float s;
  float pre;         // scale log2(e), times kTanh0 with a cap
  float slope;       // the head's slope log2(e) / s
  float k, inv;      // scale / cap, 1 / (kTanh0 k)
  float lim, b1, b2; // |c| up to which the polynomial holds, its coefficients
};

struct PromptArgs {
  const char *q, *k, *v;
  char* out;
  int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss, v_sb, v_sh, v_ss, o_sb, o_sh, o_ss;  // bytes
  int32_t B, Hq, Hkv, G, Sq, Skv, T, qblocks;  // T: full tiles that the evict mask covers
  const int32_t* docs;
  int64_t docs_sb;
  const int2* ranges;  // (B, tiles) smallest and largest document of each tile
  const float* slopes;
  const int32_t* prefix;
  const uint8_t* evict;
  int64_t e_sb, e_sh;
  Change change;  // but for the slope
  int32_t cap, window;
  int32_t o_vec;  // out rows 8-byte aligned
  // The tiles of a workgroup's queries in shares of share_tiles (0: one share).
  // Each share's sums, of row ((b Hq + h) Sq + query) shares + share: m, l, acc.
  int32_t shares, share_tiles;
  float *pm, *pl, *pacc;
};

// The tiles that queries at places lo .. hi may see, as a range.
struct TileRange {
  int lo, hi;
};
__device__ __forceinline__ TileRange tile_range(int lo, int hi, int window, int prefix, int kv_len) {
  return {prefix > 0 || window >= lo ? 0 : (lo - window + 1) / 64, (min(max(max(hi + 1, prefix), 0), kv_len) + 63) / 64};
}
__device__ __forceinline__ int prefix_of(const int32_t* prefix, int b, int kv_len) {
  return prefix ? min(max(prefix[b], 0), kv_len) : 0;
}

// The kernel's arguments, read again from memory where they are used: held
// across the tile loop they would fill the scalar registers and push others out.
__device__ __forceinline__ const PromptArgs __attribute__((address_space(4))) * prompt_args() {
  auto p = (const PromptArgs __attribute__((address_space(4)))*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// the smallest and largest document of each 64-token tile: one wave a tile
__global__ __launch_bounds__(256) void doc_range_kernel(const int32_t* docs, int64_t docs_sb, int n, int tiles, int all,
                                                        int2* out) {
  const int w = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (w >= all) return;
  const int b = w / tiles, t = w - b * tiles;
  const int j = min(64 * t + lane, n - 1);
  int lo = docs[b * docs_sb + j], hi = lo;
  for (int o = 32; o > 0; o >>= 1) {
    lo = min(lo, __shfl_xor(lo, o, 64));
    hi = max(hi, __shfl_xor(hi, o, 64));
  }
  if (lane == 0) out[w] = int2{lo, hi};
}

// What the wave's queries see: query x is at place w_lo + x.
struct Sight {
  int w_lo, window, prefix;  // window: INT_MAX without one
  const int* qdoc;           // LDS: documents of the wave's 16 queries; null where they need not be looked at
  const int* tdoc;           // LDS: documents of the tile's 64 tokens
};

// The cap: a raw score c becomes tanh(k c) / (kTanh0 k), k = scale / cap.
// float32 takes tanhf.  The 16-bit kernels take c (1 + b1 c^2 + b2 c^4) while
// |k c| is at most kTanhFit (tanh(y) / y by a quadratic in y^2, fitted with a
// relative error of 4.0e-7 there), and 1 - 2 / (1 + e^2y) with the hardware's
// exponential and reciprocal where a score of the wave's tile is larger: four
// full-rate instructions against three and two quarter-rate ones.
constexpr float kTanhFit = 0.25f;
constexpr float kNoCap = 1e-37f;  // k below which there is no cap: 1 / k would not be finite
constexpr float kTanh0 = 0.999999604f, kTanh1 = -0.333219082f, kTanh2 = 0.128416128f;

template <int DT>
__device__ __forceinline__ void cap_scores(f32x4 (&c)[4], const Change& h) {
  if constexpr (DT == OC_F32) {
#pragma unroll
    for (int tb = 0; tb < 4; ++tb)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[tb][i] = h.k == 0.f ? c[tb][i] : tanhf(c[tb][i] * h.k) * h.inv;
  } else {
    float top = 0.f;
#pragma unroll
    for (int tb = 0; tb < 4; ++tb)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(c[tb][i]));
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > h.lim) != 0, 0)) {
#pragma unroll
      for (int tb = 0; tb < 4; ++tb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          c[tb][i] = __builtin_fmaf(
              -2.f * h.inv, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(c[tb][i] * (2.f * kLog2e * h.k))), h.inv);
    } else {
#pragma unroll
      for (int tb = 0; tb < 4; ++tb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = c[tb][i] * c[tb][i];
          c[tb][i] *= __builtin_fmaf(__builtin_fmaf(h.b2, u, h.b1), u, 1.f);
        }
    }
  }
}

// Online-softmax update of one tile (as pf_softmax) with the scores changed: c
// becomes 2^(z - m) for the tokens seen, 0 for the others.
template <int DT, int D, bool CAP, bool BIAS>
__device__ __forceinline__ void prompt_softmax(PfState& st, f32x4 (&acc)[D / 16], f32x4 (&c)[4], const Change& h,
                                               const Sight& e, int tok0, bool full) {
  float mt = -__builtin_inff();
  if constexpr (CAP) cap_scores<DT>(c, h);
  if (__builtin_expect(h.pre < kSmallest, 0)) {
#pragma unroll
    for (int tb = 0; tb < 4; ++tb) c[tb] *= h.pre;
  }
  // the lane's place in the tile, formed from the thread index (lane =
  // threadIdx.x mod 64) so that nothing of it is kept across the tile loop
  int tx = threadIdx.x;
  asm volatile("" : "+v"(tx));
  const int r4 = (tx >> 2) & 12, x = tx & 15;
  const int rel = e.w_lo + x - tok0 - r4;  // distance of the lane's query to its first token of the tile
  // the bias: -slope (d0 - n) for the lane's token n of the tile, n = 16 tb + i.
  // Where every token seen is at or before the query, its part in d0 is one
  // offset for the lane's scores; only behind a prefix can one be after it.
  float off = 0.f;
  if constexpr (BIAS) {
    const float d0 = (float)rel;
    if (e.prefix <= tok0 || tok0 + 63 <= e.w_lo) {
      off = h.slope * d0 * h.s;
#pragma unroll
      for (int tb = 0; tb < 4; ++tb)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[tb][i] = __builtin_fmaf(h.slope, (float)(16 * tb + i), c[tb][i]);
    } else {
#pragma unroll
      for (int tb = 0; tb < 4; ++tb)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[tb][i] = __builtin_fmaf(-h.slope, fabsf(d0 - (float)(16 * tb + i)), c[tb][i]);
    }
  }
  if (__builtin_expect(full, 1)) {
#pragma unroll
    for (int tb = 0; tb < 4; ++tb)
#pragma unroll
      for (int i = 0; i < 4; ++i) mt = fmaxf(mt, c[tb][i]);
  } else {
    const int pre = e.prefix - tok0 - r4;
    if (!e.qdoc && e.prefix <= tok0) {  // the causal border and the window alone
#pragma unroll
      for (int tb = 0; tb < 4; ++tb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // the distance in [0, window), both bounds in one comparison
          c[tb][i] = (unsigned)(rel - (16 * tb + i)) < (unsigned)e.window ? c[tb][i] : -__builtin_inff();
          mt = fmaxf(mt, c[tb][i]);
        }
    } else {
      const int doc = e.qdoc ? e.qdoc[x] : 0;
#pragma unroll
      for (int tb = 0; tb < 4; ++tb) {
        int4 td = {0, 0, 0, 0};
        if (e.qdoc) td = *reinterpret_cast<const int4*>(e.tdoc + 16 * tb + r4);
        const int tdv[4] = {td.x, td.y, td.z, td.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool ok = ((unsigned)(rel - (16 * tb + i)) < (unsigned)e.window || 16 * tb + i < pre) && tdv[i] == doc && doc >= 0;
          c[tb][i] = ok ? c[tb][i] : -__builtin_inff();
          mt = fmaxf(mt, c[tb][i]);
        }
      }
    }
  }
  float s = h.s;
  mt = __builtin_fmaf(mt, s, -off);
  float lo, hi;  // over the query's four lanes: a lane's own and its partner's, in either order
  row_pair<16>(mt, lo, hi);
  row_pair<32>(fmaxf(lo, hi), lo, hi);
  mt = fmaxf(lo, hi);
  // Far from zero the maximum's rounding is no longer small against 1, and the
  // fma below would see it: there the scores are rounded like the maximum.
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(fabsf(mt) > 16777216.f) != 0, 0)) {
#pragma unroll
    for (int tb = 0; tb < 4; ++tb)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[tb][i] = __builtin_fmaf(c[tb][i], s, -off);
    s = 1.f;
    off = 0.f;
  }
  const bool move = mt > st.m + kPfSlack;
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(move) != 0, 0)) {
    const float mn = move ? mt : st.m;
    const float alpha = __builtin_amdgcn_exp2f(st.m - mn);
    st.m = mn;
    st.l *= alpha;
#pragma unroll
    for (int nc = 0; nc < D / 16; ++nc) acc[nc] *= alpha;
  }
  float ls = 0.f;
  off += st.m;
#pragma unroll
  for (int tb = 0; tb < 4; ++tb)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(c[tb][i], s, -off));
      ls += p;
      c[tb][i] = p;
    }
  st.l += ls;
}

// one word of V (two 16-bit values, or a float32) split: its finite values (0
// in place of the others), and 1 where it is +inf or NaN, or -inf or NaN
template <int DT>
__device__ __forceinline__ void split_word(uint32_t w, uint32_t& fin, uint32_t& plus, uint32_t& minus) {
  if constexpr (DT == OC_F32) {
    const bool odd = (w & 0x7F800000u) == 0x7F800000u, nan = odd && (w << 9) != 0;
    fin = odd ? 0u : w;
    plus = odd && (nan || !(w >> 31)) ? 0x3F800000u : 0u;
    minus = odd && (nan || w >> 31) ? 0x3F800000u : 0u;
  } else {
    constexpr uint32_t E = DT == OC_BF16 ? 0x7F80u : 0x7C00u, ONE = DT == OC_BF16 ? 0x3F80u : 0x3C00u;
    fin = plus = minus = 0u;
#pragma unroll
    for (int k = 0; k < 32; k += 16) {
      const uint32_t v = (w >> k) & 0xFFFFu;
      const bool odd = (v & E) == E, nan = odd && (v & 0x7FFFu) != E;
      fin |= (odd ? 0u : v) << k;
      plus |= (odd && (nan || !(v >> 15)) ? ONE : 0u) << k;
      minus |= (odd && (nan || v >> 15) ? ONE : 0u) << k;
    }
  }
}

// pf_pv of a tile whose V holds infinities or NaN: a token of probability 0
// adds nothing, whatever its V.  The finite values are multiplied as ever; the
// same products with 1 in the place of what is not finite say which outputs
// have such a token among those of probability above 0, and get the infinity
// (two of different sign, or a NaN: NaN).
template <int DT, int D>
__device__ __forceinline__ void prompt_pv_any(f32x4 (&acc)[D / 16], const f32x4 (&c)[4], const char* svb, int lane) {
  const float inf = __builtin_inff();
#pragma unroll
  for (int nc = 0; nc < D / 16; ++nc) {
    int ln = lane;  // addresses formed here, not kept in registers over the column blocks
    asm volatile("" : "+v"(ln));
    const int x = ln & 15, kg = ln >> 4;
    f32x4 up = {0.f, 0.f, 0.f, 0.f}, down = {0.f, 0.f, 0.f, 0.f};
    if constexpr (DT == OC_F32) {
#pragma unroll
      for (int tb = 0; tb < 4; ++tb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = reinterpret_cast<const uint32_t*>(svb)[(16 * tb + 4 * kg + i) * D + 16 * nc + x];
          uint32_t fin, plus, minus;
          split_word<DT>(w, fin, plus, minus);
          acc[nc] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(fin), c[tb][i], acc[nc], 0, 0, 0);
          up = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(plus), c[tb][i], up, 0, 0, 0);
          down = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(minus), c[tb][i], down, 0, 0, 0);
        }
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // operands as in pf_pv
        uint32_t p[4], fin[4], plus[4], minus[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = pf_pack<DT>(c[2 * j + e / 2][2 * (e % 2)], c[2 * j + e / 2][2 * (e % 2) + 1]);
        const int vrow = 32 * j + 8 * kg + (x >> 2);
        const uint16_t* rowp = reinterpret_cast<const uint16_t*>(svb) + vrow * D + 4 * (x & 3) +
                               16 * (nc ^ PfTile<DT, D>::vswz(vrow));
        const u32x2 w0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                       (__attribute__((address_space(3))) s16x4*)rowp));
        const u32x2 w1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                       (__attribute__((address_space(3))) s16x4*)(rowp + 4 * D)));
        split_word<DT>(w0[0], fin[0], plus[0], minus[0]);
        split_word<DT>(w0[1], fin[1], plus[1], minus[1]);
        split_word<DT>(w1[0], fin[2], plus[2], minus[2]);
        split_word<DT>(w1[1], fin[3], plus[3], minus[3]);
        acc[nc] = mfma_qk<DT>(fin, p, acc[nc]);
        up = mfma_qk<DT>(plus, p, up);
        down = mfma_qk<DT>(minus, p, down);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      acc[nc][u] += up[u] > 0.f ? inf : 0.f;
      acc[nc][u] -= down[u] > 0.f ? inf : 0.f;
    }
    __builtin_amdgcn_sched_barrier(0);  // one column block at a time in registers
  }
}

// whether one of 16 bytes of type DT is infinite or NaN
template <int DT>
__device__ __forceinline__ bool not_finite(const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  constexpr uint32_t E = DT == OC_F32 ? 0x7F800000u : (DT == OC_BF16 ? 0x7F80u : 0x7C00u);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bad |= (w[i] & E) == E;
    if constexpr (DT != OC_F32) bad |= (w[i] >> 16 & E) == E;
  }
  return bad;
}

// A thread's part of the loads of pf_fetch_lds: its row and 16-byte piece of K
// and of V in the tile's first 512 pieces.  The others are whole rows of 512
// pieces further, in K and V as in LDS (the layouts repeat there), so that one
// offset each is all there is to keep.
template <int DT, int D>
struct PromptFetch {
  using L = PfTile<DT, D>;
  static constexpr int STEP = kPfThreads / L::LPT;  // rows per 512 pieces
  static_assert(L::NL == 1 || (STEP % 32 == 0 && STEP / L::RB % L::LPT == 0), "layouts that repeat every STEP rows");
  int k, v;

  __device__ static __forceinline__ PromptFetch of(const PrefillArgs& a, int tid) {
    const int r = (unsigned)tid / L::LPT, c = tid & (L::LPT - 1), swz = (unsigned)r / L::RB % L::LPT;
    return {r * (int)a.k_ss + 16 * (c ^ swz),
            DT == OC_F32 ? r * (int)a.v_ss + 16 * c : pf_vtok(r) * (int)a.v_ss + 16 * (c ^ (2 * L::vswz(r)))};
  }

  // n within 0 .. most, in scalar registers (the compiler's clamp is a vector instruction, and so then are the products)
  __device__ static __forceinline__ int rows_of(int n, int most) {
    n = min(n, most);
    asm("" : "+s"(n));
    return max(n, 0);
  }

  // tile t straight to LDS, rows at or past kv_len as zeros; by the first wave
  // the tile's documents too (past the last: 0, of places that no one sees)
  __device__ __forceinline__ void operator()(const PrefillArgs& a, const char* kh, const char* vh, const int32_t* docs,
                                             int t, int tid, char* nk, char* nv, int* nd) const {
    t = __builtin_amdgcn_readfirstlane(t);
    const int wbase = __builtin_amdgcn_readfirstlane(tid & ~63);
#pragma unroll
    for (int j = 0; j < L::NL; ++j) {
      const int row = 64 * t + STEP * j, n = rows_of(a.Skv - row, 64 - STEP * j);
      const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
          (void*)pf_uniform(kh + (int64_t)row * (int)a.k_ss), (short)0, __builtin_amdgcn_readfirstlane(n * (int)a.k_ss), 0x00020000);
      const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
          (void*)pf_uniform(vh + (int64_t)row * (int)a.v_ss), (short)0, __builtin_amdgcn_readfirstlane(n * (int)a.v_ss), 0x00020000);
      pf_load_lds16(rk, nk + 16 * (wbase + kPfThreads * j), k);
      pf_load_lds16(rv, nv + 16 * (wbase + kPfThreads * j), v);
    }
    if (docs && wbase == 0) {
      const __amdgpu_buffer_rsrc_t rd = __builtin_amdgcn_make_buffer_rsrc(
          (void*)pf_uniform((const char*)docs), (short)0, __builtin_amdgcn_readfirstlane(a.Skv * 4), 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rd, (__attribute__((address_space(3))) void*)nd, 4,
                                               4 * (64 * t + (int)__lane_id()), 0, 0, 0);
    }
  }
};

__device__ __forceinline__ int wave_min_i(int v) {
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ int wave_max_i(int v) {
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return v;
}

template <int DT, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(kPfThreads) __attribute__((amdgpu_waves_per_eu(DT == OC_F32 && D == 128 ? 1 : 4))) void prompt_kernel(
    const PromptArgs a) {
  using L = PfTile<DT, D>;
  // One LDS array for all: with several, the compiler takes the loads into one
  // stage for writes to the other, and waits for them before each tile's reads.
  // Behind the stages: the documents of the two stages' tokens and of the
  // workgroup's queries, their ranges, and the tile of each stage that holds V
  // values which are not finite.
  __shared__ __attribute__((aligned(16))) char sh[L::LDS + 4 * (2 * 64 + kPfRows + 4 * kPfWaves + 2)];
  int* const sdoc0 = reinterpret_cast<int*>(sh + L::LDS);
  int* const sqdoc = sdoc0 + 2 * 64;
  int* const swave = sqdoc + kPfRows;  // four of each wave: documents of its queries, and of the workgroup's
  int* const bad_tile = swave + 4 * kPfWaves;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // scalar: so are the tests of what the wave sees
  // (batch, head) pairs and query blocks as in the prefill kernel: an eighth
  // of the pairs per XCD, longest causal windows first
  const int nbh = a.B * a.Hq;
  const int i = blockIdx.x;
  int bh, e;
  if (nbh % 8 == 0) {
    const int hpx = nbh / 8, j = i / 8;
    bh = (i % 8) * hpx + j % hpx;
    e = j / hpx;
  } else {
    bh = i % nbh;
    e = i / nbh;
  }
  const int qb = a.qblocks - 1 - e;
  const int b = bh / a.Hq;
  const int h = bh % a.Hq;
  const int kv = h / a.G;
  const int pos0 = qb * kPfRows + 16 * wave;
  const int off = a.Skv - a.Sq;
  const int x = lane & 15;
  const int window = a.window > 0 ? a.window : INT_MAX;
  const int prefix = prefix_of(a.prefix, b, a.Skv);
  const int32_t* docs = a.docs ? a.docs + b * a.docs_sb : nullptr;
  auto doc_at = [&](int s) {  // the document of query s, -1 for none
    const int p = s + off;
    return s < a.Sq && p >= 0 ? docs[p] : -1;
  };
  if (docs) {
    // documents of the wave's queries, and of the workgroup's: the least and the most of those that are not negative
    const int doc = doc_at(pos0 + x);
    if (lane < 16) sqdoc[16 * wave + lane] = doc;  // read by this wave alone, like swave
    const int d0 = doc_at(qb * kPfRows + lane), d1 = doc_at(qb * kPfRows + 64 + lane);
    auto least = [](int d) { return d < 0 ? INT_MAX : d; };
    const int wd0 = wave_min_i(least(doc)), wd1 = wave_max_i(doc);
    const int gd0 = wave_min_i(min(least(d0), least(d1))), gd1 = wave_max_i(max(d0, d1));
    // (a wave with a query of no document is not of one document)
    const bool none = __builtin_amdgcn_ballot_w64(doc < 0 && pos0 + x < a.Sq) != 0;
    if (lane == 0) *reinterpret_cast<int4*>(swave + 4 * wave) = int4{wd0, none ? INT_MAX : wd1, gd0, gd1};
  }
  // places of the wave's first and last query, and of the workgroup's
  const int w_lo = pos0 + off, w_hi = min(pos0 + 15, a.Sq - 1) + off;
  const int g_lo = qb * kPfRows + off, g_hi = min(qb * kPfRows + kPfRows - 1, a.Sq - 1) + off;
  auto needed = [&](int t, int lo, int hi) {  // whether queries at places lo .. hi see a token of tile t
    return (64 * t <= hi && (window == INT_MAX || 64 * t + 63 > lo - window)) || 64 * t < prefix;
  };
  auto whole = [&](int t, int lo, int hi) {  // whether they all see all of it (documents apart)
    return 64 * t + 63 < a.Skv &&
           ((64 * t + 63 <= lo && (window == INT_MAX || hi - 64 * t < window)) || 64 * t + 63 < prefix);
  };
  const TileRange all = tile_range(g_lo, g_hi, window, prefix, a.Skv);
  int t_hi = all.hi;
  int t_lo = 0;
  if (a.shares > 1) {
    t_lo = all.lo + (int)blockIdx.y * a.share_tiles;
    t_hi = min(t_hi, t_lo + a.share_tiles);
    if (t_lo >= t_hi) return;  // nothing to see: the join counts on no such share
  }
  const bool active = pos0 < a.Sq;

  PrefillArgs pa;  // what the tile staging and the q load read
  pa.q_ss = a.q_ss, pa.Sq = a.Sq, pa.Skv = a.Skv, pa.k_ss = a.k_ss, pa.v_ss = a.v_ss;
  PfQ<DT, D> q;
  pf_load_q<DT, D>(pa, a.q + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh, pos0, lane, q);
  const char* kh = a.k + (int64_t)b * a.k_sb + (int64_t)kv * a.k_sh;
  const char* vh = a.v + (int64_t)b * a.v_sb + (int64_t)kv * a.v_sh;
  Change change = a.change;
  change.slope = BIAS ? a.slopes[h] * kLog2e / change.s : 0.f;

  // The tiles of the workgroup, 64 at a time, and what is true of each: that the
  // wave needs it, that all its queries see all of it (documents apart), that
  // its documents are all the wave's one document, and that some query of the
  // workgroup does not see all of it.
  int word = 0;
  uint64_t bits = 0, w_need = 0, w_whole = 0, w_one = 0, g_border = 0;
  auto load_word = [&](int w) {
    const auto ap = prompt_args();
    const int t = 64 * w + (int)__lane_id();
    bool keep = t < t_hi && needed(t, g_lo, g_hi);
    if (ap->evict) {
      const uint8_t* row = ap->evict + (int64_t)b * ap->e_sb + (int64_t)kv * ap->e_sh;
      keep = keep && !(t < ap->T && row[min(t, ap->T - 1)]);
    }
    bool one = true;
    if (docs) {
      const int last = (ap->Skv - 1) / 64;
      const int2 d = ap->ranges[(int64_t)b * (last + 1) + min(t, last)];
      const int4 q = *reinterpret_cast<const int4*>(swave + 4 * wave);
      keep = keep && d.y >= q.z && d.x <= q.w;
      one = d.x == d.y && d.x == q.x && d.x == q.y;
    }
    bits = __builtin_amdgcn_ballot_w64(keep);
    w_need = __builtin_amdgcn_ballot_w64(active && needed(t, w_lo, w_hi));
    w_whole = __builtin_amdgcn_ballot_w64(whole(t, w_lo, w_hi));
    w_one = __builtin_amdgcn_ballot_w64(one);
    g_border = __builtin_amdgcn_ballot_w64(docs || !whole(t, g_lo, g_hi));
  };
  struct Tile {
    int t;  // t_hi when there is none
    bool need, whole, one, border;
  };
  auto next_tile = [&]() {
    while (bits == 0) {
      if (64 * ++word >= t_hi) return Tile{t_hi, false, false, false, false};
      load_word(word);
    }
    const uint64_t b = bits & -bits;
    const Tile r{64 * word + __builtin_ctzll(bits), (w_need & b) != 0, (w_whole & b) != 0, (w_one & b) != 0, (g_border & b) != 0};
    bits &= bits - 1;
    return r;
  };

  PfState st;
  f32x4 accp[D / 16];
  auto stage_k = [&](int s) { return sh + s * 2 * L::KV; };
  auto stage_v = [&](int s) { return sh + s * 2 * L::KV + L::KV; };
  // One pass over the tiles.  The first takes V to be finite where it matters
  // and gives up (true) at the first border tile whose V is not; the second
  // then starts over with prompt_pv_any.  (Both forms of p.V in one loop need
  // more registers than two workgroups a CU leave.)
  auto pass = [&](auto any_c) -> bool {
    constexpr bool ANY = decltype(any_c)::value;
    word = t_lo / 64;
    bits = 0;
    if (t_lo < t_hi) load_word(word);
    bits &= ~0ull << (t_lo & 63);
    st = PfState{kNoScore, 0.f, 0.f, 0};
#pragma unroll
    for (int nc = 0; nc < D / 16; ++nc) accp[nc] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (tid < 2) bad_tile[tid] = -1;
    Tile cur = next_tile();
    __syncthreads();  // bad_tile
    if constexpr (L::STAGES == 2) {
      // what this thread staged of a border tile's V, looked at once its loads have landed
      auto landed = [&](const Tile& n, int s) {
        if (ANY || !n.border || n.t >= t_hi) return;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < L::NL; ++j)
          bad |= not_finite<DT>(*reinterpret_cast<const uint4*>(stage_v(s) + 16 * (tid + kPfThreads * j)));
        if (bad) bad_tile[s] = n.t;
      };
      const auto first = PromptFetch<DT, D>::of(pa, tid);
      if (cur.t < t_hi) first(pa, kh, vh, docs, cur.t, tid, stage_k(0), stage_v(0), sdoc0);
      __builtin_amdgcn_s_waitcnt(0);
      landed(cur, 0);
      int s = 0;
      // the stages are restrict parameters, as in the prefill kernel: no wait for
      // the loads into one before the reads of the other
      auto step = [&](const Tile& n, char* __restrict__ nk, char* __restrict__ nv, int* __restrict__ nd,
                      const char* __restrict__ ck, const char* __restrict__ cv, const int* __restrict__ cd) {
        if (n.t < t_hi) {
          if constexpr (CAP || BIAS) {
            int tf = tid;  // the offsets formed again: two registers less across the tile
            asm volatile("" : "+v"(tf));
            PromptFetch<DT, D>::of(pa, tf)(pa, kh, vh, docs, n.t, tid, nk, nv, nd);
          } else {
            first(pa, kh, vh, docs, n.t, tid, nk, nv, nd);
          }
        }
        if (__builtin_expect(cur.need, 1)) {
          f32x4 c[4];
          pf_logits<DT, D>(q, ck, lane, c);
          const Sight eye{w_lo, window, prefix, docs && !cur.one ? sqdoc + 16 * wave : nullptr, cd};
          prompt_softmax<DT, D, CAP, BIAS>(st, accp, c, change, eye, cur.t * 64, cur.whole && cur.one);
          if constexpr (ANY) prompt_pv_any<DT, D>(accp, c, cv, lane);
          else pf_pv<DT, D, false, true>(accp, c, cv, lane);
        }
      };
      while (cur.t < t_hi) {
        __syncthreads();  // stage s is complete; every wave is done with stage s ^ 1
        if (!ANY && cur.border && bad_tile[s] == cur.t) return true;  // (uniform; no load is in flight)
        const Tile n = next_tile();
        step(n, stage_k(1 - s), stage_v(1 - s), sdoc0 + 64 * (1 - s), stage_k(s), stage_v(s), sdoc0 + 64 * s);
        __builtin_amdgcn_s_waitcnt(0);
        s = 1 - s;
        landed(n, s);
        cur = n;
      }
    } else {
      // one stage (float32, head_dim 128): the next tile waits in registers
      PfStage<DT, D> reg;
      int dn = 0;
      auto fetch = [&](int t) {
        pf_fetch<DT, D>(pa, kh, vh, t, tid, reg);
        if (docs && wave == 0) dn = docs[min(64 * t + lane, a.Skv - 1)];
      };
      auto stash = [&](const Tile& n) {
        pf_stash<DT, D>(reg, tid, stage_k(0), stage_v(0));
        if (docs && wave == 0) sdoc0[lane] = dn;
        if (ANY || !n.border) return;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < L::NL; ++j) bad |= not_finite<DT>(reg.v[j]);
        if (bad) bad_tile[0] = n.t;
      };
      if (cur.t < t_hi) {
        fetch(cur.t);
        stash(cur);
      }
      while (cur.t < t_hi) {
        __syncthreads();  // the stage is complete
        if (!ANY && cur.border && bad_tile[0] == cur.t) return true;
        const Tile n = next_tile();
        if (n.t < t_hi) fetch(n.t);  // in flight during this tile
        if (__builtin_expect(cur.need, 1)) {
          f32x4 c[4];
          pf_logits<DT, D>(q, stage_k(0), lane, c);
          const Sight eye{w_lo, window, prefix, docs && !cur.one ? sqdoc + 16 * wave : nullptr, sdoc0};
          prompt_softmax<DT, D, CAP, BIAS>(st, accp, c, change, eye, cur.t * 64, cur.whole && cur.one);
          if constexpr (ANY) prompt_pv_any<DT, D>(accp, c, stage_v(0), lane);
          else pf_pv<DT, D, false, true>(accp, c, stage_v(0), lane);
        }
        __syncthreads();  // the stage is free again
        if (n.t < t_hi) stash(n);
        cur = n;
      }
    }
    return false;
  };
  if (pass(std::false_type{})) {
    __syncthreads();  // every wave has read bad_tile
    pass(std::true_type{});
  }

  // sums over the query's four lanes; lane 16r + x writes columns 16nc + 4r .. + 4 of query x
  float l = st.l;
  l += xpair<16>(l);
  l += xpair<32>(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  int tl = threadIdx.x;  // formed after the loop, as in the prefill kernel
  asm volatile("" : "+v"(tl));
  const int qpos = pos0 + (tl & 15), r = (tl >> 4) & 3;
  const auto ap = prompt_args();
  if (qpos >= ap->Sq) return;
  if (ap->shares > 1) {
    const int64_t row = (((int64_t)b * ap->Hq + h) * ap->Sq + qpos) * ap->shares + blockIdx.y;
    if (r == 0) ap->pm[row] = st.m, ap->pl[row] = l;
#pragma unroll
    for (int nc = 0; nc < D / 16; ++nc) *reinterpret_cast<f32x4*>(ap->pacc + row * D + 16 * nc + 4 * r) = accp[nc];
  } else {
    char* orow = ap->out + (int64_t)b * ap->o_sb + (int64_t)h * ap->o_sh + (int64_t)qpos * ap->o_ss;
#pragma unroll
    for (int nc = 0; nc < D / 16; ++nc) {
      const int col = 16 * nc + 4 * r;
      if constexpr (DT == OC_F32) {
        *reinterpret_cast<float4*>(orow + 4 * col) =
            float4{accp[nc][0] * inv, accp[nc][1] * inv, accp[nc][2] * inv, accp[nc][3] * inv};
      } else {
        const uint2 w = {pf_pack<DT>(accp[nc][0] * inv, accp[nc][1] * inv),
                         pf_pack<DT>(accp[nc][2] * inv, accp[nc][3] * inv)};
        if (ap->o_vec) {
          *reinterpret_cast<uint2*>(orow + 2 * col) = w;
        } else {
          uint16_t* o = reinterpret_cast<uint16_t*>(orow + 2 * col);
          o[0] = (uint16_t)w.x, o[1] = (uint16_t)(w.x >> 16);
          o[2] = (uint16_t)w.y, o[3] = (uint16_t)(w.y >> 16);
        }
      }
    }
  }
}

// Joins the shares of a query: out = sum w acc / sum w l with w = 2^(m - max m).
// D / 4 threads a query; a share in which it sees nothing has l = 0, and the
// shares behind its workgroup's last tile were not run.
template <int DT, int D>
__global__ __launch_bounds__(256) void prompt_join_kernel(const PromptArgs a) {
  constexpr int LANES = D / 4;
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (row >= (int64_t)a.B * a.Hq * a.Sq) return;
  const int col = 4 * (threadIdx.x % LANES);
  const int q = (int)(row % a.Sq), bh = (int)(row / a.Sq), b = bh / a.Hq, h = bh % a.Hq;
  const int first = q / kPfRows * kPfRows, off = a.Skv - a.Sq;
  const TileRange t = tile_range(first + off, min(first + kPfRows, a.Sq) - 1 + off, a.window > 0 ? a.window : INT_MAX,
                                 prefix_of(a.prefix, b, a.Skv), a.Skv);
  const int n = (max(t.hi - t.lo, 0) + a.share_tiles - 1) / a.share_tiles;
  const int64_t r = row * a.shares;
  float M = kNoScore, l = 0.f;
  for (int s = 0; s < n; ++s) M = fmaxf(M, a.pm[r + s]);
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < n; ++s) {
    const float w = __builtin_amdgcn_exp2f(a.pm[r + s] - M), ls = a.pl[r + s];
    if (ls == 0.f || (w == 0.f && ls == ls)) continue;  // (0 times an infinite sum; a NaN stays one)
    l += w * ls;
    x += w * *reinterpret_cast<const f32x4*>(a.pacc + (r + s) * D + col);
  }
  x *= l == 0.f ? 0.f : 1.f / l;
  char* o = a.out + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)q * a.o_ss;
  if constexpr (DT == OC_F32) {
    *reinterpret_cast<f32x4*>(o + 4 * col) = x;
  } else {
    const uint2 w = {pf_pack<DT>(x[0], x[1]), pf_pack<DT>(x[2], x[3])};
    uint16_t* o16 = reinterpret_cast<uint16_t*>(o) + col;
    if (a.o_vec) {
      *reinterpret_cast<uint2*>(o16) = w;
    } else {
      o16[0] = (uint16_t)w.x, o16[1] = (uint16_t)(w.x >> 16);
      o16[2] = (uint16_t)w.y, o16[3] = (uint16_t)(w.y >> 16);
    }
  }
}

template <int DT, int D>
void launch_prompt(const PromptArgs& a, unsigned blocks, hipStream_t s) {
  const bool cap = a.cap != 0, bias = a.slopes != nullptr;
  auto k = cap ? (bias ? prompt_kernel<DT, D, true, true> : prompt_kernel<DT, D, true, false>)
               : (bias ? prompt_kernel<DT, D, false, true> : prompt_kernel<DT, D, false, false>);
  hipLaunchKernelGGL(k, dim3(blocks, (unsigned)a.shares), dim3(kPfThreads), 0, s, a);
  if (a.shares > 1) {
    const int64_t rows = (int64_t)a.B * a.Hq * a.Sq, per = 256 / (D / 4);
    hipLaunchKernelGGL((prompt_join_kernel<DT, D>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s, a);
  }
}

template <int DT>
void launch_prompt_d(const PromptArgs& a, int d, unsigned blocks, hipStream_t s) {
  if (d == 64) launch_prompt<DT, 64>(a, blocks, s);
  else launch_prompt<DT, 128>(a, blocks, s);
}

constexpr int kMaxKv = 1 << 24;  // distances are exact in float32 up to here

int check_prompt(const oc_attend_prompt_params* p) {
  if (!p) return fail(OC_ERR_INVALID, "NULL parameters");
  if (!paged_float(p->dtype)) return fail(OC_ERR_INVALID, "dtype %d", p->dtype);
  if (p->head_dim != 64 && p->head_dim != 128) return fail(OC_ERR_UNSUPPORTED, "head_dim %d (64 or 128)", p->head_dim);
  if (p->batch < 0 || p->num_q_heads < 0 || p->num_kv_heads < 0 || p->q_len < 0 || p->kv_len < 0)
    return fail(OC_ERR_INVALID, "bad sizes");
  if (p->num_q_heads && (!p->num_kv_heads || p->num_q_heads % p->num_kv_heads))
    return fail(OC_ERR_INVALID, "%d query heads on %d kv heads", p->num_q_heads, p->num_kv_heads);
  if (p->kv_len > kMaxKv || p->q_len > kMaxKv) return fail(OC_ERR_UNSUPPORTED, "over 2^24 tokens");
  return check_mods(&p->mods);
}

Change change_of(float scale, float cap) {
  Change c{};
  c.pre = scale * kLog2e * (cap > 0.f ? kTanh0 : 1.f);
  c.s = c.pre < kSmallest ? 1.f : c.pre;
  if (cap > 0.f) {
    const float ratio = scale / cap, k = std::fabs(ratio) < kNoCap ? 0.f : ratio, k2 = k * k;
    c.k = k;
    c.inv = 1.f / (kTanh0 * k);
    c.lim = k2 * k2 < 1e30f ? kTanhFit / std::fabs(k) : -1.f;  // (k^4 has to be finite)
    c.b1 = kTanh1 / kTanh0 * k2;
    c.b2 = kTanh2 / kTanh0 * k2 * k2;
  }
  return c;
}

// With few queries the CUs stand idle while one workgroup after the other goes
// through a long context alone: the tiles are then split over several, and
// prompt_join_kernel adds up their sums.  The shares would fill every CU with
// the workgroups it holds, and are of eight tiles or more (float32, whose tiles
// take longer: four).  Each costs its sums, written and read, and the join a
// launch, so a call is split where by these times (of a tile, in ns; two
// workgroups on one CU take 0.9 of twice as long) it ends sooner.  Measured on
// 256 CUs, one pass against shares, bf16 / f16, head_dim 128: 16 queries on
// 32768 tokens (32 heads) 577 and 59 us, 128 on 4096 103 and 34, 512 on 4096
// 101 and 59, 8 heads of 1024 / 2048 / 4096 tokens 30 and 24, 52 and 40, 98
// and 79; float32, 4 heads of 1341 tokens, 183 and 57, 16 of 2048 299 and 195.
// Not split by the rule: 32 heads of 1024 (29, shares 39), 24 of 2560 (69,
// shares 83).
struct Shares {
  int tiles, n;  // tiles of each, and how many
};
Shares prompt_shares(const oc_attend_prompt_params* p) {
  const bool f32 = p->dtype == OC_F32, wide = p->head_dim == 128;
  const int64_t all = (p->kv_len + 63) / 64, blocks = (int64_t)p->batch * p->num_q_heads * ((p->q_len + kPfRows - 1) / kPfRows);
  // the most tiles that a workgroup sees, and those of one in the middle
  const int64_t most = p->mods.window > 0 && !p->mods.prefix_lens
                           ? std::min<int64_t>(all, ((int64_t)p->mods.window + kPfRows + 63) / 64 + 1) : all;
  const int64_t mean = std::min<int64_t>(most, (p->kv_len - std::min(p->q_len, p->kv_len) / 2 + 64) / 64);
  const int64_t cus = device_cus(), room = f32 && wide ? cus : 2 * cus;
  const int64_t tiles = std::max<int64_t>(f32 ? 4 : 8, (blocks * mean + room - 1) / room);
  if (blocks >= 2 * cus || 2 * most < 3 * tiles) return {0, 1};
  const double tile_ns = f32 ? (wide ? 9000 : 5000) : (wide ? 1500 : 1150);
  const double busy = 0.9 * blocks * mean / cus;  // tiles of a CU, if all had the same
  const double one = tile_ns * std::max<double>(most, busy);
  const double sums = (blocks * mean / (double)tiles + blocks / 2.) * kPfRows * p->head_dim * 8;
  const double split = tile_ns * std::max<double>(tiles, busy) + sums / 4900 + 4500;
  return split < one ? Shares{(int)tiles, (int)((most + tiles - 1) / tiles)} : Shares{0, 1};
}

// bytes of the documents' ranges, in the workspace before the shares' sums (which begin at a multiple of 16)
size_t range_bytes(const oc_attend_prompt_params* p) {
  return p->documents ? (size_t)p->batch * (size_t)((p->kv_len + 63) / 64) * sizeof(int2) : 0;
}

}  // namespace
}  // namespace oc

using namespace oc;

extern "C" size_t oc_attend_prompt_workspace_size(const oc_attend_prompt_params* p) {
  if (check_prompt(p) != OC_OK) return 0;
  const Shares n = prompt_shares(p);
  if (n.n == 1) return range_bytes(p);
  const size_t rows = (size_t)p->batch * p->num_q_heads * p->q_len * n.n;
  return (range_bytes(p) + 15) / 16 * 16 + (rows + 3) / 4 * 4 * 8 + rows * p->head_dim * 4;
}

extern "C" int oc_attend_prompt(const oc_attend_prompt_params* p, void* stream) {
  if (const int rc = check_prompt(p)) return rc;
  if (p->batch == 0 || p->num_q_heads == 0 || p->q_len == 0) return OC_OK;
  if (!p->q || !p->out || (p->kv_len && (!p->k || !p->v))) return fail(OC_ERR_INVALID, "NULL pointer");
  const int es = p->dtype == OC_F32 ? 4 : 2;
  for (const void* t : {p->q, p->k, p->v})
    if ((uintptr_t)t % 16) return fail(OC_ERR_INVALID, "q/k/v must be 16-byte aligned");
  for (int64_t st : {p->q_stride_b, p->q_stride_h, p->q_stride_s, p->k_stride_b, p->k_stride_h, p->k_stride_s,
                     p->v_stride_b, p->v_stride_h, p->v_stride_s})
    if ((st * es) % 16) return fail(OC_ERR_INVALID, "q/k/v strides must be multiples of 16 bytes");
  if (p->dtype == OC_F32)
    for (int64_t st : {(int64_t)(uintptr_t)p->out, p->out_stride_b * es, p->out_stride_h * es, p->out_stride_s * es})
      if (st % 16) return fail(OC_ERR_INVALID, "float32 out rows must be 16-byte aligned");
  if (p->k_stride_s * es * 64 > 0x7FFFFFFF || p->v_stride_s * es * 64 > 0x7FFFFFFF)
    return fail(OC_ERR_UNSUPPORTED, "token stride too large");
  if (p->kv_len && (p->k_stride_s < p->head_dim || p->v_stride_s < p->head_dim))
    return fail(OC_ERR_INVALID, "token stride smaller than head_dim");
  const size_t need = oc_attend_prompt_workspace_size(p);
  if (need && (!p->workspace || p->workspace_bytes < need))
    return fail(OC_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", p->workspace_bytes, need);
  if (need && (uintptr_t)p->workspace % 16) return fail(OC_ERR_INVALID, "the workspace must be 16-byte aligned");
  PromptArgs a{};
  a.q = (const char*)p->q, a.k = (const char*)p->k, a.v = (const char*)p->v, a.out = (char*)p->out;
  a.q_sb = p->q_stride_b * es, a.q_sh = p->q_stride_h * es, a.q_ss = p->q_stride_s * es;
  a.k_sb = p->k_stride_b * es, a.k_sh = p->k_stride_h * es, a.k_ss = p->k_stride_s * es;
  a.v_sb = p->v_stride_b * es, a.v_sh = p->v_stride_h * es, a.v_ss = p->v_stride_s * es;
  a.o_sb = p->out_stride_b * es, a.o_sh = p->out_stride_h * es, a.o_ss = p->out_stride_s * es;
  a.o_vec = ((uintptr_t)p->out | a.o_sb | a.o_sh | a.o_ss) % 8 == 0;
  a.B = p->batch, a.Hq = p->num_q_heads, a.Hkv = p->num_kv_heads, a.G = p->num_q_heads / p->num_kv_heads;
  a.Sq = p->q_len, a.Skv = p->kv_len, a.qblocks = (p->q_len + kPfRows - 1) / kPfRows;
  a.T = std::min(p->kv_len / 64, p->mods.evict ? p->mods.evict_cols : 0);
  a.docs = p->kv_len ? p->documents : nullptr, a.docs_sb = p->documents_stride_b, a.ranges = (const int2*)p->workspace;
  a.slopes = p->mods.slopes, a.prefix = p->mods.prefix_lens;
  a.evict = a.T > 0 ? p->mods.evict : nullptr, a.e_sb = p->mods.evict_stride_b, a.e_sh = p->mods.evict_stride_h;
  a.cap = p->mods.softcap > 0.f, a.window = p->mods.window;
  a.change = change_of(p->mods.scale, p->mods.softcap);
  const Shares shares = prompt_shares(p);
  a.shares = shares.n, a.share_tiles = shares.tiles;
  const size_t rows = ((size_t)p->batch * p->num_q_heads * p->q_len * shares.n + 3) / 4 * 4;
  a.pm = (float*)((char*)p->workspace + (range_bytes(p) + 15) / 16 * 16), a.pl = a.pm + rows, a.pacc = a.pl + rows;
  const int64_t blocks = (int64_t)p->batch * p->num_q_heads * a.qblocks;
  const int64_t tiles = (int64_t)p->batch * ((p->kv_len + 63) / 64);
  if (blocks > 0x7FFFFFFF || tiles > 0x7FFFFFFF || (int64_t)p->batch * p->num_q_heads > 0x7FFFFFFF)
    return fail(OC_ERR_UNSUPPORTED, "too many workgroups");
  const hipStream_t s = (hipStream_t)stream;
  if (a.docs)
    hipLaunchKernelGGL(doc_range_kernel, dim3((unsigned)((tiles + 3) / 4)), dim3(256), 0, s, a.docs, a.docs_sb, a.Skv,
                       (a.Skv + 63) / 64, (int)tiles, (int2*)p->workspace);
  if (p->dtype == OC_F32) launch_prompt_d<OC_F32>(a, p->head_dim, (unsigned)blocks, s);
  else if (p->dtype == OC_F16) launch_prompt_d<OC_F16>(a, p->head_dim, (unsigned)blocks, s);
  else launch_prompt_d<OC_BF16>(a, p->head_dim, (unsigned)blocks, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? OC_OK : hip_fail(e, "prompt launch");
}
