// Attention of one new token per sequence over a paged cache, with changed
// scores (declared in include/orthocache_paged.h): the tiles of a sequence that
// its token sees are split over workgroups, each walks its share once with the
// running maximum and sum of an online softmax, and a second kernel joins the
// shares.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>

#include "oc_kernels.h"
#include "oc_paged.h"
#include "oc_status.h"
#include "orthocache_hip.h"
#include "orthocache_paged.h"

namespace oc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoScore = -3e38f;  // the running maximum before the first score: below every finite one
constexpr int kPaMaxDim = 512;

struct PagedArgs {
  const char *q, *k, *v;
  char* out;
  int64_t q_sb, q_sh, o_sb, o_sh;                    // bytes
  int64_t k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;        // bytes (block, head, slot)
  const int32_t* tables;
  int64_t bt_stride, num_blocks;
  const int32_t* lens;
  int32_t max_blocks, block_log2, dtype, n, Hq, Hkv, G, d;
  const float* slopes;
  const int32_t* prefix;
  const uint8_t* evict;
  int64_t e_sb, e_sh;
  int32_t e_cols, window;     // window: INT_MAX without one
  float scale, cap, v_scale;  // scale: k_scale included
  int32_t P;
  int32_t* error_flag;
  float* pm;  // states of row b * Hq + h, share s: at row * P + s (base-2 units)
  float* pl;
  float* pacc;
};

// What the token of sequence b sees: tiles [0, pre) and [first, tiles), of L tokens.
struct Seen {
  int L, prefix, pre, first, tiles;
  __device__ __forceinline__ int count() const { return pre + tiles - first; }
  __device__ __forceinline__ int tile(int i) const { return i < pre ? i : first + i - pre; }
};

__device__ __forceinline__ Seen seen_of(const PagedArgs& a, int b) {
  Seen s;
  const int64_t cap = (int64_t)a.max_blocks << a.block_log2;
  const int n = a.lens[b];
  s.L = (int)(n < 0 ? 0 : n < cap ? n : cap);
  s.prefix = a.prefix ? min(max(a.prefix[b], 0), s.L) : 0;
  s.tiles = (s.L + 63) / 64;
  s.first = a.window < s.L ? (s.L - a.window) / 64 : 0;
  s.pre = min((s.prefix + 63) / 64, s.first);
  return s;
}

// the changed score, in base-2 units; dist = L - 1 - j
__device__ __forceinline__ float changed(const PagedArgs& a, float dot, float slope2, int dist) {
  float z = dot * a.scale;
  if (a.cap > 0.f) z = a.cap * tanhf(z / a.cap);
  return __builtin_fmaf(-slope2, (float)dist, z * kLog2e);
}

// W words from p, aligned to all of them up to 16 bytes
template <int W>
__device__ __forceinline__ void load_words(const char* p, uint32_t* w) {
  if constexpr (W % 4 == 0) {
#pragma unroll
    for (int u = 0; u < W; u += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(p + 4 * u);
      w[u] = x.x, w[u + 1] = x.y, w[u + 2] = x.z, w[u + 3] = x.w;
    }
  } else if constexpr (W == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
    static_assert(W == 1);
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// the value of lane 4 (lane / 4) + I
template <int I>
__device__ __forceinline__ int64_t quad_lane(int64_t v) {
  const int lo = __builtin_amdgcn_mov_dpp((int)v, 0x55 * I, 0xF, 0xF, true);
  const int hi = __builtin_amdgcn_mov_dpp((int)(v >> 32), 0x55 * I, 0xF, 0xF, true);
  return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}
// the sum over the four lanes of a quad, in each of them
__device__ __forceinline__ float quad_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, true));  // lanes 1 0 3 2
  return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, true));  // lanes 2 3 0 1
}

constexpr int kPortWaves = 4;
constexpr int kPortThreads = kPortWaves * kWave;
constexpr int kPortHeads = 4;  // query heads of a workgroup

// The portable kernel: every head_dim (a multiple of 8 up to 512), block size
// and type, four query heads a workgroup.  A wave takes a tile of 64 tokens.
// Scores: a quad of lanes per token, eight columns each of 32, in four rounds
// (a lane per token would read 64 rows at once, more than the L1 holds); then
// lane i has the scores of token i.  p.V: the tokens seen are put together in
// LDS, and a lane adds up four columns (twice four above head_dim 256) of every
// TP-th of them, TP as many rows as 64 lanes hold, VA rows of loads ahead.
// Bound by latency more than bytes: float32, 16 x 4096 tokens, 32 / 8 heads, 84
// us (4.3 TB/s); float32 queries on an fp8 cache, 5 x 94499 tokens, 48 us (2.2
// TB/s; 208 with a lane per token and one V row at a time).
template <int CT, int NI>
__global__ __launch_bounds__(kPortThreads) void paged_portable_kernel(const PagedArgs a) {
  constexpr int ES = Elem<CT>::size;
  constexpr int VW = ES;  // words of four values
  constexpr int DM = 256 * NI;
  constexpr int VA = NI == 1 ? 8 : 4;  // steps of loads ahead
  __shared__ __attribute__((aligned(16))) float sq[DM / 8 * 9][kPortHeads];
  __shared__ __attribute__((aligned(16))) float sp[kPortWaves][kWave][kPortHeads];
  __shared__ int64_t srow[kPortWaves][kWave];
  __shared__ float sacc[kPortHeads][DM];
  __shared__ float sm[kPortWaves][kPortHeads], sl[kPortWaves][kPortHeads];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int chunks = (a.G + kPortHeads - 1) / kPortHeads;
  const int b = blockIdx.z, kv = blockIdx.y / chunks, split = blockIdx.x;
  const int g0 = (blockIdx.y % chunks) * kPortHeads;
  const int ng = min(kPortHeads, a.G - g0);
  const int h0 = kv * a.G + g0;
  const Seen s = seen_of(a, b);
  const int qes = a.dtype == OC_F32 ? 4 : 2;
  // column c at row c + c / 8: the four lanes of a quad read in different banks; zeros up to a multiple of 32
  auto q_row = [](int c) { return c + (c >> 3); };
  const int dq = (a.d + 31) & ~31;
  for (int i = tid; i < kPortHeads * dq; i += kPortThreads) {
    const int g = i / dq, c = i - g * dq;
    sq[q_row(c)][g] = g < ng && c < a.d ? load_scalar(a.q + b * a.q_sb + (h0 + g) * a.q_sh + c * qes, a.dtype) : 0.f;
  }
  __syncthreads();
  const int32_t* row = a.tables + b * a.bt_stride;
  const uint8_t* ev = a.evict ? a.evict + b * a.e_sb + kv * a.e_sh : nullptr;
  // lanes of a V row (a power of two), and the lane's row and first column
  const int lpr = min(64, 1 << (32 - __builtin_clz((a.d + 3) / 4 - 1)));
  const int tp = 64 / lpr, mine = lane / lpr, col = 4 * (lane % lpr);
  const int part = 8 * (lane & 3);
  float m[kPortHeads], l[kPortHeads], acc[kPortHeads][NI][4], slope2[kPortHeads];
#pragma unroll
  for (int g = 0; g < kPortHeads; ++g) {
    m[g] = kNoScore;
    l[g] = 0.f;
    slope2[g] = a.slopes && g < ng ? a.slopes[h0 + g] * kLog2e : 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[g][i][e] = 0.f;
  }
  const int64_t all = s.count();
  const int lo = (int)(all * split / a.P), hi = (int)(all * (split + 1) / a.P);
  for (int i = lo + wave; i < hi; i += kPortWaves) {
    const int t = s.tile(i);
    if (ev && t < a.e_cols && t < s.L / 64 && ev[t]) continue;
    const int j = 64 * t + lane, dist = s.L - 1 - j;
    bool ok = dist >= 0 && (dist < a.window || j < s.prefix);
    int64_t id = -1;
    if (ok) {
      id = row[j >> a.block_log2];
      if (id < 0 || id >= a.num_blocks) {
        if (a.error_flag) atomicOr(a.error_flag, 1);
        ok = false;
      }
    }
    const int slot = j & ((1 << a.block_log2) - 1);
    const uint64_t seen = __builtin_amdgcn_ballot_w64(ok);
    if (!seen) continue;
    // K of token 4 quad + f in round f; of the tile's first token seen for those that are not
    int64_t ko = id * a.k_sb + slot * a.k_ss;
    const int one = __builtin_ctzll(seen);
    const int64_t ko1 = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(ko >> 32), one) << 32) |
                                  (uint32_t)__builtin_amdgcn_readlane((int)ko, one));
    if (!ok) ko = ko1;
    const char* kh = a.k + kv * a.k_sh;
    const char* kp[4] = {kh + quad_lane<0>(ko), kh + quad_lane<1>(ko), kh + quad_lane<2>(ko), kh + quad_lane<3>(ko)};
    float dots[4][kPortHeads] = {};
    uint32_t w[4][2 * ES];
#pragma unroll
    for (int f = 0; f < 4; ++f) load_words<2 * ES>(kp[f] + min(part, a.d - 8) * ES, w[f]);
    for (int c0 = 0; c0 < a.d; c0 += 32) {
      const int c = c0 + part;
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        if (c0 + 32 > a.d && c >= a.d) {
#pragma unroll
          for (int u = 0; u < 2 * ES; ++u) w[f][u] = 0;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float kf = elem<CT>(w[f], e);
          const float4 qv = *reinterpret_cast<const float4*>(sq[q_row(c) + e]);
          dots[f][0] = __builtin_fmaf(qv.x, kf, dots[f][0]);
          dots[f][1] = __builtin_fmaf(qv.y, kf, dots[f][1]);
          dots[f][2] = __builtin_fmaf(qv.z, kf, dots[f][2]);
          dots[f][3] = __builtin_fmaf(qv.w, kf, dots[f][3]);
        }
        load_words<2 * ES>(kp[f] + min(c + 32, a.d - 8) * ES, w[f]);  // (the last again rather than a branch)
      }
    }
    float dot[kPortHeads];
#pragma unroll
    for (int g = 0; g < kPortHeads; ++g) {
#pragma unroll
      for (int f = 0; f < 4; ++f) dots[f][g] = quad_sum(dots[f][g]);
      dot[g] = lane & 2 ? (lane & 1 ? dots[3][g] : dots[2][g]) : (lane & 1 ? dots[1][g] : dots[0][g]);
    }
    float p[kPortHeads];
#pragma unroll
    for (int g = 0; g < kPortHeads; ++g) {
      const float z = g < ng && ok ? changed(a, dot[g], slope2[g], dist) : -__builtin_inff();
      const float mt = fmaxf(m[g], wave_max(z));
      const float alpha = __builtin_amdgcn_exp2f(m[g] - mt);
      p[g] = __builtin_amdgcn_exp2f(z - mt);
      l[g] = l[g] * alpha + wave_sum(p[g]);
      m[g] = mt;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[g][i][e] *= alpha;
    }
    if (ok) {
      const int u = __builtin_popcountll(seen & ((1ull << lane) - 1));
      srow[wave][u] = id * a.v_sb + slot * a.v_ss;
      *reinterpret_cast<float4*>(sp[wave][u]) = float4{p[0], p[1], p[2], p[3]};
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const char* vh = a.v + kv * a.v_sh + col * ES;
    const int count = __builtin_popcountll(seen);
    for (int u0 = mine; u0 < count + mine; u0 += VA * tp) {  // (uniform: a lane's rows are u0, u0 + tp, ..)
      uint32_t w[VA][NI][VW];
#pragma unroll
      for (int f = 0; f < VA; ++f) {
        const int u = u0 + f * tp;
        const bool in = u < count;
        const char* vp = vh + srow[wave][in ? u : 0];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
#pragma unroll
          for (int e = 0; e < VW; ++e) w[f][i][e] = 0;
          if (in && col + 256 * i < a.d) load_words<VW>(vp + 256 * i * ES, w[f][i]);
        }
      }
#pragma unroll
      for (int f = 0; f < VA; ++f) {
        const int u = u0 + f * tp;
        const float4 pv = *reinterpret_cast<const float4*>(sp[wave][u < count ? u : 0]);  // (past the last: times 0)
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float vf = elem<CT>(w[f][i], e);
            acc[0][i][e] = __builtin_fmaf(pv.x, vf, acc[0][i][e]);
            acc[1][i][e] = __builtin_fmaf(pv.y, vf, acc[1][i][e]);
            acc[2][i][e] = __builtin_fmaf(pv.z, vf, acc[2][i][e]);
            acc[3][i][e] = __builtin_fmaf(pv.w, vf, acc[3][i][e]);
          }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  // join the wave's rows, then the waves, in their order
  for (int o = lpr; o < 64; o <<= 1)
#pragma unroll
    for (int g = 0; g < kPortHeads; ++g)
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[g][i][e] += __shfl_xor(acc[g][i][e], o, 64);
#pragma unroll
  for (int g = 0; g < kPortHeads; ++g)
    if (lane == 0) {
      sm[wave][g] = m[g];
      sl[wave][g] = l[g];
    }
  __syncthreads();
  float M[kPortHeads], L[kPortHeads];
#pragma unroll
  for (int g = 0; g < kPortHeads; ++g) {
    M[g] = kNoScore;
    L[g] = 0.f;
    for (int w = 0; w < kPortWaves; ++w) M[g] = fmaxf(M[g], sm[w][g]);
    for (int w = 0; w < kPortWaves; ++w) L[g] += sl[w][g] * __builtin_amdgcn_exp2f(sm[w][g] - M[g]);
  }
  for (int w = 0; w < kPortWaves; ++w) {
    if (wave == w && mine == 0) {
#pragma unroll
      for (int g = 0; g < kPortHeads; ++g) {
        const float f = __builtin_amdgcn_exp2f(m[g] - M[g]);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = col + 256 * i + e;
            if (c < a.d) sacc[g][c] = (w ? sacc[g][c] : 0.f) + acc[g][i][e] * f;
          }
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < ng * a.d; i += kPortThreads) {
    const int g = i / a.d, c = i - g * a.d;
    float Mg = M[0], Lg = L[0];
#pragma unroll
    for (int u = 1; u < kPortHeads; ++u)
      if (g == u) Mg = M[u], Lg = L[u];
    if (a.P == 1) {
      store_scalar(a.out + b * a.o_sb + (h0 + g) * a.o_sh + c * qes, a.dtype, Lg == 0.f ? 0.f : sacc[g][c] * a.v_scale / Lg);
    } else {
      const int64_t r = ((int64_t)b * a.Hq + h0 + g) * a.P + split;
      a.pacc[r * a.d + c] = sacc[g][c];
      if (c == 0) {
        a.pm[r] = Mg;
        a.pl[r] = Lg;
      }
    }
  }
}

// ------------------------------------------------------------ matrix cores
//
// 16-bit queries over a 16-bit or fp8 cache, head_dim 64, 128 or 256, blocks of
// 8 tokens or more.  A workgroup of four waves takes a share of one (sequence,
// kv head) for up to 16 query heads; a wave takes units of 32 tokens, K and V in
// registers, and asks for the next unit's K as soon as the scores have used this
// one's, for its V as soon as p.V has.  Nothing but the block ids goes through
// LDS:
//
//   S^T = K q^T, K as the A operand: row 4r + i of instruction tb is token 8r +
//   4tb + i, so lane (r, head) ends up with the scores of tokens 8r .. 8r + 7.
//   O^T += V^T P^T, V^T as the A operand: lane (kg, x) loads columns 8x .. 8x +
//   7 (4x .. at head_dim 64) of the tokens 8kg .. 8kg + 7, a whole row per 16
//   lanes, and instruction nc takes column 8x + nc of its eight tokens: the 8x8
//   block is turned in registers by one v_perm per two values.  P^T, the B
//   operand, is the lane's own eight probabilities.
//
// Bound by the bytes of K and V: a unit of 32 tokens of 128 columns is 16 KiB
// of loads to about 500 cycles of work.  Measured with the join: 16 sequences of
// up to 32768 tokens, 32 / 8 heads, bf16, 1.41 GB in 241 us (5.9 TB/s; the
// portable kernel 290); 4 of up to 131072, 64 / 8 heads, fp8, 0.84 GB in 153 us
// (5.5 TB/s; portable 379).

constexpr int kPmWaves = 4;
constexpr int kPmThreads = kPmWaves * kWave;
constexpr int kPmHeads = 16;
constexpr int kPmUnit = 32;
constexpr int kPmPages = kPmUnit / 8;  // blocks that a unit may touch

template <int CT, int D>
struct PmBuf {
  static constexpr bool F8 = CT == OC_FP8_E4M3FN;
  static constexpr int KW = D / 32 * (F8 ? 2 : 4);  // words of a token's K in a lane (its quarter of the columns)
  static constexpr int CPL = D == 64 ? 4 : 8;       // V columns of a lane's chunk
  static constexpr int CH = D / (16 * CPL);         // chunks of a lane
  static constexpr int VW = CPL * (F8 ? 1 : 2) / 4; // words of a chunk
  uint32_t k[2][KW];
  uint32_t v[8][CH][VW];
};

template <int W>
__device__ __forceinline__ void pm_load(const char* p, uint32_t* w) {
  typedef uint32_t v4u __attribute__((ext_vector_type(4)));
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  if constexpr (W == 4) {
    const v4u u = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(p));
    w[0] = u[0], w[1] = u[1], w[2] = u[2], w[3] = u[3];
  } else if constexpr (W == 2) {
    const v2u u = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(p));
    w[0] = u[0], w[1] = u[1];
  } else {
    w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
}

// two fp8 values (half h of word w) as a pair of the 16-bit type MT, exactly
template <int MT>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, bool high) {
  if constexpr (MT == OC_BF16)
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
  else
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
}

template <int MT>
__device__ __forceinline__ uint32_t pair16(float lo, float hi) {
  if constexpr (MT == OC_BF16) return bf16_bits(lo) | (bf16_bits(hi) << 16);
  else
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) |
           ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16);
}

template <int CT, int MT, int D>
__global__ __launch_bounds__(kPmThreads) __attribute__((amdgpu_waves_per_eu(D == 256 && CT != OC_FP8_E4M3FN ? 1 : 2))) void paged_mfma_kernel(
    const PagedArgs a) {
  using B = PmBuf<CT, D>;
  constexpr bool F8 = B::F8;
  constexpr int ES = F8 ? 1 : 2;
  __shared__ int sid[kPmWaves][kWave][kPmPages];
  __shared__ float sacc[kPmWaves][kPmHeads][D + 4];
  __shared__ float sm[kPmWaves][kPmHeads], sl[kPmWaves][kPmHeads];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int x = lane & 15, r = lane >> 4;
  const int chunks = (a.G + kPmHeads - 1) / kPmHeads;
  const int b = blockIdx.z, kv = blockIdx.y / chunks, split = blockIdx.x;
  const int g0 = (blockIdx.y % chunks) * kPmHeads;
  const int ng = min(kPmHeads, a.G - g0);
  const int h0 = kv * a.G + g0;
  const Seen s = seen_of(a, b);
  // q as the B operand: lane (kg = r, head x), columns q_col(kg, dc) .. + 8 for instruction dc
  uint32_t q[D / 32][4];
#pragma unroll
  for (int dc = 0; dc < D / 32; ++dc) {
    uint4 u = {0u, 0u, 0u, 0u};
    if (x < ng) u = *reinterpret_cast<const uint4*>(a.q + b * a.q_sb + (h0 + x) * a.q_sh + 2 * q_col<F8>(r, dc));
    q[dc][0] = u.x, q[dc][1] = u.y, q[dc][2] = u.z, q[dc][3] = u.w;
  }
  const float slope2 = a.slopes && x < ng ? a.slopes[h0 + x] * kLog2e : 0.f;
  const bool capped = a.cap > 0.f;
  // capped: z = cap - 2 cap / (1 + e^(2 s / cap)), all in base-2 units
  const float ex2 = capped ? 2.f * kLog2e * a.scale / a.cap : a.scale * kLog2e;
  const float cap2 = a.cap * kLog2e;

  const int32_t* row = a.tables + b * a.bt_stride;
  const uint8_t* ev = a.evict ? a.evict + b * a.e_sb + kv * a.e_sh : nullptr;
  const int bs = 1 << a.block_log2;
  const int64_t all = 2 * (int64_t)s.count();
  const int lo = (int)(all * split / a.P), hi = (int)(all * (split + 1) / a.P);

  // The wave's units lo + wave, + 4, ...: 64 at a time, a lane each finds its
  // unit's first token, whether anything of it is seen, and its block ids.
  int word = 0, first_tok = 0;  // first_tok: of this lane's unit of the word
  uint64_t bits = 0;
  auto load_word = [&]() {
    const int64_t i = lo + wave + (int64_t)kPmWaves * (64 * word + lane);
    bool keep = i < hi;
    int t0 = 0;
    if (keep) {
      const int t = s.tile((int)(i >> 1));
      t0 = 64 * t + 32 * (int)(i & 1);
      auto seen = [&](int from, int to) {  // any of the tokens from .. to - 1
        return from < s.L && (s.L - min(to, s.L) < a.window || from < s.prefix);
      };
      keep = seen(t0, t0 + kPmUnit) && !(ev && t < a.e_cols && t < s.L / 64 && ev[t]);
      if (keep) {
        const int step = min(bs, kPmUnit);
        int id = -1;
        for (int p = 0; p < kPmPages; ++p) {
          const int from = t0 + 8 * p;
          if (8 * p % step == 0) {
            id = -1;
            if (seen(from, from + step)) {
              id = row[from >> a.block_log2];
              if (id < 0 || id >= a.num_blocks) {
                if (a.error_flag) atomicOr(a.error_flag, 1);
                id = -1;
              }
            }
          }
          sid[wave][lane][p] = id;
        }
      }
    }
    first_tok = t0;
    bits = __builtin_amdgcn_ballot_w64(keep);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  const int nwords = hi > lo + wave ? (int)(((hi - lo - wave + kPmWaves - 1) / kPmWaves + 63) / 64) : 0;
  if (nwords) load_word();

  auto sees = [&](int j) { return j < s.L && (s.L - 1 - j < a.window || j < s.prefix); };
  // the unit at hand: its first token (-1: none), whether every token of it is
  // seen, the lane's blocks (of its K, and of its V and scores; -1: none)
  int tok0 = -1, ik = -1, iv = -1;
  bool full = false;
  auto next = [&]() {
    while (bits == 0) {
      if (++word >= nwords) {
        tok0 = -1;
        return;
      }
      load_word();
    }
    const int i = __builtin_ctzll(bits);
    bits &= bits - 1;
    tok0 = __builtin_amdgcn_readlane(first_tok, i);
    ik = sid[wave][i][x >> 2];
    iv = sid[wave][i][r];
    full = tok0 + kPmUnit <= s.L && (s.L - 1 - tok0 < a.window || tok0 + kPmUnit <= s.prefix) &&
           __builtin_amdgcn_ballot_w64(iv < 0) == 0;
  };
  B buf;
  auto load_k = [&]() {
    const char* base = a.k + (int64_t)ik * a.k_sb + (int64_t)kv * a.k_sh + 16 * r;
#pragma unroll
    for (int tb = 0; tb < 2; ++tb) {
      const int j = tok0 + 8 * (x >> 2) + 4 * tb + (x & 3);
      const char* p = base + (int64_t)(j & (bs - 1)) * a.k_ss;
      if (full || (ik >= 0 && sees(j))) {
#pragma unroll
        for (int w = 0; w < B::KW; w += 4) pm_load<4>(p + 16 * w, buf.k[tb] + w);
      } else {
#pragma unroll
        for (int w = 0; w < B::KW; ++w) buf.k[tb][w] = 0u;
      }
    }
  };
  auto load_v = [&]() {
    const char* base = a.v + (int64_t)iv * a.v_sb + (int64_t)kv * a.v_sh + B::CPL * ES * x;
    const int s0 = (tok0 + 8 * r) & (bs - 1);  // eight slots in a row
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const char* p = base + (int64_t)(s0 + t) * a.v_ss;
      if (full || (iv >= 0 && sees(tok0 + 8 * r + t))) {
#pragma unroll
        for (int c = 0; c < B::CH; ++c) pm_load<B::VW>(p + 16 * B::CPL * ES * c, buf.v[t][c]);
      } else {
#pragma unroll
        for (int c = 0; c < B::CH; ++c)
#pragma unroll
          for (int w = 0; w < B::VW; ++w) buf.v[t][c][w] = 0u;
      }
    }
  };

  float m = kNoScore, l = 0.f;
  f32x4 acc[D / 16];
#pragma unroll
  for (int nc = 0; nc < D / 16; ++nc) acc[nc] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (nwords) next();
  if (tok0 >= 0) {
    load_k();
    load_v();
  }
  while (tok0 >= 0) {
    f32x4 c[2];
#pragma unroll
    for (int tb = 0; tb < 2; ++tb) {
      c[tb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dc = 0; dc < D / 32; ++dc) {
        uint32_t kw[4];
        if constexpr (F8) {
#pragma unroll
          for (int w = 0; w < 4; ++w) kw[w] = fp8_pair<MT>(buf.k[tb][2 * dc + w / 2], w & 1);
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w) kw[w] = buf.k[tb][4 * dc + w];
        }
        c[tb] = mfma_qk<MT>(kw, q[dc], c[tb]);
      }
    }
    // the changed scores of tokens tok0 + 8 r + 4 tb + i
    const float d0 = (float)(s.L - 1 - tok0 - 8 * r);
    float mt = -__builtin_inff();
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float z = c[tb][i] * ex2;
        if (capped) z = __builtin_fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z)), cap2);
        z = __builtin_fmaf(-slope2, d0 - (float)(4 * tb + i), z);
        if (!full) z = iv >= 0 && sees(tok0 + 8 * r + 4 * tb + i) ? z : -__builtin_inff();
        c[tb][i] = z;
        mt = fmaxf(mt, z);
      }
    __builtin_amdgcn_sched_barrier(0);
    next();
    if (tok0 >= 0) load_k();
    __builtin_amdgcn_sched_barrier(0);
    mt = fmaxf(mt, xpair<16>(mt));
    mt = fmaxf(mt, xpair<32>(mt));
    // rescaled only once a head's maximum has passed its reference by 8: until
    // then its probabilities are at most 2^8, of the same relative precision
    const bool move = mt > m + 8.f;
    if (__builtin_amdgcn_ballot_w64(move)) {
      const float mn = move ? mt : m;
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int nc = 0; nc < D / 16; ++nc) acc[nc] *= alpha;
    }
    // p as a 16-bit part and the 16-bit rounding of the rest: the matrix cores
    // have time, and p keeps 16 bits and more
    uint32_t ph[4], pl[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float p0 = __builtin_amdgcn_exp2f(c[w / 2][2 * (w & 1)] - m);
      const float p1 = __builtin_amdgcn_exp2f(c[w / 2][2 * (w & 1) + 1] - m);
      l += p0 + p1;
      ph[w] = pair16<MT>(p0, p1);
      const uint32_t hw[1] = {ph[w]};
      pl[w] = pair16<MT>(p0 - elem<MT>(hw, 0), p1 - elem<MT>(hw, 1));
    }
#pragma unroll
    for (int ch = 0; ch < B::CH; ++ch)
#pragma unroll
      for (int cw = 0; cw < B::CPL / 2; ++cw) {  // two columns: word cw of the chunk's 16-bit values
        uint32_t v[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] = F8 ? fp8_pair<MT>(buf.v[t][ch][cw / 2], cw & 1) : buf.v[t][ch][cw % B::VW];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t w[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) w[t] = __builtin_amdgcn_perm(v[2 * t + 1], v[2 * t], e ? 0x07060302u : 0x05040100u);
          f32x4& o = acc[B::CPL * ch + 2 * cw + e];
          o = mfma_qk<MT>(w, ph, o);
          o = mfma_qk<MT>(w, pl, o);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    if (tok0 >= 0) load_v();
  }

  // join the four waves: row 4r + i of acc[nc] is lane 4r + i's column nc
  l += xpair<16>(l);
  l += xpair<32>(l);
  if (r == 0) {
    sm[wave][x] = m;
    sl[wave][x] = l;
  }
#pragma unroll
  for (int nc = 0; nc < D / 16; ++nc)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sacc[wave][x][16 * B::CPL * (nc / B::CPL) + B::CPL * (4 * r + i) + nc % B::CPL] = acc[nc][i];
  __syncthreads();
  for (int o = tid; o < ng * D; o += kPmThreads) {
    const int g = o / D, col = o % D;
    float M = kNoScore, L = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < kPmWaves; ++w) M = fmaxf(M, sm[w][g]);
#pragma unroll
    for (int w = 0; w < kPmWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w][g] - M);
      L = __builtin_fmaf(sl[w][g], f, L);
      v = __builtin_fmaf(sacc[w][g][col], f, v);
    }
    if (a.P == 1) {
      store_scalar(a.out + b * a.o_sb + (h0 + g) * a.o_sh + 2 * col, MT, L == 0.f ? 0.f : v * a.v_scale / L);
    } else {
      const int64_t rr = ((int64_t)b * a.Hq + h0 + g) * a.P + split;
      a.pacc[rr * D + col] = v;
      if (col == 0) {
        a.pm[rr] = M;
        a.pl[rr] = L;
      }
    }
  }
}

// Joins the shares of one (sequence, query head): out = sum w acc / sum w l
// with w = 2^(m - max m).  The weights are formed by all threads at once, then
// each group of d / 4 threads adds up every so manieth share, four loads at a
// time: one share after the other waits for memory as often as there are shares.
constexpr int kMaxSplits = 1024;
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedArgs a) {
  __shared__ float sw[kMaxSplits], sm[4], sl[4];
  __shared__ float4 sx[256];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = ((int64_t)b * a.Hq + h) * a.P;
  float M = kNoScore, L = 0.f;
  for (int s = tid; s < a.P; s += 256) M = fmaxf(M, a.pm[r + s]);
  M = wave_max(M);
  if (lane == 0) sm[wave] = M;
  __syncthreads();
  M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  for (int s = tid; s < a.P; s += 256) {
    const float w = __builtin_amdgcn_exp2f(a.pm[r + s] - M), l = a.pl[r + s];
    sw[s] = w;
    if (w != 0.f || l != l) L += l * w;  // (a NaN stays one)
  }
  L = wave_sum(L);
  if (lane == 0) sl[wave] = L;
  __syncthreads();
  L = (sl[0] + sl[1]) + (sl[2] + sl[3]);
  const int lanes = a.d / 4, groups = 256 / lanes, g = tid / lanes, c = 4 * (tid % lanes);
  float4 x = {0.f, 0.f, 0.f, 0.f};
  if (g < groups) {
    auto add = [&](float w, const float4& v) {
      if (w == 0.f) return;  // (0 times an infinite sum)
      x.x += w * v.x, x.y += w * v.y, x.z += w * v.z, x.w += w * v.w;
    };
    const float* p = a.pacc + r * a.d + c;
    int s = g;
    for (; s + 3 * groups < a.P; s += 4 * groups) {
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const float4*>(p + (int64_t)(s + u * groups) * a.d);
#pragma unroll
      for (int u = 0; u < 4; ++u) add(sw[s + u * groups], v[u]);
    }
    for (; s < a.P; s += groups) add(sw[s], *reinterpret_cast<const float4*>(p + (int64_t)s * a.d));
    sx[tid] = x;
  }
  __syncthreads();
  if (g > 0) return;
  for (int u = 1; u < groups; ++u) {
    const float4 v = sx[u * lanes + tid];
    x.x += v.x, x.y += v.y, x.z += v.z, x.w += v.w;
  }
  const int es = a.dtype == OC_F32 ? 4 : 2;
  const float f = L == 0.f ? 0.f : a.v_scale / L;
  char* o = a.out + b * a.o_sb + h * a.o_sh + c * es;
  const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) store_scalar(o + e * es, a.dtype, L == 0.f ? 0.f : y[e] * f);
}

int check_paged(const oc_attend_paged_params* p) {
  if (!p) return fail(OC_ERR_INVALID, "NULL parameters");
  if (!paged_float(p->dtype)) return fail(OC_ERR_INVALID, "dtype %d", p->dtype);
  if (p->cache_dtype != p->dtype && p->cache_dtype != OC_FP8_E4M3FN)
    return fail(OC_ERR_UNSUPPORTED, "cache dtype %d with queries of dtype %d", p->cache_dtype, p->dtype);
  if (p->num_seqs < 0 || p->num_q_heads < 0 || p->num_kv_heads < 0 || p->max_blocks < 0 || p->num_blocks < 0 ||
      p->num_splits < 0)
    return fail(OC_ERR_INVALID, "bad sizes");
  if (p->head_dim < 8 || p->head_dim % 8 || p->head_dim > kPaMaxDim)
    return fail(OC_ERR_UNSUPPORTED, "head_dim %d (a multiple of 8 up to %d)", p->head_dim, kPaMaxDim);
  if (p->num_q_heads && (!p->num_kv_heads || p->num_q_heads % p->num_kv_heads))
    return fail(OC_ERR_INVALID, "%d query heads on %d kv heads", p->num_q_heads, p->num_kv_heads);
  if (log2_exact(p->block_size) < 0) return fail(OC_ERR_INVALID, "block_size %d is not a power of two", p->block_size);
  if (((int64_t)p->max_blocks * p->block_size) > (1 << 24)) return fail(OC_ERR_UNSUPPORTED, "tables of over 2^24 tokens");
  if (p->num_seqs > 65535 || p->num_q_heads > 65535) return fail(OC_ERR_UNSUPPORTED, "over 65535 sequences or heads");
  if (p->num_splits > 65535) return fail(OC_ERR_UNSUPPORTED, "num_splits %d", p->num_splits);
  return check_mods(&p->mods);
}

// whether the matrix-core kernel takes the call: its shapes, and 16-byte vectors of q, K and V (V rows in lanes of
// 8 bytes at head_dim 64 and in fp8, which are aligned then too)
bool paged_tuned(const oc_attend_paged_params* p) {
  if (p->portable || p->dtype == OC_F32 || p->block_size < 8) return false;
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return false;
  const int ces = paged_elem_size(p->cache_dtype);
  for (int64_t x : {(int64_t)(uintptr_t)p->q, p->q_stride_b * 2, p->q_stride_h * 2, (int64_t)(uintptr_t)p->k,
                    (int64_t)(uintptr_t)p->v, p->k_stride_b * ces, p->k_stride_h * ces, p->k_stride_s * ces,
                    p->v_stride_b * ces, p->v_stride_h * ces, p->v_stride_s * ces})
    if (x % 16) return false;
  return true;
}

// Shares of a sequence: four workgroups per CU, of eight tiles or more (four
// while there is not one for every CU); eight per CU where that leaves 32 tiles
// each.  Measured on 256 CUs (bf16, head_dim
// 128, 8 kv heads; shares: us): 16 x 32768 tokens 8: 253, 16: 241, 32: 246; 128 x
// 4096 1: 246, 2: 239, 4: 242; 16 x 4096 4: 44, 8: 46, 16: 49; 4 x 8192 8: 31,
// 16: 26, 32: 30; 1 x 32768 32: 32, 64: 30, 128: 34; fp8, 4 x 131072 16: 165, 32:
// 154, 64: 154, 128: 171; 3 x 300 1: 9.4, 2: 11.4; f16, one kv head, 2 x 17782
// 34: 17.3, 69: 14.5.
int paged_splits(const oc_attend_paged_params* p) {
  const int64_t tiles = ((int64_t)p->max_blocks * p->block_size + 63) / 64;
  if (p->num_splits > 0) return (int)std::max<int64_t>(1, std::min<int64_t>({p->num_splits, tiles, kMaxSplits}));
  const int64_t g = p->num_q_heads / p->num_kv_heads;
  const int heads = paged_tuned(p) ? kPmHeads : kPortHeads;
  const int64_t blocks = (int64_t)p->num_seqs * p->num_kv_heads * ((g + heads - 1) / heads);
  const int64_t cus = device_cus(), b = std::max<int64_t>(blocks, 1), four = 4 * cus / b, eight = 8 * cus / b;
  const int64_t n = eight > 0 && tiles / eight >= 32 ? eight : std::min(four, std::max(tiles / 8, std::min(tiles / 4, cus / b)));
  return (int)std::max<int64_t>(1, std::min<int64_t>(n, kMaxSplits));
}

template <int CT>
void launch_portable(const PagedArgs& a, dim3 grid, hipStream_t s) {
  if (a.d <= 256) hipLaunchKernelGGL((paged_portable_kernel<CT, 1>), grid, dim3(kPortThreads), 0, s, a);
  else hipLaunchKernelGGL((paged_portable_kernel<CT, 2>), grid, dim3(kPortThreads), 0, s, a);
}

template <int CT, int MT>
void launch_paged_mfma(const PagedArgs& a, dim3 grid, hipStream_t s) {
  if (a.d == 64) hipLaunchKernelGGL((paged_mfma_kernel<CT, MT, 64>), grid, dim3(kPmThreads), 0, s, a);
  else if (a.d == 128) hipLaunchKernelGGL((paged_mfma_kernel<CT, MT, 128>), grid, dim3(kPmThreads), 0, s, a);
  else hipLaunchKernelGGL((paged_mfma_kernel<CT, MT, 256>), grid, dim3(kPmThreads), 0, s, a);
}

}  // namespace
}  // namespace oc

using namespace oc;

extern "C" size_t oc_attend_paged_workspace_size(const oc_attend_paged_params* p) {
  if (check_paged(p) != OC_OK || p->num_q_heads == 0 || p->num_seqs == 0) return 0;
  const int P = paged_splits(p);
  const size_t states = (size_t)p->num_seqs * p->num_q_heads * P;
  return P == 1 ? 0 : (states + 3) / 4 * 4 * 8 + states * p->head_dim * 4;
}

extern "C" int oc_attend_paged(const oc_attend_paged_params* p, void* stream) {
  if (const int rc = check_paged(p)) return rc;
  if (p->num_seqs == 0 || p->num_q_heads == 0) return OC_OK;
  if (!p->q || !p->k || !p->v || !p->out || !p->context_lens || (p->max_blocks && !p->block_tables))
    return fail(OC_ERR_INVALID, "NULL pointer");
  const int es = p->dtype == OC_F32 ? 4 : 2, ces = paged_elem_size(p->cache_dtype);
  // the portable kernel reads eight elements at a time
  const int al = std::min(16, 8 * ces);
  for (int64_t x : {(int64_t)(uintptr_t)p->k, (int64_t)(uintptr_t)p->v, p->k_stride_b * ces, p->k_stride_h * ces,
                    p->k_stride_s * ces, p->v_stride_b * ces, p->v_stride_h * ces, p->v_stride_s * ces})
    if (x % al) return fail(OC_ERR_INVALID, "cache rows must be %d-byte aligned", al);
  const size_t need = oc_attend_paged_workspace_size(p);
  if (need && (!p->workspace || p->workspace_bytes < need))
    return fail(OC_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", p->workspace_bytes, need);
  PagedArgs a{};
  a.q = (const char*)p->q, a.k = (const char*)p->k, a.v = (const char*)p->v, a.out = (char*)p->out;
  a.q_sb = p->q_stride_b * es, a.q_sh = p->q_stride_h * es, a.o_sb = p->out_stride_b * es, a.o_sh = p->out_stride_h * es;
  a.k_sb = p->k_stride_b * ces, a.k_sh = p->k_stride_h * ces, a.k_ss = p->k_stride_s * ces;
  a.v_sb = p->v_stride_b * ces, a.v_sh = p->v_stride_h * ces, a.v_ss = p->v_stride_s * ces;
  a.tables = p->block_tables, a.bt_stride = p->bt_stride, a.num_blocks = p->num_blocks, a.lens = p->context_lens;
  a.max_blocks = p->max_blocks, a.block_log2 = log2_exact(p->block_size), a.dtype = p->dtype;
  a.n = p->num_seqs, a.Hq = p->num_q_heads, a.Hkv = p->num_kv_heads, a.G = p->num_q_heads / p->num_kv_heads, a.d = p->head_dim;
  a.slopes = p->mods.slopes, a.prefix = p->mods.prefix_lens, a.evict = p->mods.evict, a.e_sb = p->mods.evict_stride_b;
  a.e_sh = p->mods.evict_stride_h, a.e_cols = p->mods.evict_cols, a.window = p->mods.window > 0 ? p->mods.window : INT_MAX;
  a.scale = p->mods.scale * p->k_scale, a.cap = p->mods.softcap, a.v_scale = p->v_scale;
  a.P = paged_splits(p), a.error_flag = p->error_flag;
  const int64_t rows = (int64_t)a.n * a.Hq;
  a.pm = (float*)p->workspace, a.pl = a.pm + (rows * a.P + 3) / 4 * 4, a.pacc = a.pl + (rows * a.P + 3) / 4 * 4;
  const hipStream_t s = (hipStream_t)stream;
  const bool tuned = paged_tuned(p);
  const int heads = tuned ? kPmHeads : kPortHeads;
  const int chunks = (a.G + heads - 1) / heads;
  const dim3 grid((unsigned)a.P, (unsigned)(a.Hkv * chunks), (unsigned)a.n);
  if (tuned) {
    if (p->cache_dtype == OC_BF16) launch_paged_mfma<OC_BF16, OC_BF16>(a, grid, s);
    else if (p->cache_dtype == OC_F16) launch_paged_mfma<OC_F16, OC_F16>(a, grid, s);
    else if (p->dtype == OC_BF16) launch_paged_mfma<OC_FP8_E4M3FN, OC_BF16>(a, grid, s);
    else launch_paged_mfma<OC_FP8_E4M3FN, OC_F16>(a, grid, s);
  } else switch (p->cache_dtype) {
    case OC_F32: launch_portable<OC_F32>(a, grid, s); break;
    case OC_F16: launch_portable<OC_F16>(a, grid, s); break;
    case OC_BF16: launch_portable<OC_BF16>(a, grid, s); break;
    default: launch_portable<OC_FP8_E4M3FN>(a, grid, s);
  }
  if (a.P > 1) hipLaunchKernelGGL(paged_join_kernel, dim3((unsigned)a.Hq, (unsigned)a.n), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? OC_OK : hip_fail(e, "paged attention launch");
}
