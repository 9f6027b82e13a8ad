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

constexpr int kPortWaves = 4;
constexpr int kPortThreads = kPortWaves * kWave;
constexpr int kPortHeads = 4;  // query heads of a workgroup

// The portable kernel: every head_dim (a multiple of 8 up to 512), block size
// and type.  A wave takes a tile: a lane per token forms the scores of four
// query heads, and then a lane per column adds up p.V token by token.
template <int CT>
__global__ __launch_bounds__(kPortThreads) void paged_portable_kernel(const PagedArgs a) {
  constexpr int ES = Elem<CT>::size;
  constexpr int NI = kPaMaxDim / kWave;
  __shared__ float sq[kPortHeads][kPaMaxDim];
  __shared__ float sp[kPortWaves][kPortHeads][kWave];
  __shared__ int64_t srow[kPortWaves][kWave];
  __shared__ float sacc[kPortHeads][kPaMaxDim];
  __shared__ float sm[kPortWaves][kPortHeads], sl[kPortWaves][kPortHeads];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunks = (a.G + kPortHeads - 1) / kPortHeads;
  const int b = blockIdx.z, kv = blockIdx.y / chunks, split = blockIdx.x;
  const int g0 = (blockIdx.y % chunks) * kPortHeads;
  const int ng = min(kPortHeads, a.G - g0);
  const int h0 = kv * a.G + g0;
  const Seen s = seen_of(a, b);
  const int qes = a.dtype == OC_F32 ? 4 : 2;
  for (int i = tid; i < ng * a.d; i += kPortThreads) {
    const int g = i / a.d, c = i - g * a.d;
    sq[g][c] = load_scalar(a.q + b * a.q_sb + (h0 + g) * a.q_sh + c * qes, a.dtype);
  }
  __syncthreads();
  const int32_t* row = a.tables + b * a.bt_stride;
  const uint8_t* ev = a.evict ? a.evict + b * a.e_sb + kv * a.e_sh : nullptr;
  float m[kPortHeads], l[kPortHeads], acc[kPortHeads][NI], slope2[kPortHeads];
#pragma unroll
  for (int g = 0; g < kPortHeads; ++g) {
    m[g] = kNoScore;
    l[g] = 0.f;
    slope2[g] = a.slopes && g < ng ? a.slopes[h0 + g] * kLog2e : 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) acc[g][i] = 0.f;
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
    float dot[kPortHeads] = {0.f, 0.f, 0.f, 0.f};
    if (ok) {
      const char* kp = a.k + id * a.k_sb + kv * a.k_sh + slot * a.k_ss;
      for (int c = 0; c < a.d; c += 8) {
        uint32_t w[2 * ES];
        if constexpr (ES == 1) {
          const uint2 u = *reinterpret_cast<const uint2*>(kp + c);
          w[0] = u.x, w[1] = u.y;
        } else {
#pragma unroll
          for (int u = 0; u < ES / 2; ++u) {
            const uint4 x = *reinterpret_cast<const uint4*>(kp + c * ES + 16 * u);
            w[4 * u] = x.x, w[4 * u + 1] = x.y, w[4 * u + 2] = x.z, w[4 * u + 3] = x.w;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float kf = elem<CT>(w, e);
#pragma unroll
          for (int g = 0; g < kPortHeads; ++g) dot[g] = __builtin_fmaf(sq[g][c + e], kf, dot[g]);
        }
      }
    }
    srow[wave][lane] = id * a.v_sb + slot * a.v_ss;
    uint64_t left = __builtin_amdgcn_ballot_w64(ok);
#pragma unroll
    for (int g = 0; g < kPortHeads; ++g) {
      float z = g < ng && ok ? changed(a, dot[g], slope2[g], dist) : -__builtin_inff();
      const float mt = fmaxf(m[g], wave_max(z));
      const float alpha = __builtin_amdgcn_exp2f(m[g] - mt);
      const float p = __builtin_amdgcn_exp2f(z - mt);
      l[g] = l[g] * alpha + wave_sum(p);
      m[g] = mt;
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[g][i] *= alpha;
      sp[wave][g][lane] = p;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    while (left) {
      const int u = __builtin_ctzll(left);
      left &= left - 1;
      const char* vp = a.v + kv * a.v_sh + srow[wave][u];
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int c = lane + 64 * i;
        if (c < a.d) {
          float vf;
          if constexpr (CT == OC_FP8_E4M3FN) {
            const uint32_t w[1] = {*reinterpret_cast<const uint8_t*>(vp + c)};
            vf = elem<CT>(w, 0);
          } else {
            vf = load_scalar(vp + c * ES, CT);
          }
#pragma unroll
          for (int g = 0; g < kPortHeads; ++g) acc[g][i] = __builtin_fmaf(sp[wave][g][u], vf, acc[g][i]);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  // join the waves, in their order
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
    if (wave == w) {
#pragma unroll
      for (int g = 0; g < kPortHeads; ++g) {
        const float f = __builtin_amdgcn_exp2f(m[g] - M[g]);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int c = lane + 64 * i;
          if (c < a.d) sacc[g][c] = (w ? sacc[g][c] : 0.f) + acc[g][i] * f;
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

// Joins the shares of one (sequence, query head): out = sum w acc / sum w l
// with w = 2^(m - max m).
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedArgs a) {
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int64_t r = ((int64_t)b * a.Hq + h) * a.P;
  float M = kNoScore, L = 0.f;
  for (int s = 0; s < a.P; ++s) M = fmaxf(M, a.pm[r + s]);
  for (int s = 0; s < a.P; ++s) L += a.pl[r + s] * __builtin_amdgcn_exp2f(a.pm[r + s] - M);
  const int es = a.dtype == OC_F32 ? 4 : 2;
  for (int c = tid; c < a.d; c += 256) {
    float x = 0.f;
    for (int s = 0; s < a.P; ++s) x += a.pacc[(r + s) * a.d + c] * __builtin_amdgcn_exp2f(a.pm[r + s] - M);
    store_scalar(a.out + b * a.o_sb + h * a.o_sh + c * es, a.dtype, L == 0.f ? 0.f : x * a.v_scale / L);
  }
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

// Shares of a sequence: about four workgroups per CU, at least four tiles each.
int paged_splits(const oc_attend_paged_params* p) {
  const int64_t tiles = ((int64_t)p->max_blocks * p->block_size + 63) / 64;
  if (p->num_splits > 0) return (int)std::max<int64_t>(1, std::min<int64_t>(p->num_splits, tiles));
  const int64_t g = p->num_q_heads / p->num_kv_heads;
  const int64_t blocks = (int64_t)p->num_seqs * p->num_kv_heads * ((g + kPortHeads - 1) / kPortHeads);
  return (int)std::max<int64_t>(1, std::min<int64_t>({4 * (int64_t)device_cus() / std::max<int64_t>(blocks, 1), tiles / 4, 1024}));
}

}  // namespace
}  // namespace oc

using namespace oc;

extern "C" size_t oc_attend_paged_workspace_size(const oc_attend_paged_params* p) {
  if (check_paged(p) != OC_OK || p->num_q_heads == 0 || p->num_seqs == 0) return 0;
  const int P = paged_splits(p);
  return P == 1 ? 0 : (size_t)p->num_seqs * p->num_q_heads * P * (p->head_dim + 2) * 4;
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
  a.pm = (float*)p->workspace, a.pl = a.pm + rows * a.P, a.pacc = a.pl + rows * a.P;
  const hipStream_t s = (hipStream_t)stream;
  const int chunks = (a.G + kPortHeads - 1) / kPortHeads;
  const dim3 grid((unsigned)a.P, (unsigned)(a.Hkv * chunks), (unsigned)a.n);
  switch (p->cache_dtype) {
    case OC_F32: hipLaunchKernelGGL(paged_portable_kernel<OC_F32>, grid, dim3(kPortThreads), 0, s, a); break;
    case OC_F16: hipLaunchKernelGGL(paged_portable_kernel<OC_F16>, grid, dim3(kPortThreads), 0, s, a); break;
    case OC_BF16: hipLaunchKernelGGL(paged_portable_kernel<OC_BF16>, grid, dim3(kPortThreads), 0, s, a); break;
    default: hipLaunchKernelGGL(paged_portable_kernel<OC_FP8_E4M3FN>, grid, dim3(kPortThreads), 0, s, a);
  }
  if (a.P > 1) hipLaunchKernelGGL(paged_join_kernel, dim3((unsigned)a.Hq, (unsigned)a.n), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? OC_OK : hip_fail(e, "paged attention launch");
}
