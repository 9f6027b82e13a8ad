// Rotary positions, on tensors and on the way into a paged cache (declared in
// include/orthocache_paged.h).
//
// A workgroup takes one or kRotTokens tokens.  It forms the sine and cosine of
// each (token, pair) once, into LDS, and turns every head's row with them: the
// 2 x 4 KiB that a token of 32 + 8 heads of 128 reads need 64 angles, not 2560.
// An angle n * f is formed in float64 and reduced there to turns in [-1/2,
// 1/2], so that far positions lose nothing; sine and cosine of the reduced
// angle are float32.  Each thread turns one vector of pairs at a time: 16 bytes
// of the first and of the second half of a row, or 16 bytes of interleaved
// pairs.  Bound by the bytes (one read, one write) but for few tokens, where
// the chain of dependent loads (sequence, length, block id) is what is left.
// Measured: 4096 tokens of 32 + 8 heads of 128 in bf16 14.9 us (84 MB, 5.6
// TB/s); the same heads into pages, 16 tokens 5.4 us, 4762 into fp8 32.5 us
// (137 MB, 4.2 TB/s; vector instructions fill over 80% of the cycles there).
#include <hip/hip_runtime.h>

#include <cmath>

#include "oc_kernels.h"
#include "oc_paged.h"
#include "oc_status.h"
#include "orthocache_hip.h"
#include "orthocache_paged.h"

namespace oc {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 4;     // tokens per workgroup where there are many
constexpr int kRotMaxDim = 512;

// N consecutive elements of type DT as float32 (16 bytes for the vector forms)
template <int DT, int N>
__device__ __forceinline__ void load_n(const char* p, float (&f)[N]) {
  if constexpr (N == 1) {
    f[0] = load_scalar(p, DT);
  } else if constexpr (N == 2) {
    f[0] = load_scalar(p, DT);
    f[1] = load_scalar(p + Elem<DT>::size, DT);
  } else {
    static_assert(N * Elem<DT>::size == 16, "16-byte vectors");
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = elem<DT>(w, i);
  }
}

// float32 -> fp8-e4m3fn byte, ties to even; beyond the largest value (448) the
// largest value, NaN stays NaN
__device__ __forceinline__ float fp8_clamp(float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); }

// A number that values are divided by, and its reciprocal (0: to be divided by
// as it is).
struct Divisor {
  float d, r;
  __device__ static Divisor one() { return {1.f, 1.f}; }
  static Divisor of(float d) {
    return {d, d >= 0x1p-60f && d <= 0x1p60f ? 1.f / d : 0.f};  // (so that no difference is lost below the normal numbers)
  }
};

// x / d as a product and its correction: with r = 1 / d rounded correctly, q =
// x r is within a step or two, q d - x is exact in an fma, and the correction's
// own error is far below half a step of the quotient.  Beyond 1000 (the store
// clamps at 448) q is held there, so that an infinite x stays one.  Four
// instructions in place of the division's dozen: 33.9 to 32.5 us for the 4762
// tokens.
__device__ __forceinline__ float fp8_quotient(float x, Divisor v) {
  if (v.r == 0.f) return x / v.d;
  const float q = __builtin_amdgcn_fmed3f(x * v.r, -1000.f, 1000.f);
  return __builtin_fmaf(-__builtin_fmaf(q, v.d, -x), v.r, q);
}

// N consecutive float32 values rounded to dtype; fp8 stores x / div
template <int N>
__device__ __forceinline__ void store_n(char* p, int dtype, Divisor div, const float (&f)[N]) {
  if (dtype == OC_FP8_E4M3FN) {
    if constexpr (N <= 2) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        p[i] = (char)(__builtin_amdgcn_cvt_pk_fp8_f32(fp8_clamp(fp8_quotient(f[i], div)), 0.f, 0, false) & 0xFF);
    } else {
      uint32_t w[N / 4];
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        int u = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_clamp(fp8_quotient(f[4 * i], div)), fp8_clamp(fp8_quotient(f[4 * i + 1], div)), 0, false);
        u = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_clamp(fp8_quotient(f[4 * i + 2], div)), fp8_clamp(fp8_quotient(f[4 * i + 3], div)), u, true);
        w[i] = (uint32_t)u;
      }
      if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = uint2{w[0], w[1]};
      else *reinterpret_cast<uint32_t*>(p) = w[0];
    }
  } else if constexpr (N <= 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) store_scalar(p + i * (dtype == OC_F32 ? 4 : 2), dtype, f[i]);
  } else if (dtype == OC_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(p + 4 * i) = float4{f[i], f[i + 1], f[i + 2], f[i + 3]};
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if (dtype == OC_BF16) w[i] = bf16_bits(f[2 * i]) | (bf16_bits(f[2 * i + 1]) << 16);
      else
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * i]) |
               ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * i + 1]) << 16);
    }
    if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = uint4{w[0], w[1], w[2], w[3]};
    else *reinterpret_cast<uint2*>(p) = uint2{w[0], w[1]};
  }
}

// The vectors of a row: first those of pairs, then those of columns copied.
// VEC: 16-byte vectors (8 or 4 elements), else single pairs and elements.
template <int DT, bool VEC, bool INTER>
struct RowVecs {
  static constexpr int ES = Elem<DT>::size;
  static constexpr int N = VEC ? 16 / ES : 1;
  static constexpr int NP = INTER && !VEC ? 2 : N;  // elements of an interleaved vector
  __device__ static int turned(int rot) { return INTER ? rot / NP : rot / 2 / N; }
  __device__ static int count(int rot, int d) { return turned(rot) + (d - rot) / N; }
};

// A vector on its way: read, then turned and stored.  Two are in flight per
// thread, so that a row of 16-byte vectors fills memory's latency like one of
// 32-byte pairs does.
template <int DT, bool VEC, bool INTER>
struct TurnVec {
  using R = RowVecs<DT, VEC, INTER>;
  float x0[R::NP], x1[INTER ? 1 : R::N];
  char* dst;        // of the row
  const float2* sc; // the token's (cos, sin) pairs
  Divisor div;
  int u, rot, dtype, es;

  // vector u of the row at src, into x0 and x1
  __device__ __forceinline__ void read(const char* src) {
    const int nt = R::turned(rot);
    if constexpr (INTER && !VEC) {
      if (u >= nt) {
        x0[0] = load_scalar(src + (rot + u - nt) * R::ES, DT);
        x0[1] = 0.f;
      } else {
        load_n<DT, 2>(src + 2 * u * R::ES, x0);
      }
    } else {
      load_n<DT, R::N>(src + (u >= nt ? rot + (u - nt) * R::N : u * R::N) * R::ES, x0);
      if constexpr (!INTER)
        if (u < nt) load_n<DT, R::N>(src + (rot / 2 + u * R::N) * R::ES, x1);
    }
  }

  __device__ __forceinline__ void finish() const {
    const int nt = R::turned(rot);
    if (u >= nt) {
      float o[R::N];
#pragma unroll
      for (int i = 0; i < R::N; ++i) o[i] = x0[i];
      store_n<R::N>(dst + (rot + (u - nt) * R::N) * es, dtype, div, o);
    } else if constexpr (INTER) {
      const int c = u * R::NP;
      float o[R::NP];
#pragma unroll
      for (int i = 0; i < R::NP / 2; ++i) {
        const float2 t = sc[c / 2 + i];
        o[2 * i] = x0[2 * i] * t.x - x0[2 * i + 1] * t.y;
        o[2 * i + 1] = x0[2 * i + 1] * t.x + x0[2 * i] * t.y;
      }
      store_n<R::NP>(dst + c * es, dtype, div, o);
    } else {
      const int c = u * R::N;
      float o0[R::N], o1[R::N];
#pragma unroll
      for (int i = 0; i < R::N; ++i) {
        const float2 t = sc[c + i];
        o0[i] = x0[i] * t.x - x1[i] * t.y;
        o1[i] = x1[i] * t.x + x0[i] * t.y;
      }
      store_n<R::N>(dst + c * es, dtype, div, o0);
      store_n<R::N>(dst + (rot / 2 + c) * es, dtype, div, o1);
    }
  }
};

// (cos, sin) of position n's pair, times scale; the angle in turns, float64
__device__ __forceinline__ float2 angle_of(int64_t n, double f, float scale, bool backward) {
  double t = (double)n * f * 0.15915494309189533577;  // 1 / (2 pi)
  t -= __builtin_rint(t);
  float s, c;
  sincospif(2.f * (float)t, &s, &c);
  return float2{c * scale, (backward ? -s : s) * scale};
}

__device__ __forceinline__ int64_t position_at(const void* p, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// Division of 0 <= n < 2^31 by a number fixed for the launch, as a high product
// and a shift (the compiler's own takes some 40 instructions, and a vector needs
// three: the 4762-token chunks into fp8 pages went from 36 to 33.5 us).
struct Div {
  uint32_t mul, shift;
  Div() = default;
  explicit Div(uint32_t d) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi(mul, (uint32_t)n) + (uint32_t)n) >> shift); }
};

// strides in bytes
struct RotArgs {
  const char* x[2];
  char* y[2];
  int64_t x_sb[2], x_sh[2], x_ss[2], y_sb[2], y_sh[2], y_ss[2];
  int32_t heads[2];
  int32_t batch, tokens, d, rot, backward, positions_64, per;  // per: tokens per workgroup
  const void* positions;
  int64_t pos_sb;
  const double* inv_freq;
  float scale;
  Div by_nu, by_rows, by_half;  // vectors of a row, rows of a token, pairs of a row
};

template <int DT, bool VEC, bool INTER>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(const RotArgs a) {
  using R = RowVecs<DT, VEC, INTER>;
  __shared__ float2 sc[kRotTokens][kRotMaxDim / 2];
  const int tid = threadIdx.x;
  const int h = a.rot / 2;
  const int64_t all = (int64_t)a.batch * a.tokens;
  const int64_t n0 = (int64_t)blockIdx.x * a.per;
  const int nt = (int)(all - n0 < a.per ? all - n0 : a.per);
  // the group's first token's batch element and place; the others follow
  const int b0 = (int)(n0 / a.tokens), s0 = (int)(n0 - (int64_t)b0 * a.tokens);
  auto place = [&](int t, int64_t& b, int64_t& s) {
    b = b0, s = s0 + t;
    while (s >= a.tokens) s -= a.tokens, ++b;
  };
  for (int i = tid; i < nt * h; i += kRotThreads) {
    const int t = a.by_half(i), f = i - t * h;
    int64_t b, s;
    place(t, b, s);
    sc[t][f] = angle_of(position_at(a.positions, a.positions_64, b * a.pos_sb + s), a.inv_freq[f], a.scale, a.backward);
  }
  __syncthreads();
  const int nu = R::count(a.rot, a.d);
  const int rows = a.heads[0] + a.heads[1], vecs = nt * rows * nu;
  auto read = [&](int i, TurnVec<DT, VEC, INTER>& v) {
    const int r = a.by_nu(i);
    v.u = i - r * nu;
    const int t = a.by_rows(r);
    int head = r - t * rows;
    const int w = head >= a.heads[0];
    if (w) head -= a.heads[0];
    int64_t b, s;
    place(t, b, s);
    v.dst = a.y[w] + b * a.y_sb[w] + head * a.y_sh[w] + s * a.y_ss[w];
    v.sc = sc[t], v.div = Divisor::one(), v.rot = a.rot, v.dtype = DT, v.es = R::ES;
    v.read(a.x[w] + b * a.x_sb[w] + head * a.x_sh[w] + s * a.x_ss[w]);
  };
  for (int i = tid; i < vecs; i += 2 * kRotThreads) {
    TurnVec<DT, VEC, INTER> v0, v1;
    const bool two = i + kRotThreads < vecs;
    read(i, v0);
    if (two) read(i + kRotThreads, v1);
    v0.finish();
    if (two) v1.finish();
  }
}

struct AppendArgs {
  const char *q, *k, *v;
  char *q_out, *kc, *vc;
  int64_t q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, o_ss, o_sh;  // bytes
  int64_t kc_sb, kc_sh, kc_ss, vc_sb, vc_sh, vc_ss;        // bytes
  int32_t cache_dtype, tokens, num_seqs, Hq, Hkv, d, rot, block_log2, max_blocks, positions_64, per;
  int64_t num_blocks;
  const int32_t* tables;
  int64_t bt_stride;
  const int32_t* lens;
  const int32_t* cu;
  const void* positions;
  const double* inv_freq;
  float scale;
  Divisor k_scale, v_scale;
  int32_t* error_flag;
  Div by_nu, by_nc, by_per, by_half;  // vectors of a turned row, of a copied one, of a token; pairs of a row
};

// The sequence of row `row`: the last b with cu[b] <= row, -1 where cu[0] > row.
// The wave's 64 lanes look at 64 entries at a time.
__device__ __forceinline__ int seq_of_row(const int32_t* cu, int num_seqs, int row, int lane) {
  int lo = 0, n = num_seqs;
  while (true) {
    const int step = (n + 63) / 64;
    const int at = lane * step;
    const uint64_t below = __builtin_amdgcn_ballot_w64(at < n && cu[lo + min(at, n - 1)] <= row);
    if (below == 0) return -1;
    const int c = __builtin_popcountll(below) - 1;
    lo += c * step;
    n = min(step, n - c * step);
    if (step == 1) return lo;
  }
}

template <int DT, bool VEC, bool INTER>
__global__ __launch_bounds__(kRotThreads) void append_kernel(const AppendArgs a) {
  using R = RowVecs<DT, VEC, INTER>;
  __shared__ float2 sc[kRotTokens][kRotMaxDim / 2];
  __shared__ int64_t pos[kRotTokens];
  __shared__ int64_t blk[kRotTokens];  // block id; -1: not stored, -2: no token
  __shared__ int slot[kRotTokens];
  static_assert(kRotTokens <= kRotThreads / kWave, "one wave finds each token's place");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n0 = blockIdx.x * a.per;
  const int nt = min(a.tokens - n0, a.per);
  if (wave < nt) {
    const int row = n0 + wave;
    int b = row;
    int64_t i = 0;
    bool real = true;
    if (a.cu) {
      b = seq_of_row(a.cu, a.num_seqs, row, lane);
      real = b >= 0 && row < a.cu[max(b, 0) + 1];
      b = max(b, 0);
      i = (int64_t)row - a.cu[b];
    }
    const int len = a.lens[b];
    real = real && len >= 0;
    int64_t id = -2, n = 0;
    if (real) {
      n = len + i;
      const int64_t col = n >> a.block_log2;
      id = -1;
      if (col < a.max_blocks) {
        const int64_t e = a.tables[b * a.bt_stride + col];
        if (e >= 0 && e < a.num_blocks) id = e;
      }
      if (id < 0 && a.error_flag && lane == 0) atomicOr(a.error_flag, 1);
    }
    if (lane == 0) {
      blk[wave] = id;
      slot[wave] = (int)(n & ((1 << a.block_log2) - 1));
      pos[wave] = a.positions ? position_at(a.positions, a.positions_64, row) : n;
    }
  }
  __syncthreads();
  const int h = a.rot / 2;
  for (int i = tid; i < nt * h; i += kRotThreads) {
    const int t = a.by_half(i), f = i - t * h;
    sc[t][f] = angle_of(pos[t], a.inv_freq[f], a.scale, false);
  }
  __syncthreads();
  const int nu = R::count(a.rot, a.d);   // vectors of a turned row; of a copied one (rotary_dim 0):
  const int nc = a.d / R::N;
  const int nq = a.Hq * nu, nk = a.Hkv * nu, nv = a.Hkv * nc;
  const int per = nq + nk + nv;
  const int es = a.cache_dtype == OC_F32 ? 4 : (a.cache_dtype == OC_FP8_E4M3FN ? 1 : 2);
  // vector i of the group's tokens; false where there is nothing to store
  auto read = [&](int i, TurnVec<DT, VEC, INTER>& v) {
    const int t = a.by_per(i);
    int j = i - t * per;
    const int64_t row = n0 + t;
    const int64_t id = blk[t];
    v.sc = sc[t], v.rot = a.rot;
    if (j < nq) {
      const int head = a.by_nu(j);
      v.u = j - head * nu;
      v.dst = a.q_out + row * a.o_ss + head * a.o_sh;
      if (id == -2) {  // no token: its queries are zeros
        const float z[1] = {0.f};
        for (int c = v.u; c < a.d; c += nu) store_n<1>(v.dst + c * R::ES, DT, Divisor::one(), z);
        return false;
      }
      v.div = Divisor::one(), v.dtype = DT, v.es = R::ES;
      v.read(a.q + row * a.q_ss + head * a.q_sh);
      return true;
    }
    if (id < 0) return false;
    j -= nq;
    v.dtype = a.cache_dtype, v.es = es;
    if (j < nk) {
      const int head = a.by_nu(j);
      v.u = j - head * nu, v.div = a.k_scale;
      v.dst = a.kc + id * a.kc_sb + head * a.kc_sh + slot[t] * a.kc_ss;
      v.read(a.k + row * a.k_ss + head * a.k_sh);
    } else {
      j -= nk;
      const int head = a.by_nc(j);
      v.u = j - head * nc, v.div = a.v_scale, v.rot = 0;
      v.dst = a.vc + id * a.vc_sb + head * a.vc_sh + slot[t] * a.vc_ss;
      v.read(a.v + row * a.v_ss + head * a.v_sh);
    }
    return true;
  };
  const int all = nt * per;
  for (int i = tid; i < all; i += 2 * kRotThreads) {
    TurnVec<DT, VEC, INTER> v0, v1;
    const bool one = read(i, v0);
    const bool two = i + kRotThreads < all && read(i + kRotThreads, v1);
    if (one) v0.finish();
    if (two) v1.finish();
  }
}

bool multiple(std::initializer_list<int64_t> v, int64_t of) {
  for (int64_t x : v)
    if (x % of) return false;
  return true;
}

// whether 16-byte vectors of the source type cover the pairs and the rest
bool whole_vecs(int dtype, int d, int rot, bool inter) {
  const int n = dtype == OC_F32 ? 4 : 8;
  return (inter ? rot % n == 0 : (rot / 2) % n == 0) && (d - rot) % n == 0 && d % n == 0;
}

// RowVecs' numbers of vectors, for the host
int row_vecs(int dtype, bool vec, bool inter, int rot, int d) {
  const int n = vec ? (dtype == OC_F32 ? 4 : 8) : 1;
  return (inter ? rot / (vec ? n : 2) : rot / 2 / n) + (d - rot) / n;
}

template <int DT, typename K1, typename K2, typename K3, typename K4, typename Args>
void launch4(bool vec, bool inter, K1 vh, K2 vi, K3 sh, K4 si, unsigned blocks, hipStream_t s, const Args& a) {
  if (vec && !inter) hipLaunchKernelGGL(vh, dim3(blocks), dim3(kRotThreads), 0, s, a);
  else if (vec) hipLaunchKernelGGL(vi, dim3(blocks), dim3(kRotThreads), 0, s, a);
  else if (!inter) hipLaunchKernelGGL(sh, dim3(blocks), dim3(kRotThreads), 0, s, a);
  else hipLaunchKernelGGL(si, dim3(blocks), dim3(kRotThreads), 0, s, a);
}

template <int DT>
void launch_rotary(bool vec, bool inter, unsigned blocks, hipStream_t s, const RotArgs& a) {
  launch4<DT>(vec, inter, rotary_kernel<DT, true, false>, rotary_kernel<DT, true, true>,
              rotary_kernel<DT, false, false>, rotary_kernel<DT, false, true>, blocks, s, a);
}

template <int DT>
void launch_append(bool vec, bool inter, unsigned blocks, hipStream_t s, const AppendArgs& a) {
  launch4<DT>(vec, inter, append_kernel<DT, true, false>, append_kernel<DT, true, true>,
              append_kernel<DT, false, false>, append_kernel<DT, false, true>, blocks, s, a);
}

// tokens per workgroup: kRotTokens once every CU has two workgroups of them
// (1, 2, 4 tokens: 40, 36, 33.5 us for 4762 into pages; 5.7, 6.2, 9.3 for 16)
int tokens_per_group(int64_t tokens) { return tokens >= (int64_t)2 * kRotTokens * device_cus() ? kRotTokens : 1; }

}  // namespace
}  // namespace oc

using namespace oc;

extern "C" int oc_apply_rotary(const oc_rotary_params* p, void* stream) {
  if (!p) return fail(OC_ERR_INVALID, "NULL parameters");
  if (!paged_float(p->dtype)) return fail(OC_ERR_INVALID, "dtype %d", p->dtype);
  if (p->batch < 0 || p->tokens < 0 || p->heads[0] < 0 || p->heads[1] < 0 || p->head_dim < 1)
    return fail(OC_ERR_INVALID, "bad sizes");
  if (p->head_dim > kRotMaxDim) return fail(OC_ERR_UNSUPPORTED, "head_dim %d > %d", p->head_dim, kRotMaxDim);
  if (p->rotary_dim < 0 || p->rotary_dim > p->head_dim || p->rotary_dim % 2)
    return fail(OC_ERR_INVALID, "rotary_dim %d for head_dim %d (even, at most head_dim)", p->rotary_dim, p->head_dim);
  const int64_t all = (int64_t)p->batch * p->tokens;
  const int h1 = p->x[1] ? p->heads[1] : 0;
  if (all == 0 || p->heads[0] + h1 == 0) return OC_OK;
  if (!p->x[0] || !p->y[0] || (h1 && !p->y[1]) || (p->rotary_dim && (!p->inv_freq || !p->positions)))
    return fail(OC_ERR_INVALID, "NULL pointer");
  if ((int64_t)p->heads[0] + h1 > 65536) return fail(OC_ERR_UNSUPPORTED, "over 65536 heads");
  const int es = p->dtype == OC_F32 ? 4 : 2;
  RotArgs a{};
  bool vec = whole_vecs(p->dtype, p->head_dim, p->rotary_dim, p->interleaved != 0);
  for (int i = 0; i < 2; ++i) {
    if (i && !h1) break;
    a.x[i] = (const char*)p->x[i], a.y[i] = (char*)p->y[i];
    a.x_sb[i] = p->x_stride_b[i] * es, a.x_sh[i] = p->x_stride_h[i] * es, a.x_ss[i] = p->x_stride_s[i] * es;
    a.y_sb[i] = p->y_stride_b[i] * es, a.y_sh[i] = p->y_stride_h[i] * es, a.y_ss[i] = p->y_stride_s[i] * es;
    vec = vec && multiple({(int64_t)(uintptr_t)a.x[i], (int64_t)(uintptr_t)a.y[i], a.x_sb[i], a.x_sh[i], a.x_ss[i],
                           a.y_sb[i], a.y_sh[i], a.y_ss[i]}, 16);
  }
  a.heads[0] = p->heads[0], a.heads[1] = h1;
  a.batch = p->batch, a.tokens = p->tokens, a.d = p->head_dim, a.rot = p->rotary_dim, a.backward = p->backward != 0;
  a.positions = p->positions, a.positions_64 = p->positions_64, a.pos_sb = p->positions_stride_b;
  a.inv_freq = p->inv_freq, a.scale = p->scale;
  a.per = tokens_per_group(all);
  const int64_t blocks = (all + a.per - 1) / a.per;
  if (blocks > 0x7FFFFFFF) return fail(OC_ERR_UNSUPPORTED, "too many tokens");
  const bool inter = p->interleaved != 0;
  a.by_nu = Div(std::max(row_vecs(p->dtype, vec, inter, a.rot, a.d), 1));
  a.by_rows = Div(a.heads[0] + a.heads[1]), a.by_half = Div(std::max(a.rot / 2, 1));
  const hipStream_t s = (hipStream_t)stream;
  if (p->dtype == OC_F32) launch_rotary<OC_F32>(vec, inter, (unsigned)blocks, s, a);
  else if (p->dtype == OC_F16) launch_rotary<OC_F16>(vec, inter, (unsigned)blocks, s, a);
  else launch_rotary<OC_BF16>(vec, inter, (unsigned)blocks, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? OC_OK : hip_fail(e, "rotary launch");
}

extern "C" int oc_append_paged(const oc_append_params* p, void* stream) {
  if (!p) return fail(OC_ERR_INVALID, "NULL parameters");
  if (!paged_float(p->dtype)) return fail(OC_ERR_INVALID, "dtype %d", p->dtype);
  const int ces = paged_elem_size(p->cache_dtype);
  if (!ces) return fail(OC_ERR_INVALID, "cache dtype %d", p->cache_dtype);
  if (p->tokens < 0 || p->num_seqs < 0 || p->num_q_heads < 0 || p->num_kv_heads < 0 || p->head_dim < 1 ||
      p->max_blocks < 0 || p->num_blocks < 0)
    return fail(OC_ERR_INVALID, "bad sizes");
  if (p->head_dim > kRotMaxDim) return fail(OC_ERR_UNSUPPORTED, "head_dim %d > %d", p->head_dim, kRotMaxDim);
  const int rot = p->inv_freq ? p->rotary_dim : 0;
  if (rot < 0 || rot > p->head_dim || rot % 2)
    return fail(OC_ERR_INVALID, "rotary_dim %d for head_dim %d (even, at most head_dim)", rot, p->head_dim);
  const int bl = log2_exact(p->block_size);
  if (bl < 0) return fail(OC_ERR_INVALID, "block_size %d is not a power of two", p->block_size);
  if (!p->cu_seqlens && p->tokens != p->num_seqs)
    return fail(OC_ERR_INVALID, "%d tokens for %d sequences need cu_seqlens", p->tokens, p->num_seqs);
  if (p->tokens == 0 || p->num_seqs == 0 || p->num_q_heads + p->num_kv_heads == 0) return OC_OK;
  if ((int64_t)p->num_q_heads + 2 * (int64_t)p->num_kv_heads > 65536) return fail(OC_ERR_UNSUPPORTED, "over 65536 heads");
  const int hq = p->q ? p->num_q_heads : 0;
  if (!p->k || !p->v || !p->k_cache || !p->v_cache || !p->block_tables || !p->context_lens || (hq && !p->q_out))
    return fail(OC_ERR_INVALID, "NULL pointer");
  const int es = p->dtype == OC_F32 ? 4 : 2;
  AppendArgs a{};
  a.q = (const char*)p->q, a.k = (const char*)p->k, a.v = (const char*)p->v;
  a.q_out = (char*)p->q_out, a.kc = (char*)p->k_cache, a.vc = (char*)p->v_cache;
  a.q_ss = p->q_stride_s * es, a.q_sh = p->q_stride_h * es, a.k_ss = p->k_stride_s * es, a.k_sh = p->k_stride_h * es;
  a.v_ss = p->v_stride_s * es, a.v_sh = p->v_stride_h * es;
  a.o_ss = p->q_out_stride_s * es, a.o_sh = p->q_out_stride_h * es;
  a.kc_sb = p->k_cache_stride_b * ces, a.kc_sh = p->k_cache_stride_h * ces, a.kc_ss = p->k_cache_stride_s * ces;
  a.vc_sb = p->v_cache_stride_b * ces, a.vc_sh = p->v_cache_stride_h * ces, a.vc_ss = p->v_cache_stride_s * ces;
  a.cache_dtype = p->cache_dtype, a.tokens = p->tokens, a.num_seqs = p->num_seqs;
  a.Hq = hq, a.Hkv = p->num_kv_heads, a.d = p->head_dim, a.rot = rot, a.block_log2 = bl, a.max_blocks = p->max_blocks;
  a.positions = p->positions, a.positions_64 = p->positions_64, a.num_blocks = p->num_blocks;
  a.tables = p->block_tables, a.bt_stride = p->bt_stride, a.lens = p->context_lens, a.cu = p->cu_seqlens;
  a.inv_freq = p->inv_freq, a.scale = p->scale, a.k_scale = Divisor::of(p->k_scale), a.v_scale = Divisor::of(p->v_scale);
  a.error_flag = p->error_flag;
  // 16 bytes of the source; its vector in the cache's type is 8 ces (4 ces for float32) bytes, at most 16 a store
  const int cb = std::min(16, (16 / es) * ces);
  bool vec = whole_vecs(p->dtype, p->head_dim, rot, p->interleaved != 0) &&
             multiple({(int64_t)(uintptr_t)a.k, (int64_t)(uintptr_t)a.v, a.k_ss, a.k_sh, a.v_ss, a.v_sh}, 16) &&
             multiple({(int64_t)(uintptr_t)a.kc, (int64_t)(uintptr_t)a.vc, a.kc_sb, a.kc_sh, a.kc_ss, a.vc_sb, a.vc_sh,
                       a.vc_ss}, cb);
  if (hq)
    vec = vec && multiple({(int64_t)(uintptr_t)a.q, (int64_t)(uintptr_t)a.q_out, a.q_ss, a.q_sh, a.o_ss, a.o_sh}, 16);
  a.per = tokens_per_group(p->tokens);
  const unsigned blocks = (unsigned)((p->tokens + a.per - 1) / a.per);
  const bool inter = p->interleaved != 0;
  const int nu = row_vecs(p->dtype, vec, inter, rot, a.d), nc = row_vecs(p->dtype, vec, inter, 0, a.d);
  a.by_nu = Div(std::max(nu, 1)), a.by_nc = Div(nc), a.by_half = Div(std::max(rot / 2, 1));
  a.by_per = Div(std::max((a.Hq + a.Hkv) * nu + a.Hkv * nc, 1));
  const hipStream_t s = (hipStream_t)stream;
  if (p->dtype == OC_F32) launch_append<OC_F32>(vec, inter, blocks, s, a);
  else if (p->dtype == OC_F16) launch_append<OC_F16>(vec, inter, blocks, s, a);
  else launch_append<OC_BF16>(vec, inter, blocks, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? OC_OK : hip_fail(e, "append launch");
}

extern "C" void oc_paged_params_bytes(size_t sizes[6]) {
  sizes[0] = sizeof(oc_rotary_params);
  sizes[1] = sizeof(oc_append_params);
  sizes[2] = sizeof(oc_attend_paged_params);
  sizes[3] = sizeof(oc_attend_prompt_params);
  sizes[4] = sizeof(oc_fork_params);
  sizes[5] = sizeof(oc_evict_params);
}
