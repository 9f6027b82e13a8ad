// Operators on the block tables of a paged cache (declared in
// include/orthocache_paged.h): forking, ending and extending sequences, and
// taking evicted tiles out.
//
// Both work from the old tables to new ones, so a call can be repeated and
// needs no order among its workgroups but that of its two launches.  Block
// counts change by integer atomics, whose order does not matter; everything
// else is a prefix sum, so the result depends on the inputs alone.
//
// Small calls are two launches and a few dependent loads each: 8 beams of 700
// tokens 9.5 us (plan 4.5, rows 3.7), 8 x 4096 tokens with half the tiles out
// 9.7 (2.1 and 5.1), 256 x 32768 12.5 (2.2 and 10.6).  Copies run at memory's
// rate: 64 sequences' last blocks in 16 layers (132 MB) 36 us, 25 of them the
// copies (5.3 TB/s).
#include <hip/hip_runtime.h>

#include "oc_kernels.h"
#include "oc_paged.h"
#include "oc_status.h"
#include "orthocache_hip.h"
#include "orthocache_paged.h"

namespace oc {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;
constexpr int kMaxSeqs = 4096;   // sequences and children of a call (the plan's LDS arrays)
constexpr int kRowThreads = 256;
constexpr int kPagesTile = 64;
constexpr int kMaxBlockBytes = 1 << 30;  // of a block's rows: offsets of their units stay in 32 bits
constexpr int kMaxCols = 1 << 20, kMaxBlocks = 1 << 30;  // table columns and blocks: sums of them stay in 32 bits

// Exclusive prefix sum of x over the workgroup and its total; every thread
// calls it.  sh: one int per wave, free again after the next barrier.
template <int THREADS>
__device__ __forceinline__ int block_excl_scan(int x, int* sh, int& total) {
  constexpr int W = THREADS / kWave;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int incl = wave_incl_scan(x);
  __syncthreads();  // sh is free
  if (lane == 63) sh[wave] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int s = sh[w];
    before += w < wave ? s : 0;
    all += s;
  }
  total = all;
  return before + incl - x;
}

struct ForkArgs {
  char *kc, *vc;
  int64_t k_sl, k_sb, k_sh, k_ss, v_sl, v_sb, v_sh, v_ss;  // bytes
  int32_t layers, heads, row_bytes, block_log2;
  int32_t n_in, n_out, max_blocks, out_max_blocks;
  int64_t num_blocks;
  const int32_t* tables;
  int64_t bt_stride;
  const int32_t* lens;
  const int32_t* refs;
  const int32_t* parents;
  const int32_t* fresh;
  int32_t* out_tables;
  int64_t out_bt_stride;
  int32_t* out_lens;
  int32_t* out_refs;
  int32_t* status;
  // the plan, in the workspace
  int32_t* take;    // (n_out) first fresh block of the child among those taken
  int32_t* have;    // (n_out) blocks it takes from its parent; bit 30: its last block is copied
  int32_t* count;   // (n_in) children; bit 30: the first child keeps the last block
  int32_t* free;    // fresh blocks, lowest first
  int32_t* plan;    // 0: the call is carried out, else its status
  int32_t free_cap;
};
constexpr int kFlag = 1 << 30;

// sequence s's tokens, as far as its row holds them
__device__ __forceinline__ int64_t fork_len(const ForkArgs& a, int s) {
  const int64_t n = a.lens[s];
  return n > 0 ? n : 0;
}

// Workgroup 0 plans the call; the others copy the counts.  The plan: the
// number of children of every sequence and the first of them (LDS), which
// children need a copy, how many fresh blocks each takes, their prefix sum, and
// the first that many blocks that no one holds.
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(const ForkArgs a) {
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    for (int64_t i = (int64_t)(blockIdx.x - 1) * kPlanThreads + tid; i < a.num_blocks;
         i += (int64_t)(gridDim.x - 1) * kPlanThreads)
      a.out_refs[i] = a.refs[i];
    return;
  }
  __shared__ int kids[kMaxSeqs], first[kMaxSeqs];
  __shared__ int scan[kPlanWaves];
  __shared__ int bad;
  for (int s = tid; s < a.n_in; s += kPlanThreads) {
    kids[s] = 0;
    first[s] = a.n_out;
  }
  if (tid == 0) bad = 0;
  __syncthreads();
  for (int i = tid; i < a.n_out; i += kPlanThreads) {
    const int s = a.parents ? a.parents[i] : i;
    if (s < -1 || s >= a.n_in) {
      atomicOr(&bad, OC_PAGES_BAD_PARENT);
    } else if (s >= 0) {
      atomicAdd(&kids[s], 1);
      atomicMin(&first[s], i);
    }
  }
  __syncthreads();
  const int bs = 1 << a.block_log2;
  // the last block of a sequence that has one that is not full: kept by the
  // first child where no one else holds it
  for (int s = tid; s < a.n_in; s += kPlanThreads) {
    const int64_t n = fork_len(a, s);
    const int64_t full = n >> a.block_log2;
    int keep = 0;
    if (((n + bs - 1) >> a.block_log2) > a.max_blocks) {
      atomicOr(&bad, OC_PAGES_TOO_LONG);
    } else if (n & (bs - 1)) {
      const int id = a.tables[s * a.bt_stride + full];
      if (id < 0 || id >= a.num_blocks) atomicOr(&bad, OC_PAGES_BAD_BLOCK);
      else keep = a.refs[id] <= 1;
    }
    a.count[s] = kids[s] | (keep ? kFlag : 0);
    if (!keep) first[s] = -1;  // no child keeps it
  }
  __syncthreads();
  int64_t base = 0;
  for (int i0 = 0; i0 < a.n_out; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int need = 0;
    if (i < a.n_out) {
      const int s = a.parents ? a.parents[i] : i;
      int have = 0;
      if (s >= 0 && s < a.n_in) {
        const int64_t n = fork_len(a, s);
        const int64_t more = a.fresh ? max(a.fresh[i], 0) : 0;
        const int64_t blocks = (n + more + bs - 1) >> a.block_log2;
        if (blocks > a.out_max_blocks) {
          atomicOr(&bad, OC_PAGES_TOO_LONG);
        } else {
          const bool part = (n & (bs - 1)) != 0;
          const bool copy = part && first[s] != i;
          have = (int)(n >> a.block_log2) + (part && !copy);
          need = (int)blocks - have;
          if (copy) have |= kFlag;
        }
      }
      a.have[i] = have;
    }
    int total;
    const int before = block_excl_scan<kPlanThreads>(need, scan, total);
    if (i < a.n_out) a.take[i] = (int)(base + before);
    base += total;
    if (base > a.free_cap) break;  // (uniform) more than the pool holds
  }
  if (base > a.free_cap && tid == 0) atomicOr(&bad, OC_PAGES_NO_ROOM);
  __syncthreads();
  const int want = bad ? 0 : (int)base;
  // the first `want` blocks that no one holds, four entries a thread
  int found = 0;
  for (int64_t b0 = 0; b0 < a.num_blocks && found < want; b0 += 4 * kPlanThreads) {
    int n = 0;
    bool f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t b = b0 + 4 * tid + j;
      f[j] = b < a.num_blocks && a.refs[b] == 0;
      n += f[j];
    }
    int total;
    int at = found + block_excl_scan<kPlanThreads>(n, scan, total);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (f[j]) {
        if (at < want) a.free[at] = (int)(b0 + 4 * tid + j);
        ++at;
      }
    found += total;
  }
  if (tid == 0) *a.status = *a.plan = found < want ? bad | OC_PAGES_NO_ROOM : bad;
}

// Workgroups: n_out rows of the new tables, n_in old rows whose blocks change
// holders, then (child, layer, K or V) triples that copy a last block.
__global__ __launch_bounds__(kRowThreads) void fork_rows_kernel(const ForkArgs a) {
  const int tid = threadIdx.x;
  const bool ok = *a.plan == 0;
  const int bs = 1 << a.block_log2;
  int64_t g = blockIdx.x;
  if (g < a.n_out) {
    const int i = (int)g;
    const int s = ok ? (a.parents ? a.parents[i] : i) : -1;
    int32_t* row = a.out_tables + i * a.out_bt_stride;
    int64_t n = 0;
    int blocks = 0, have = 0, take = 0;
    if (s >= 0) {
      n = fork_len(a, s);
      have = a.have[i] & ~kFlag;
      take = a.take[i];
      const int64_t more = a.fresh ? max(a.fresh[i], 0) : 0;
      blocks = (int)((n + more + bs - 1) >> a.block_log2);
    }
    if (tid == 0) a.out_lens[i] = (int)n;
    for (int c = tid; c < a.out_max_blocks; c += kRowThreads) {
      int id = -1;
      if (c < have) {
        id = a.tables[s * a.bt_stride + c];
        if (id < 0 || id >= a.num_blocks) id = -1;  // the parent's row below says so
      } else if (c < blocks) {
        id = a.free[take + c - have];
        atomicAdd(a.out_refs + id, 1);
      }
      row[c] = id;
    }
    return;
  }
  if (!ok) return;
  g -= a.n_out;
  if (g < a.n_in) {
    // holders of an old row's blocks: one less, and one more for every child
    // that shares them (full blocks: every child; the last: its keeper)
    const int s = (int)g;
    const int64_t n = fork_len(a, s);
    const int64_t full = n >> a.block_log2;
    const int kids = a.count[s] & ~kFlag;
    const int last = (n & (bs - 1)) && (a.count[s] & kFlag) && kids > 0 ? 1 : 0;
    for (int c = tid; c < a.max_blocks; c += kRowThreads) {
      const int change = (c < full ? kids : c == full ? last : 0) - 1;
      const int id = a.tables[s * a.bt_stride + c];
      if (id < 0 || id >= a.num_blocks) {
        if (c < full) atomicOr(a.status, OC_PAGES_BAD_BLOCK);
      } else if (change != 0) {
        atomicAdd(a.out_refs + id, change);
      }
    }
    return;
  }
  g -= a.n_in;
  const int i = (int)(g / (2 * a.layers));
  const int layer = (int)(g % (2 * a.layers)) >> 1;
  const bool is_v = g & 1;
  if (!(a.have[i] & kFlag)) return;
  const int s = a.parents ? a.parents[i] : i;
  const int64_t n = fork_len(a, s);
  const int part = (int)(n & (bs - 1));
  const int64_t src = a.tables[s * a.bt_stride + (n >> a.block_log2)];
  const int64_t dst = a.free[a.take[i]];
  const int64_t sb = is_v ? a.v_sb : a.k_sb, sh = is_v ? a.v_sh : a.k_sh, ss = is_v ? a.v_ss : a.k_ss;
  char* pool = (is_v ? a.vc + layer * a.v_sl : a.kc + layer * a.k_sl);
  // rows of row_bytes, part of them a head, in units of 16 bytes where
  // everything is a multiple of that, else of one; eight units a thread are
  // read before the first is written
  auto copy = [&](auto unit) {
    using U = decltype(unit);
    constexpr int AHEAD = 8;
    const char* from = pool + src * sb;
    char* to = pool + dst * sb;
    const int upr = a.row_bytes / (int)sizeof(U);
    const int perhead = part * upr, all = a.heads * perhead;
    for (int u0 = tid; u0 < all; u0 += AHEAD * kRowThreads) {
      int64_t off[AHEAD];
      U w[AHEAD];
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        const int u = min(u0 + e * kRowThreads, all - 1);
        const int h = u / perhead, r = u - h * perhead;
        const int t = r / upr, c = r - t * upr;
        off[e] = h * sh + t * ss + c * (int64_t)sizeof(U);
        w[e] = *reinterpret_cast<const U*>(from + off[e]);
      }
#pragma unroll
      for (int e = 0; e < AHEAD; ++e)
        if (u0 + e * kRowThreads < all) *reinterpret_cast<U*>(to + off[e]) = w[e];
    }
  };
  const int64_t odd = (int64_t)(uintptr_t)pool | sb | sh | ss | a.row_bytes;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  if (odd % 16 == 0) copy(u32x4{});
  else copy(uint8_t{});
}

struct EvictArgs {
  int32_t n, heads, block_log2, max_blocks, cols, map_cols;
  int64_t num_blocks;
  const int32_t* tables;
  int64_t bt_stride;
  const int32_t* lens;
  const int32_t* refs;
  const uint8_t* evict;
  int64_t e_sb, e_sh;
  int32_t* out_tables;
  int64_t out_bt_stride;
  int32_t* out_lens;
  int32_t* out_refs;
  int32_t* tile_map;
  int32_t* status;
};

__global__ __launch_bounds__(kRowThreads) void evict_copy_kernel(const EvictArgs a) {
  for (int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; i < a.num_blocks;
       i += (int64_t)gridDim.x * kRowThreads)
    a.out_refs[i] = a.refs[i];
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
}

// One workgroup per sequence: a thread per tile, 256 tiles at a time; a prefix
// sum of the kept ones gives each its new place, and the thread writes the
// tile's blocks there.
__global__ __launch_bounds__(kRowThreads) void evict_rows_kernel(const EvictArgs a) {
  __shared__ int scan[kRowThreads / kWave];
  const int tid = threadIdx.x, s = blockIdx.x;
  const int64_t cap = (int64_t)a.max_blocks << a.block_log2;
  int64_t n = a.lens[s];
  n = n < 0 ? 0 : n < cap ? n : cap;
  const int bs = 1 << a.block_log2;
  const int per = kPagesTile >> a.block_log2;  // blocks of a tile
  const int blocks = (int)((n + bs - 1) >> a.block_log2);
  const int tiles = (int)((n + kPagesTile - 1) / kPagesTile);
  const int whole = (int)(n / kPagesTile);
  const int32_t* row = a.tables + s * a.bt_stride;
  int32_t* out = a.out_tables + s * a.out_bt_stride;
  int32_t* map = a.tile_map + (int64_t)s * a.map_cols;
  const uint8_t* e = a.evict + s * a.e_sb;
  int base = 0, left = 0;  // kept tiles so far; blocks written so far
  for (int t0 = 0; t0 < tiles; t0 += kRowThreads) {
    const int t = t0 + tid;
    // the tile's flags of every head and its first blocks, read at once
    const bool may = t < whole && t < a.cols;
    constexpr int HELD = 8;
    int ids[HELD];
#pragma unroll
    for (int j = 0; j < HELD; ++j) ids[j] = t < tiles && j < per && t * per + j < blocks ? row[t * per + j] : -1;
    bool gone = may;
    if (may)
      for (int h0 = 0; h0 < a.heads; h0 += HELD) {
        uint8_t f[HELD];
#pragma unroll
        for (int h = 0; h < HELD; ++h) f[h] = e[min(h0 + h, a.heads - 1) * a.e_sh + t];
#pragma unroll
        for (int h = 0; h < HELD; ++h) gone = gone && f[h] != 0;
      }
    const bool kept = t < tiles && !gone;
    int total;
    const int at = base + block_excl_scan<kRowThreads>(kept ? 1 : 0, scan, total);
    if (t < tiles) {
      if (kept) map[at] = t;
      auto put = [&](int j, int id) {
        const bool good = id >= 0 && id < a.num_blocks;
        if (!good) {
          atomicOr(a.status, OC_PAGES_BAD_BLOCK);
          id = -1;
        }
        if (kept) out[at * per + j] = id;
        else if (good) atomicAdd(a.out_refs + id, -1);
      };
#pragma unroll
      for (int j = 0; j < HELD; ++j)
        if (j < per && t * per + j < blocks) put(j, ids[j]);
      for (int j = HELD; j < per && t * per + j < blocks; ++j) put(j, row[t * per + j]);
    }
    base += total;
  }
  // the last kept tile may be partial; every one before it is whole
  left = blocks - (tiles - base) * per;
  for (int c = blocks + tid; c < a.max_blocks; c += kRowThreads) {  // given back
    const int id = row[c];
    if (id >= 0 && id < a.num_blocks) atomicAdd(a.out_refs + id, -1);
  }
  for (int c = left + tid; c < a.max_blocks; c += kRowThreads) out[c] = -1;
  for (int c = base + tid; c < a.map_cols; c += kRowThreads) map[c] = -1;
  if (tid == 0) a.out_lens[s] = (int)(n - (int64_t)(tiles - base) * kPagesTile);
}

int64_t fork_free_cap(const oc_fork_params* p) {
  // no child takes more than its row holds
  const int64_t rows = (int64_t)p->num_children * p->out_max_blocks;
  return std::min<int64_t>(rows, p->num_blocks);
}

int check_fork(const oc_fork_params* p) {
  if (!p) return fail(OC_ERR_INVALID, "NULL parameters");
  if (p->layers < 0 || p->num_kv_heads < 0 || p->head_dim < 0 || p->num_seqs < 0 || p->num_children < 0 ||
      p->max_blocks < 0 || p->out_max_blocks < 0 || p->num_blocks < 0)
    return fail(OC_ERR_INVALID, "bad sizes");
  if (p->num_seqs > kMaxSeqs || p->num_children > kMaxSeqs)
    return fail(OC_ERR_UNSUPPORTED, "%d sequences, %d children (at most %d)", p->num_seqs, p->num_children, kMaxSeqs);
  if (p->num_blocks > kMaxBlocks || p->max_blocks > kMaxCols || p->out_max_blocks > kMaxCols)
    return fail(OC_ERR_UNSUPPORTED, "over 2^30 blocks or 2^20 table columns");
  if (log2_exact(p->block_size) < 0) return fail(OC_ERR_INVALID, "block_size %d is not a power of two", p->block_size);
  if (!paged_elem_size(p->cache_dtype)) return fail(OC_ERR_INVALID, "cache dtype %d", p->cache_dtype);
  if ((__int128)p->num_kv_heads * p->head_dim * paged_elem_size(p->cache_dtype) * p->block_size > kMaxBlockBytes)
    return fail(OC_ERR_UNSUPPORTED, "blocks of over 2^30 bytes");
  if (!p->parents && p->num_children != p->num_seqs)
    return fail(OC_ERR_INVALID, "%d children of %d sequences need parents", p->num_children, p->num_seqs);
  return OC_OK;
}

}  // namespace
}  // namespace oc

using namespace oc;

extern "C" size_t oc_fork_pages_workspace_size(const oc_fork_params* p) {
  if (check_fork(p) != OC_OK) return 0;
  return 4 * (size_t)(2 * (int64_t)p->num_children + p->num_seqs + fork_free_cap(p) + 1);
}

extern "C" int oc_fork_pages(const oc_fork_params* p, void* stream) {
  if (const int rc = check_fork(p)) return rc;
  if (!p->status) return fail(OC_ERR_INVALID, "NULL pointer");
  if ((p->num_seqs && (!p->context_lens || (p->max_blocks && !p->block_tables))) || (p->num_blocks && (!p->ref_counts || !p->out_ref_counts)) ||
      (p->num_children && (!p->out_context_lens || (p->out_max_blocks && !p->out_block_tables))))
    return fail(OC_ERR_INVALID, "NULL pointer");
  if (p->layers && (!p->k_cache || !p->v_cache)) return fail(OC_ERR_INVALID, "NULL cache");
  if (!p->workspace || p->workspace_bytes < oc_fork_pages_workspace_size(p))
    return fail(OC_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", p->workspace_bytes, oc_fork_pages_workspace_size(p));
  const int es = paged_elem_size(p->cache_dtype);
  ForkArgs a{};
  a.kc = (char*)p->k_cache, a.vc = (char*)p->v_cache;
  a.k_sl = p->k_stride_l * es, a.k_sb = p->k_stride_b * es, a.k_sh = p->k_stride_h * es, a.k_ss = p->k_stride_s * es;
  a.v_sl = p->v_stride_l * es, a.v_sb = p->v_stride_b * es, a.v_sh = p->v_stride_h * es, a.v_ss = p->v_stride_s * es;
  a.layers = p->layers, a.heads = p->num_kv_heads, a.row_bytes = p->head_dim * es, a.block_log2 = log2_exact(p->block_size);
  a.n_in = p->num_seqs, a.n_out = p->num_children, a.max_blocks = p->max_blocks, a.out_max_blocks = p->out_max_blocks;
  a.num_blocks = p->num_blocks, a.tables = p->block_tables, a.bt_stride = p->bt_stride, a.lens = p->context_lens;
  a.refs = p->ref_counts, a.parents = p->parents, a.fresh = p->new_tokens;
  a.out_tables = p->out_block_tables, a.out_bt_stride = p->out_bt_stride, a.out_lens = p->out_context_lens;
  a.out_refs = p->out_ref_counts, a.status = p->status;
  a.plan = (int32_t*)p->workspace;
  a.take = a.plan + 1;
  a.have = a.take + p->num_children;
  a.count = a.have + p->num_children;
  a.free = a.count + p->num_seqs;
  a.free_cap = (int32_t)fork_free_cap(p);
  const int64_t copiers = std::min<int64_t>((p->num_blocks + kPlanThreads - 1) / kPlanThreads, 256);
  const int64_t blocks = (int64_t)p->num_children + p->num_seqs + 2 * (int64_t)p->num_children * p->layers;
  if (blocks > 0x7FFFFFFF) return fail(OC_ERR_UNSUPPORTED, "too many layers");
  const hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1 + (unsigned)copiers), dim3(kPlanThreads), 0, s, a);
  if (blocks) hipLaunchKernelGGL(fork_rows_kernel, dim3((unsigned)blocks), dim3(kRowThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? OC_OK : hip_fail(e, "fork launch");
}

extern "C" int oc_evict_pages(const oc_evict_params* p, void* stream) {
  if (!p) return fail(OC_ERR_INVALID, "NULL parameters");
  if (p->num_seqs < 0 || p->num_kv_heads < 1 || p->max_blocks < 0 || p->num_blocks < 0 || p->evict_cols < 0)
    return fail(OC_ERR_INVALID, "bad sizes");
  const int bl = log2_exact(p->block_size);
  if (bl < 0 || p->block_size > kPagesTile)
    return fail(OC_ERR_INVALID, "block_size %d does not divide a tile of %d tokens", p->block_size, kPagesTile);
  if (p->num_blocks > kMaxBlocks || p->max_blocks > kMaxCols)
    return fail(OC_ERR_UNSUPPORTED, "over 2^30 blocks or 2^20 table columns");
  const int64_t tiles = (((int64_t)p->max_blocks << bl) + kPagesTile - 1) / kPagesTile;
  if (p->tile_map_cols < tiles) return fail(OC_ERR_INVALID, "tile_map has %d columns, %lld needed", p->tile_map_cols, (long long)tiles);
  if (!p->status || (p->num_blocks && (!p->ref_counts || !p->out_ref_counts)) ||
      (p->num_seqs && (!p->context_lens || !p->out_context_lens ||
                       (p->max_blocks && (!p->block_tables || !p->out_block_tables || !p->tile_map)) ||
                       (p->evict_cols && !p->evict))))
    return fail(OC_ERR_INVALID, "NULL pointer");
  EvictArgs a{};
  a.n = p->num_seqs, a.heads = p->num_kv_heads, a.block_log2 = bl, a.max_blocks = p->max_blocks, a.cols = p->evict_cols;
  a.map_cols = p->tile_map_cols, a.num_blocks = p->num_blocks, a.tables = p->block_tables, a.bt_stride = p->bt_stride;
  a.lens = p->context_lens, a.refs = p->ref_counts, a.evict = p->evict, a.e_sb = p->evict_stride_b, a.e_sh = p->evict_stride_h;
  a.out_tables = p->out_block_tables, a.out_bt_stride = p->out_bt_stride, a.out_lens = p->out_context_lens;
  a.out_refs = p->out_ref_counts, a.tile_map = p->tile_map, a.status = p->status;
  const hipStream_t s = (hipStream_t)stream;
  const int64_t copiers = std::max<int64_t>(1, std::min<int64_t>((p->num_blocks + kRowThreads - 1) / kRowThreads, 1024));
  hipLaunchKernelGGL(evict_copy_kernel, dim3((unsigned)copiers), dim3(kRowThreads), 0, s, a);
  if (a.n) hipLaunchKernelGGL(evict_rows_kernel, dim3((unsigned)a.n), dim3(kRowThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? OC_OK : hip_fail(e, "evict launch");
}
