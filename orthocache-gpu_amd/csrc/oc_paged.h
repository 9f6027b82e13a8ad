#pragma once
// Small host helpers shared by the operators of include/orthocache_paged.h.
#include <algorithm>
#include <initializer_list>

#include <cmath>

#include "oc_status.h"
#include "orthocache_hip.h"
#include "orthocache_paged.h"

namespace oc {

inline bool paged_float(int dt) { return dt == OC_F32 || dt == OC_F16 || dt == OC_BF16; }

inline int paged_elem_size(int dt) {
  return dt == OC_F32 ? 4 : dt == OC_F16 || dt == OC_BF16 ? 2 : dt == OC_FP8_E4M3FN ? 1 : 0;
}

// log2 of a power of two, -1 for any other number
inline int log2_exact(int n) {
  if (n <= 0 || (n & (n - 1))) return -1;
  return __builtin_ctz((unsigned)n);
}

// what every kind of changed scores has to satisfy
inline int check_mods(const oc_score_mods* m) {
  if (!std::isfinite(m->scale)) return fail(OC_ERR_INVALID, "scale %g", (double)m->scale);
  if (!(m->softcap >= 0.f) || !std::isfinite(m->softcap)) return fail(OC_ERR_INVALID, "softcap %g", (double)m->softcap);
  if (m->softcap > 0.f && !std::isfinite(m->scale / m->softcap))
    return fail(OC_ERR_INVALID, "scale %g over softcap %g", (double)m->scale, (double)m->softcap);
  if (m->window < 0) return fail(OC_ERR_INVALID, "window %d", m->window);
  if (m->evict && m->evict_cols < 0) return fail(OC_ERR_INVALID, "evict_cols %d", m->evict_cols);
  return OC_OK;
}

}  // namespace oc
