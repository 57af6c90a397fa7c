// Host checks of a page pool, shared by its entry points.
#pragma once

#include "si_common.h"

namespace si {

inline int check_pool(const char* what, const si_page_pool* p) {
  SI_CHECK_ARG(p != nullptr, "%s: NULL pool", what);
  SI_CHECK_ARG(dtype_ok((int)p->dtype) && p->dtype == (int)p->dtype, "%s: unsupported dtype %lld", what,
               (long long)p->dtype);
  SI_CHECK_ARG(p->precision >= SI_PREC_FP32 && p->precision <= SI_PREC_INT4, "%s: precision %lld is not 0..3",
               what, (long long)p->precision);
  constexpr int64_t top = (int64_t)1 << 31;
  SI_CHECK_ARG(p->heads > 0 && p->heads < 65536 && p->D > 0 && p->D <= 512 && p->pages > 0 && p->pages < top &&
               p->page_size > 0 && p->page_size < top, "%s: bad pool shape", what);
  SI_CHECK_ARG(p->pages <= (top - 1) / p->heads / p->page_size, "%s: pools hold fewer than 2^31 rows", what);
  SI_CHECK_ARG(p->group > 0 && p->D % p->group == 0, "%s: group must divide D", what);
  SI_CHECK_ARG(p->k && p->v, "%s: NULL pool tensor", what);
  SI_CHECK_ARG(p->precision < SI_PREC_INT8 || (p->scale_k && p->scale_v), "%s: NULL scales", what);
  SI_CHECK_ARG(((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v) |
                 reinterpret_cast<uintptr_t>(p->scale_k) | reinterpret_cast<uintptr_t>(p->scale_v)) & 15) == 0,
               "%s: pool tensors must be 16-byte aligned", what);
  return SI_OK;
}

}  // namespace si
