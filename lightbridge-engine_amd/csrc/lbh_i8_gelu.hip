// lbh_i8_gelu.hip — the 8-bit integer products (lbh_i8.hip) with bias and gelu (erf) in their epilogue.
#include "lbh_i8_forms.h"

namespace lbh {

hipError_t launch_i8_normal(const I8Args &a, int form, hipStream_t s) { return launch_epilogue<EPI_NORMAL>(a, form, s); }

}  // namespace lbh
