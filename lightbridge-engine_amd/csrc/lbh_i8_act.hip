// lbh_i8_act.hip — the 8-bit integer products (lbh_i8.hip) with bias and the activations none, relu, relu
// squared, silu and gelu (tanh) in their epilogue.
#include "lbh_i8_forms.h"

namespace lbh {

hipError_t launch_i8_sigmoid(const I8Args &a, int form, hipStream_t s) { return launch_epilogue<EPI_SIGMOID>(a, form, s); }

}  // namespace lbh
