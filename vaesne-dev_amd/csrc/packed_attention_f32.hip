// Packed-sequence attention for f32 tensors (packed_attention.h).
#include "packed_attention.h"

namespace vaesne {
namespace pk {
template <> int run_fwd<float>(const Plan& p, hipStream_t s) { return dispatch<float, false>(p, s); }
template <> int run_bwd<float>(const Plan& p, hipStream_t s) { return dispatch<float, true>(p, s); }
}  // namespace pk
}  // namespace vaesne
