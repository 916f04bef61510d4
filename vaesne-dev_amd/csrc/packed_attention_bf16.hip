// Packed-sequence attention for bf16 tensors (packed_attention.h).
#include "packed_attention.h"

namespace vaesne {
namespace pk {
template <> int run_fwd<__bf16>(const Plan& p, hipStream_t s) { return dispatch<__bf16, false>(p, s); }
template <> int run_bwd<__bf16>(const Plan& p, hipStream_t s) { return dispatch<__bf16, true>(p, s); }
}  // namespace pk
}  // namespace vaesne
