// Packed-sequence attention for f16 tensors (packed_attention.h).
#include "packed_attention.h"

namespace vaesne {
namespace pk {
template <> int run_fwd<_Float16>(const Plan& p, hipStream_t s) { return dispatch<_Float16, false>(p, s); }
template <> int run_bwd<_Float16>(const Plan& p, hipStream_t s) { return dispatch<_Float16, true>(p, s); }
}  // namespace pk
}  // namespace vaesne
