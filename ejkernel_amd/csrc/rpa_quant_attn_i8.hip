// Attention over the 8-bit paged cache with block scales: codes of type int8.
#include <type_traits>

#include "rpa_quant_attn.h"

namespace rpa {

int launch_quant_i8(const QuantArgs& a, hipStream_t stream) { return launch_quant_codes<kCodeI8>(a, stream); }

}  // namespace rpa
