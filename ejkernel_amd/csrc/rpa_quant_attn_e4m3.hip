// Attention over the 8-bit paged cache with block scales: codes of type float8_e4m3fn.
#include <type_traits>

#include "rpa_quant_attn.h"

namespace rpa {

int launch_quant_e4m3(const QuantArgs& a, hipStream_t stream) { return launch_quant_codes<kCodeE4m3>(a, stream); }

}  // namespace rpa
