// Attention over the 8-bit paged cache with block scales: codes of type float8_e5m2.
#include <type_traits>

#include "rpa_quant_attn.h"

namespace rpa {

int launch_quant_e5m2(const QuantArgs& a, hipStream_t stream) { return launch_quant_codes<kCodeE5m2>(a, stream); }

}  // namespace rpa
