// bf16 instantiations of the paged attention kernel.
#include "paged_attn.h"

namespace cmpext3 {
hipError_t launch_paged_attn_bf16(const AttnArgs& a, int wgs, hipStream_t s) { return launch_type<__bf16>(a, wgs, s); }
}  // namespace cmpext3
