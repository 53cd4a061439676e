// fp32 instantiations of the paged attention kernel.
#include "paged_attn.h"

namespace cmpext3 {
hipError_t launch_paged_attn_f32(const AttnArgs& a, int wgs, hipStream_t s) { return launch_type<float>(a, wgs, s); }
}  // namespace cmpext3
