// 4-bit linear layers over bf16 rows, and the choice of element type.
#include "linear4.hpp"

namespace asrattn {

hipError_t launch_linear4_f32(const asrlayer_linear4_params& p, hipStream_t stream);

hipError_t launch_linear4(const asrlayer_linear4_params& p, hipStream_t stream) {
  return p.dtype == ASRATTN_BF16 ? launch_l4<bf16_raw>(p, stream) : launch_linear4_f32(p, stream);
}

}  // namespace asrattn
