// 4-bit linear layers over float32 rows.
#include "linear4.hpp"

namespace asrattn {

hipError_t launch_linear4_f32(const asrlayer_linear4_params& p, hipStream_t stream);

hipError_t launch_linear4_f32(const asrlayer_linear4_params& p, hipStream_t stream) { return launch_l4<float>(p, stream); }

}  // namespace asrattn
