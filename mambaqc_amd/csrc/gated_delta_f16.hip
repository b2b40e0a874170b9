// The gated delta rule's kernels for f16 storage (gated_delta.hpp).
#include "gated_delta_launch.hpp"

namespace mqc {
namespace delta {
template int launch_fwd<f16_t>(const Args<f16_t>&, hipStream_t);
template int launch_bwd<f16_t>(const Args<f16_t>&, hipStream_t);
template int launch_step<f16_t>(const Args<f16_t>&, float*, hipStream_t);
}  // namespace delta
}  // namespace mqc
