// The gated delta rule's kernels for f32 storage (gated_delta.hpp).
#include "gated_delta_launch.hpp"

namespace mqc {
namespace delta {
template int launch_fwd<float>(const Args<float>&, hipStream_t);
template int launch_bwd<float>(const Args<float>&, hipStream_t);
template int launch_step<float>(const Args<float>&, float*, hipStream_t);
}  // namespace delta
}  // namespace mqc
