// The gated delta rule's kernels for bf16 storage (gated_delta.hpp).
#include "gated_delta_launch.hpp"

namespace mqc {
namespace delta {
template int launch_fwd<bf16_t>(const Args<bf16_t>&, hipStream_t);
template int launch_bwd<bf16_t>(const Args<bf16_t>&, hipStream_t);
template int launch_step<bf16_t>(const Args<bf16_t>&, float*, hipStream_t);
}  // namespace delta
}  // namespace mqc
