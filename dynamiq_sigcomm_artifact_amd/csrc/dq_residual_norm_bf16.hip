// the kernels of dq_residual_norm.cuh for activations of type DQ_BF16
#include "dq_residual_norm.cuh"

namespace dq {

hipError_t launch_norm_bf16(const BlockNormArgs &a, bool stream32, hipStream_t stream) { return launch_norm_in<DQ_BF16>(a, stream32, stream); }
hipError_t launch_norm_backward_bf16(const BlockNormBackArgs &a, bool stream32, hipStream_t stream) { return launch_norm_backward_in<DQ_BF16>(a, stream32, stream); }

} // namespace dq
