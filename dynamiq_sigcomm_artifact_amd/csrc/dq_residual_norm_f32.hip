// the kernels of dq_residual_norm.cuh for activations of type DQ_F32
#include "dq_residual_norm.cuh"

namespace dq {

hipError_t launch_norm_f32(const BlockNormArgs &a, bool stream32, hipStream_t stream) { return launch_norm_in<DQ_F32>(a, stream32, stream); }
hipError_t launch_norm_backward_f32(const BlockNormBackArgs &a, bool stream32, hipStream_t stream) { return launch_norm_backward_in<DQ_F32>(a, stream32, stream); }

} // namespace dq
