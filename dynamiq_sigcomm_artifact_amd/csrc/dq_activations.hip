// Activations between the linear layers: 8-bit checkpoints, and the gated activation.
//
// Both are elementwise but for the largest magnitude of a block of 32, which four neighbouring lanes share with two exchanges, and are bound by memory.
#include "dq_launch.h"
#include "dq_microscale.cuh"

namespace dq {

// ---- checkpoints --------------------------------------------------------------------------------------------

template <int DT> __global__ __launch_bounds__(256) void checkpoint_compress_kernel(CheckpointArgs a, Division blocks, uint32_t units)
{
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    if (unit >= units) return;
    const uint32_t row = blocks(unit >> 2), col = (unit - row * blocks.by * 4) * 8;
    float v[8];
    const int64_t at = (int64_t)row * a.stride + col;
    if (col + 8 <= a.cols)
        load8<DT>(a.x, at, v);
    else
        load_part<DT, 8>(a.x, at, (int64_t)row * a.stride + a.cols, v);
    uint32_t scale;
    const u32x2_t w = encode_e4m3<DT>(v, scale);
    reinterpret_cast<u32x2_t *>(a.data)[unit] = w;
    if ((threadIdx.x & 3) == 0) a.data[a.rows * 32 * blocks.by + (unit >> 2)] = (uint8_t)scale;
}

hipError_t launch_checkpoint_compress(const CheckpointArgs &a, int dtype, hipStream_t stream)
{
    const Division blocks((a.cols + 31) >> 5, 30);
    const uint32_t units = (uint32_t)(a.rows * blocks.by * 4);
    const dim3 grid((units + 255) / 256);
    if (dtype == DQ_F32)
        checkpoint_compress_kernel<DQ_F32><<<grid, 256, 0, stream>>>(a, blocks, units);
    else if (dtype == DQ_BF16)
        checkpoint_compress_kernel<DQ_BF16><<<grid, 256, 0, stream>>>(a, blocks, units);
    else
        checkpoint_compress_kernel<DQ_F16><<<grid, 256, 0, stream>>>(a, blocks, units);
    return hipGetLastError();
}

template <int DT> __global__ __launch_bounds__(256) void checkpoint_restore_kernel(const uint8_t *__restrict__ data, void *__restrict__ out, int64_t scales, uint32_t cols, Division blocks, uint32_t units)
{
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    if (unit >= units) return;
    const uint32_t row = blocks(unit >> 2), col = (unit - row * blocks.by * 4) * 8;
    if (col >= cols) return;
    float v[8];
    decode_e4m3(reinterpret_cast<const u32x2_t *>(data)[unit], data[scales + (unit >> 2)], v);
    const int64_t at = (int64_t)row * cols + col;
    if (col + 8 <= cols)
        store8<DT>(out, at, v);
    else
        store_part<DT, 8>(out, at, (int)(cols - col), v);
}

hipError_t launch_checkpoint_restore(const uint8_t *data, void *out, int64_t rows, int64_t cols, int dtype, hipStream_t stream)
{
    const Division blocks((uint32_t)((cols + 31) >> 5), 30);
    const uint32_t units = (uint32_t)(rows * blocks.by * 4);
    const int64_t scales = rows * 32 * blocks.by;
    const dim3 grid((units + 255) / 256);
    if (dtype == DQ_F32)
        checkpoint_restore_kernel<DQ_F32><<<grid, 256, 0, stream>>>(data, out, scales, (uint32_t)cols, blocks, units);
    else if (dtype == DQ_BF16)
        checkpoint_restore_kernel<DQ_BF16><<<grid, 256, 0, stream>>>(data, out, scales, (uint32_t)cols, blocks, units);
    else
        checkpoint_restore_kernel<DQ_F16><<<grid, 256, 0, stream>>>(data, out, scales, (uint32_t)cols, blocks, units);
    return hipGetLastError();
}

} // namespace dq
