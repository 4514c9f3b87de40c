// Products of 4-bit microscaled matrices on the matrix cores.
#include "dq_launch.h"
#include "dq_microscale.cuh"

namespace dq {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct ProductArgs {
    const uint8_t *a_codes, *a_scales, *b_codes, *b_scales;
    void *out;
    int64_t m, n;
    int superchunks;
};

__device__ __forceinline__ i32x8 operand(uint4 v)
{
    i32x8 x = {(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
    return x;
}

// v_mfma_scale_f32_32x32x64_f8f6f4 on E2M1: lane l holds 32 consecutive elements of row l % 32, and their scale is byte S of its scale word.  The
// order of the contraction is free as long as both sides keep it: step s takes block s of the superchunk's first half from lanes 0 .. 31 and block s of
// its second half from lanes 32 .. 63, so that a lane's four scales are one word and its four blocks 64 bytes in a row.
template <int DT> __global__ __launch_bounds__(64) void mx4_product_kernel(ProductArgs p)
{
    const int lane = threadIdx.x, half = lane >> 5, row = lane & 31;
    const int64_t i0 = (int64_t)blockIdx.y * 32, j0 = (int64_t)blockIdx.x * 32;
    const int64_t i = min(i0 + row, p.m - 1), j = min(j0 + row, p.n - 1);
    const uint4 *a = reinterpret_cast<const uint4 *>(p.a_codes + i * p.superchunks * 128 + half * 64);
    const uint4 *b = reinterpret_cast<const uint4 *>(p.b_codes + j * p.superchunks * 128 + half * 64);
    const uint32_t *as = reinterpret_cast<const uint32_t *>(p.a_scales + i * p.superchunks * 8 + half * 4);
    const uint32_t *bs = reinterpret_cast<const uint32_t *>(p.b_scales + j * p.superchunks * 8 + half * 4);
    f32x16 acc = {};
    for (int s = 0; s < p.superchunks; s++) {
        const int sa = (int)as[2 * s], sb = (int)bs[2 * s];
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(b[8 * s]), operand(a[8 * s]), acc, 4, 4, 0, sb, 0, sa);
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(b[8 * s + 1]), operand(a[8 * s + 1]), acc, 4, 4, 1, sb, 1, sa);
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(b[8 * s + 2]), operand(a[8 * s + 2]), acc, 4, 4, 2, sb, 2, sa);
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(b[8 * s + 3]), operand(a[8 * s + 3]), acc, 4, 4, 3, sb, 3, sa);
    }
    // b is the left operand: a lane holds column `row` of the transposed tile, four consecutive columns of the result at a time
    if (i0 + row < p.m) {
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const int64_t c = j0 + (k >> 2) * 8 + half * 4 + (k & 3);
            if (c < p.n) ElemIO<DT>::store(p.out, (i0 + row) * p.n + c, acc[k]);
        }
    }
}

hipError_t launch_mx4_product(const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes, const uint8_t *b_scales, void *out, int64_t m,
                              int64_t n, int64_t k, int dtype, hipStream_t stream)
{
    const ProductArgs p = {a_codes, a_scales, b_codes, b_scales, out, m, n, (int)((k + 255) >> 8)};
    const dim3 grid((uint32_t)((n + 31) >> 5), (uint32_t)((m + 31) >> 5));
    if (dtype == DQ_F32)
        return launch_with(mx4_product_kernel<DQ_F32>, grid, dim3(64), stream, p);
    return dtype == DQ_BF16 ? launch_with(mx4_product_kernel<DQ_BF16>, grid, dim3(64), stream, p)
                            : launch_with(mx4_product_kernel<DQ_F16>, grid, dim3(64), stream, p);
}

} // namespace dq
