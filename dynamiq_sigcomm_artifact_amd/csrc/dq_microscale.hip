// 4-bit microscaled matrices: quantised along the rows or the columns, and their values.
//
// Both quantisers give a block of 32 elements to four neighbouring lanes, eight each: its largest magnitude and the last two stages of its
// rotation are two exchanges within the quad, and a lane's eight codes are one word.
#include "dq_launch.h"
#include "dq_microscale.cuh"

namespace dq {

enum { kNearest = -1, kPhilox = -2 }; // otherwise the element type of the pool

template <int CTRL> __device__ __forceinline__ float quad_f32(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// H (s x) / sqrt(32) of the quad's 32 elements, in place; word: the sign bits of the block.  Stages of stride 1, 2, 4 lie within a lane, 8 and 16
// between lanes.  Every sum is one of two numbers, whichever lane takes it: the result does not depend on the layout.
__device__ __forceinline__ void rotate_block(float (&v)[8], uint32_t word, int g)
{
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = __uint_as_float(__float_as_uint(v[j]) ^ (word >> (8 * g + j) & 1u) << 31);
#pragma unroll
    for (int h = 1; h < 8; h *= 2)
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (!(j & h)) {
                const float a = v[j], b = v[j + h];
                v[j] = a + b;
                v[j + h] = a - b;
            }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float b = quad_f32<0xB1>(v[j]);
        v[j] = g & 1 ? b - v[j] : v[j] + b;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float b = quad_f32<0x4E>(v[j]);
        v[j] = (g & 2 ? b - v[j] : v[j] + b) * 0.17677669529663687f;
    }
}

// the eight uniform values of elements e .. e + 7 of the result (e a multiple of 8)
template <int RAND> __device__ __forceinline__ void uniform8(const QuantizeArgs &a, int64_t e, float (&u)[8])
{
    if constexpr (RAND >= 0) {
        load8<RAND>(a.pool, e, u);
    } else if constexpr (RAND == kPhilox) {
        uint32_t w[4];
        chunk_uniform_words(a.key, e >> 4, w);
        const uint32_t lo = e & 8 ? w[2] : w[0], hi = e & 8 ? w[3] : w[1];
#pragma unroll
        for (int j = 0; j < 8; j++) u[j] = (float)(((j < 4 ? lo : hi) >> (8 * (j & 3)) & 0xffu) | 1u) * 0.00390625f;
    }
}

// eight codes in a word, the first in the lowest bits, and the block's scale byte (the same in the quad's lanes)
template <int RAND> __device__ __forceinline__ uint32_t encode_block(const float (&v)[8], const float (&u)[8], uint32_t &scale)
{
    const uint32_t largest = block_max(v);
    scale = RAND == kNearest ? block_scale<2, 0x7fffffu>(largest) : block_scale<2, 0x400000u>(largest);
    const float down = scale_down(scale);
    uint32_t word = 0;
    if constexpr (RAND == kNearest) {
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0] * down, v[1] * down, 1.0f, 0);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2] * down, v[3] * down, 1.0f, 1);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4] * down, v[5] * down, 1.0f, 2);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6] * down, v[7] * down, 1.0f, 3);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            // codes 0 .. 3 are halves, 4 and 5 are ones from 2 on, 6 and 7 twos from 4 on
            const float y = __builtin_fabsf(v[j]) * down;
            const float t = y < 2.0f ? 2.0f * y : y < 4.0f ? y : 0.5f * y;
            const float low = __builtin_floorf(t);
            const uint32_t code = (uint32_t)(y < 2.0f ? low : y < 4.0f ? low + 2.0f : low + 4.0f) + (u[j] < t - low ? 1u : 0u);
            word |= ((code & 7u) | (v[j] < 0.0f ? 8u : 0u)) << (4 * j);
        }
    }
    return word;
}

// ---- along the rows ----------------------------------------------------------------------------------------

template <int DT, int RAND, bool ROTATE> __global__ __launch_bounds__(256) void mx4_rows_kernel(QuantizeArgs a, uint32_t superchunks)
{
    const int g = threadIdx.x & 3;
    const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; // of the result, padding included
    const int64_t sc = e >> 8;
    if (sc >= a.rows * superchunks) return;
    const int64_t row = sc / superchunks;
    const int64_t col = e - row * superchunks * 256;
    float v[8], u[8];
    const int64_t at = row * a.stride + col;
    if (col + 8 <= a.cols)
        load8<DT>(a.x, at, v);
    else
        load_part<DT, 8>(a.x, at, row * a.stride + a.cols, v);
    uniform8<RAND>(a, e, u);
    if (ROTATE) rotate_block(v, a.sign[col >> 5], g);
    uint32_t scale;
    reinterpret_cast<uint32_t *>(a.codes)[e >> 3] = encode_block<RAND>(v, u, scale);
    if (g == 0) a.scales[e >> 5] = (uint8_t)scale;
}

// ---- along the columns -------------------------------------------------------------------------------------

// A workgroup takes 256 rows x 128 columns: one superchunk of 128 rows of the result.  A wave takes 32 of the rows, a lane 8 rows x 8 columns, and a
// column's block lies in a quad as it does above.  The codes leave through LDS, as whole lines.
template <int DT, int RAND, bool ROTATE> __global__ __launch_bounds__(512) void mx4_columns_kernel(QuantizeArgs a, uint32_t superchunks)
{
    __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 128];
    __shared__ __attribute__((aligned(8))) uint8_t tile_scales[128 * 8];
    const int lane = threadIdx.x & 63, block = threadIdx.x >> 6, g = lane & 3;
    const int64_t col0 = (int64_t)blockIdx.x * 128, col = col0 + 8 * (lane >> 2);
    const int64_t row0 = (int64_t)blockIdx.y * 256 + 32 * block, row = row0 + 8 * g;
    float x[8][8]; // [row][column]
    const int cols = (int)min((int64_t)8, a.cols - col);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int64_t at = min(row + j, a.rows - 1) * a.stride;
        if (cols == 8)
            load8<DT>(a.x, at + col, x[j]);
        else
            load_part<DT, 8>(a.x, at + col, at + a.cols, x[j]);
    }
    if (row + 8 > a.rows) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (row + j >= a.rows) {
#pragma unroll
                for (int c = 0; c < 8; c++) x[j][c] = 0.0f;
            }
    }
    const uint32_t sign = ROTATE ? a.sign[row0 >> 5] : 0u;
#pragma unroll
    for (int c = 0; c < 8; c++) {
        float v[8], u[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = x[j][c];
        if (RAND == kPhilox || c < cols) uniform8<RAND>(a, ((col + c) * superchunks + blockIdx.y) * 256 + 32 * block + 8 * g, u);
        if (ROTATE) rotate_block(v, sign, g);
        uint32_t scale;
        const uint32_t word = encode_block<RAND>(v, u, scale);
        const int line = 8 * (lane >> 2) + c;
        *reinterpret_cast<uint32_t *>(tile + line * 128 + ((block ^ (line >> 3 & 7)) << 4) + 4 * g) = word;
        if (g == 0) tile_scales[line * 8 + block] = (uint8_t)scale;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int s = threadIdx.x + 512 * k, line = s >> 3, piece = s & 7;
        if (col0 + line < a.cols)
            reinterpret_cast<uint4 *>(a.codes)[((col0 + line) * superchunks + blockIdx.y) * 8 + piece] =
                *reinterpret_cast<const uint4 *>(tile + line * 128 + ((piece ^ (line >> 3 & 7)) << 4));
    }
    if (threadIdx.x < 128 && col0 + threadIdx.x < a.cols)
        reinterpret_cast<uint2 *>(a.scales)[(col0 + threadIdx.x) * superchunks + blockIdx.y] = reinterpret_cast<const uint2 *>(tile_scales)[threadIdx.x];
}

template <int DT, int RAND> static hipError_t launch_quantize(const QuantizeArgs &a, bool columns, hipStream_t stream)
{
    const uint32_t superchunks = (uint32_t)(((columns ? a.rows : a.cols) + 255) >> 8);
    if (columns) {
        const dim3 grid((uint32_t)((a.cols + 127) >> 7), superchunks);
        if (a.sign)
            mx4_columns_kernel<DT, RAND, true><<<grid, 512, 0, stream>>>(a, superchunks);
        else
            mx4_columns_kernel<DT, RAND, false><<<grid, 512, 0, stream>>>(a, superchunks);
    } else {
        const dim3 grid((uint32_t)((a.rows * superchunks + 7) >> 3));
        if (a.sign)
            mx4_rows_kernel<DT, RAND, true><<<grid, 256, 0, stream>>>(a, superchunks);
        else
            mx4_rows_kernel<DT, RAND, false><<<grid, 256, 0, stream>>>(a, superchunks);
    }
    return hipGetLastError();
}

template <int DT> static hipError_t launch_quantize_of(const QuantizeArgs &a, bool columns, bool stochastic, int pool_dtype, hipStream_t stream)
{
    if (!stochastic) return launch_quantize<DT, kNearest>(a, columns, stream);
    if (!a.pool) return launch_quantize<DT, kPhilox>(a, columns, stream);
    return pool_dtype == DQ_F32 ? launch_quantize<DT, DQ_F32>(a, columns, stream)
         : pool_dtype == DQ_BF16 ? launch_quantize<DT, DQ_BF16>(a, columns, stream) : launch_quantize<DT, DQ_F16>(a, columns, stream);
}

hipError_t launch_mx4_quantize(const QuantizeArgs &a, int dtype, bool columns, bool stochastic, int pool_dtype, hipStream_t stream)
{
    return dtype == DQ_F32 ? launch_quantize_of<DQ_F32>(a, columns, stochastic, pool_dtype, stream)
         : dtype == DQ_BF16 ? launch_quantize_of<DQ_BF16>(a, columns, stochastic, pool_dtype, stream)
                            : launch_quantize_of<DQ_F16>(a, columns, stochastic, pool_dtype, stream);
}

// ---- and back ----------------------------------------------------------------------------------------------

template <int DT>
__global__ __launch_bounds__(256) void mx4_values_kernel(const uint32_t *__restrict__ codes, const uint8_t *__restrict__ scales, void *__restrict__ out,
                                                        int64_t rows, int64_t cols, uint32_t superchunks)
{
    const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8, sc = e >> 8;
    if (sc >= rows * superchunks) return;
    const int64_t row = sc / superchunks;
    const int64_t col = e - row * superchunks * 256;
    if (col >= cols) return;
    const uint32_t word = codes[e >> 3];
    const float up = scale_up(scales[e >> 5]);
    float v[8];
    const f32x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 1);
    const f32x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 3);
    v[0] = p0.x * up; v[1] = p0.y * up; v[2] = p1.x * up; v[3] = p1.y * up;
    v[4] = p2.x * up; v[5] = p2.y * up; v[6] = p3.x * up; v[7] = p3.y * up;
    if (col + 8 <= cols)
        store8<DT>(out, row * cols + col, v);
    else
        store_part<DT, 8>(out, row * cols + col, (int)(cols - col), v);
}

hipError_t launch_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, void *out, int64_t rows, int64_t cols, int dtype, hipStream_t stream)
{
    const uint32_t superchunks = (uint32_t)((cols + 255) >> 8);
    const dim3 grid((uint32_t)((rows * superchunks + 7) >> 3));
    const uint32_t *words = reinterpret_cast<const uint32_t *>(codes);
    if (dtype == DQ_F32)
        mx4_values_kernel<DQ_F32><<<grid, 256, 0, stream>>>(words, scales, out, rows, cols, superchunks);
    else if (dtype == DQ_BF16)
        mx4_values_kernel<DQ_BF16><<<grid, 256, 0, stream>>>(words, scales, out, rows, cols, superchunks);
    else
        mx4_values_kernel<DQ_F16><<<grid, 256, 0, stream>>>(words, scales, out, rows, cols, superchunks);
    return hipGetLastError();
}

} // namespace dq
