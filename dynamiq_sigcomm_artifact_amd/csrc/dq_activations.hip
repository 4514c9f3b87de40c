// Activations between the linear layers: 8-bit checkpoints, and the gated activation.
//
// Both are elementwise but for the largest magnitude of a block of 32, which four neighbouring lanes share with two exchanges, and are bound by memory.
#include "dq_launch.h"
#include "dq_microscale.cuh"

namespace dq {

// ---- checkpoints --------------------------------------------------------------------------------------------

// What is beyond the 256 MB cache is loaded with the hint that nothing of it is wanted again soon: 8192 x 14336 bf16 in 59 us, 6.0 TB/s (65 without).
inline bool passes(int64_t rows, uint32_t cols, int arrays, int dtype) { return rows * cols * arrays * (dtype == DQ_F32 ? 4 : 2) > (int64_t)128 << 20; }

struct CompressCall {
    CheckpointArgs a;
    Division blocks;
    uint32_t units;
};
template <int DT, bool PASSING> __global__ __launch_bounds__(256) void checkpoint_compress_kernel(CompressCall call)
{
    const CheckpointArgs &a = call.a;
    const Division &blocks = call.blocks;
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    if (unit >= call.units) return;
    const uint32_t row = blocks(unit >> 2), col = (unit - row * blocks.by * 4) * 8;
    float v[8];
    const int64_t at = (int64_t)row * a.stride + col;
    if (col + 8 <= a.cols)
        load8<DT, PASSING>(a.x, at, v);
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
    const CompressCall call = {a, blocks, (uint32_t)(a.rows * blocks.by * 4)};
    const auto launch = [&](auto passing, auto whole) { return launch_with(passes(a.rows, a.cols, 1, dtype) ? passing : whole, dim3((call.units + 255) / 256), dim3(256), stream, call); };
    return dtype == DQ_F32 ? launch(checkpoint_compress_kernel<DQ_F32, true>, checkpoint_compress_kernel<DQ_F32, false>)
         : dtype == DQ_BF16 ? launch(checkpoint_compress_kernel<DQ_BF16, true>, checkpoint_compress_kernel<DQ_BF16, false>)
                            : launch(checkpoint_compress_kernel<DQ_F16, true>, checkpoint_compress_kernel<DQ_F16, false>);
}

// 8192 x 14336 to bf16 in 55 us, 6.5 TB/s
struct RestoreCall {
    const uint8_t *data;
    void *out;
    int64_t scales;
    uint32_t cols, units;
    Division blocks;
};
template <int DT> __global__ __launch_bounds__(256) void checkpoint_restore_kernel(RestoreCall a)
{
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    if (unit >= a.units) return;
    const uint32_t row = a.blocks(unit >> 2), col = (unit - row * a.blocks.by * 4) * 8;
    if (col >= a.cols) return;
    float v[8];
    decode_e4m3(reinterpret_cast<const u32x2_t *>(a.data)[unit], a.data[a.scales + (unit >> 2)], v);
    const int64_t at = (int64_t)row * a.cols + col;
    if (col + 8 <= a.cols)
        store8<DT>(a.out, at, v);
    else
        store_part<DT, 8>(a.out, at, (int)(a.cols - col), v);
}

hipError_t launch_checkpoint_restore(const uint8_t *data, void *out, int64_t rows, int64_t cols, int dtype, hipStream_t stream)
{
    const Division blocks((uint32_t)((cols + 31) >> 5), 30);
    const RestoreCall call = {data, out, rows * 32 * blocks.by, (uint32_t)cols, (uint32_t)(rows * blocks.by * 4), blocks};
    const dim3 grid((call.units + 255) / 256), block(256);
    return dtype == DQ_F32 ? launch_with(checkpoint_restore_kernel<DQ_F32>, grid, block, stream, call)
         : dtype == DQ_BF16 ? launch_with(checkpoint_restore_kernel<DQ_BF16>, grid, block, stream, call) : launch_with(checkpoint_restore_kernel<DQ_F16>, grid, block, stream, call);
}

// ---- the gated activation -----------------------------------------------------------------------------------

// sigmoid(q) and 1 - sigmoid(q), neither from the other: with e = exp(-|q|) they are 1 / (1 + e) and e / (1 + e).  For 16-bit types e is the machine's power of two of -|q| log2(e), off by
// (2 + 2 |q|) 2^-24 of itself, and the quotient its reciprocal, by 2^-23: 2^-16 at |q| = 88, the largest, a fortieth at most of the rounding to 16 bits that follows.  With the functions that
// binary32 takes 8192 x 14336 bf16 is 141 us for 112 forward (160 for 129 with the checkpoint), 363 for 351 in both passes with checkpoints.
template <int DT> __device__ __forceinline__ void sigmoids(float q, float &s, float &rest)
{
    const float e = DT == DQ_F32 ? expf(-__builtin_fabsf(q)) : __expf(-__builtin_fabsf(q));
    const float big = DT == DQ_F32 ? 1.0f / (1.0f + e) : __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
    s = q >= 0.0f ? big : small;
    rest = q >= 0.0f ? small : big;
}
// act(g) = g sigmoid(q(g)): q = g, or for the hyperbolic tangent's form of gelu q = 2 sqrt(2 / pi) (g + 0.044715 g^3), of which from 20 on nothing changes the sigmoid any more
template <int KIND> __device__ __forceinline__ float exponent_of(float g, float &slope)
{
    if (KIND == DQ_SILU) {
        slope = 1.0f;
        return g;
    }
    constexpr float c = 1.5957691216057308f;
    const float x = __builtin_amdgcn_fmed3f(g, -20.0f, 20.0f), square = x * x;
    slope = c + 3 * 0.044715f * c * square;
    return x * (c + 0.044715f * c * square);
}

struct GatedCall {
    GatedArgs a;
    Division blocks;
    uint32_t units;
};
static_assert(sizeof(GatedCall) <= 128, "a launch whose arguments are longer takes longer");

// A lane takes eight elements, four of them a block of 32, padding included: the last block of a row may be a part.  Bound by memory: 8192 x 14336 bf16 with all three checkpoints
// in 158 to 170 us by the box (6.3 to 6.8 TB/s, where loads and the result carry the hint; 178 without, and 175 with it on the checkpoints too), backward from them in 165 to 179
// (5.3 to 5.7 TB/s): half of that is stores, in two streams.  The hint on its stores takes 161 on one box and 190 on another, on its loads 173 and 170; two units a lane 8 % more,
// workgroups of 1024 5 %.  Without checkpoints 112 (6.3 TB/s) and 205 (5.7 TB/s); fp32 4096 x 14336 138 and 203.
template <int DT, int KIND, bool EIGHT, bool PASSING> __global__ __launch_bounds__(256) void gated_kernel(GatedCall call)
{
    const GatedArgs &a = call.a;
    const Division &blocks = call.blocks;
    const uint32_t units = call.units;
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    if (unit >= units) return;
    const uint32_t row = blocks(unit >> 2), col = (unit - row * blocks.by * 4) * 8;
    if (!EIGHT && col >= a.cols) return;
    const bool whole = col + 8 <= a.cols;
    const int64_t at_gate = row * a.gate_stride + col, at_up = row * a.up_stride + col, at = (int64_t)row * a.cols + col;
    float g[8], u[8], v[8];
    if (whole) {
        load8<DT, PASSING>(a.gate, at_gate, g);
        load8<DT, PASSING>(a.up, at_up, u);
    } else {
        load_part<DT, 8>(a.gate, at_gate, row * a.gate_stride + a.cols, g);
        load_part<DT, 8>(a.up, at_up, row * a.up_stride + a.cols, u);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float slope, s, rest;
        sigmoids<DT>(exponent_of<KIND>(g[j], slope), s, rest);
        v[j] = ElemIO<DT>::round(g[j] * s * u[j]);
    }
    if (whole)
        store8<DT, PASSING>(a.out, at, v);
    else if (col < a.cols)
        store_part<DT, 8>(a.out, at, (int)(a.cols - col), v);
    if (EIGHT) {
        const int64_t scales = (int64_t)units * 8 + (unit >> 2);
        const auto put = [&](uint8_t *data, const float (&x)[8]) {
            if (!data) return; // (the same for every lane)
            uint32_t scale;
            const u32x2_t w = encode_e4m3<DT>(x, scale);
            reinterpret_cast<u32x2_t *>(data)[unit] = w;
            if ((threadIdx.x & 3) == 0) data[scales] = (uint8_t)scale;
        };
        put(a.out8, v);
        put(a.gate8, g);
        put(a.up8, u);
    }
}

template <int DT, int KIND, bool EIGHT> __global__ __launch_bounds__(256) void gated_backward_kernel(GatedCall call)
{
    const GatedArgs &a = call.a;
    const Division &blocks = call.blocks;
    const uint32_t units = call.units;
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    if (unit >= units) return;
    const uint32_t row = blocks(unit >> 2), col = (unit - row * blocks.by * 4) * 8;
    if (col >= a.cols) return;
    const bool whole = col + 8 <= a.cols;
    const int64_t at = (int64_t)row * a.cols + col;
    float g[8], u[8], d[8];
    if (whole)
        load8<DT>(a.out, at, d);
    else
        load_part<DT, 8>(a.out, at, (int64_t)(row + 1) * a.cols, d);
    if (EIGHT) {
        const int64_t scales = (int64_t)units * 8 + (unit >> 2);
        decode_e4m3(reinterpret_cast<const u32x2_t *>(a.gate8)[unit], a.gate8[scales], g);
        decode_e4m3(reinterpret_cast<const u32x2_t *>(a.up8)[unit], a.up8[scales], u);
    } else if (whole) {
        load8<DT>(a.gate, row * a.gate_stride + col, g);
        load8<DT>(a.up, row * a.up_stride + col, u);
    } else {
        load_part<DT, 8>(a.gate, row * a.gate_stride + col, row * a.gate_stride + a.cols, g);
        load_part<DT, 8>(a.up, row * a.up_stride + col, row * a.up_stride + a.cols, u);
    }
    // act' = s + g s (1 - s) q'
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float slope, s, rest;
        sigmoids<DT>(exponent_of<KIND>(g[j], slope), s, rest);
        const float value = g[j] * s;
        g[j] = d[j] * u[j] * (s + value * (rest * slope));
        u[j] = d[j] * value;
    }
    const int64_t to_gate = row * a.dgate_stride + col, to_up = row * a.dup_stride + col;
    if (a.dgate) {
        if (whole)
            store8<DT>(a.dgate, to_gate, g);
        else
            store_part<DT, 8>(a.dgate, to_gate, (int)(a.cols - col), g);
    }
    if (a.dup) {
        if (whole)
            store8<DT>(a.dup, to_up, u);
        else
            store_part<DT, 8>(a.dup, to_up, (int)(a.cols - col), u);
    }
}

template <int DT, int KIND, bool EIGHT> static hipError_t launch_gated_of(const GatedArgs &a, bool backward, hipStream_t stream)
{
    const Division blocks((a.cols + 31) >> 5, 30);
    const GatedCall call = {a, blocks, (uint32_t)(a.rows * blocks.by * 4)};
    const dim3 grid((call.units + 255) / 256), block(256);
    if (backward) return launch_with(gated_backward_kernel<DT, KIND, EIGHT>, grid, block, stream, call);
    return passes(a.rows, a.cols, 4, DT) ? launch_with(gated_kernel<DT, KIND, EIGHT, true>, grid, block, stream, call) : launch_with(gated_kernel<DT, KIND, EIGHT, false>, grid, block, stream, call);
}
template <int DT> static hipError_t launch_gated_with(const GatedArgs &a, int kind, bool backward, hipStream_t stream)
{
    const bool eight = backward ? a.gate8 != nullptr : a.out8 || a.gate8 || a.up8;
    if (kind == DQ_SILU) return eight ? launch_gated_of<DT, DQ_SILU, true>(a, backward, stream) : launch_gated_of<DT, DQ_SILU, false>(a, backward, stream);
    return eight ? launch_gated_of<DT, DQ_GELU_TANH, true>(a, backward, stream) : launch_gated_of<DT, DQ_GELU_TANH, false>(a, backward, stream);
}

hipError_t launch_gated(const GatedArgs &a, int dtype, int kind, bool backward, hipStream_t stream)
{
    return dtype == DQ_F32 ? launch_gated_with<DQ_F32>(a, kind, backward, stream)
         : dtype == DQ_BF16 ? launch_gated_with<DQ_BF16>(a, kind, backward, stream) : launch_gated_with<DQ_F16>(a, kind, backward, stream);
}

} // namespace dq
