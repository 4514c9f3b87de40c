// Microscaled blocks: 32 consecutive elements share a power of two 2^k, stored as the byte k + 127 (255: the block is not a number).
// What the 4-bit operands of products, the 8-bit optimizer states and the 8-bit activation checkpoints have in common.
#pragma once

#include "dq_device.cuh"

namespace dq {

// n / by for n below 2^bits (at most 30): (n mul) >> shift with mul = ceil(2^shift / by) and shift = bits + ceil(log2 by), whose excess is less than n 2^-shift
struct Division {
    uint32_t by, mul, shift;
    Division() = default;
    explicit Division(uint32_t by_, uint32_t bits = 27) : by(by_), shift(bits)
    {
        while (((uint64_t)1 << (shift - bits)) < by) shift++;
        mul = (uint32_t)((((uint64_t)1 << shift) + by - 1) / by);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (uint32_t)((uint64_t)n * mul >> shift); }
};

// ---- four or eight consecutive elements of a vector that may lie anywhere: a view into a gradient bucket is aligned to its elements only, and
// gfx950 loads and stores 16 bytes from any address.  PASSING: with the hint that nothing of it is wanted again soon ----
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

template <int DT> __device__ __forceinline__ void unpack2(uint32_t w, float &a, float &b)
{
    if (DT == DQ_BF16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    } else {
        a = f16_bits_to_f32(w & 0xffffu);
        b = f16_bits_to_f32(w >> 16);
    }
}
template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b)
{
    return DT == DQ_BF16 ? f32x2_to_bf16x2(a, b) : f32_to_f16_bits(a) | (f32_to_f16_bits(b) << 16);
}

template <int DT, bool PASSING = false> __device__ __forceinline__ void load4(const void *p, int64_t i, float *v)
{
    if (DT == DQ_F32) {
        const f32x4_any *q = reinterpret_cast<const f32x4_any *>(static_cast<const float *>(p) + i);
        const f32x4_any a = PASSING ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = a[j];
    } else {
        const u32x2_any *q = reinterpret_cast<const u32x2_any *>(static_cast<const uint16_t *>(p) + i);
        const u32x2_any a = PASSING ? __builtin_nontemporal_load(q) : *q;
        unpack2<DT>(a[0], v[0], v[1]);
        unpack2<DT>(a[1], v[2], v[3]);
    }
}

template <int DT, bool PASSING = false> __device__ __forceinline__ void load8(const void *p, int64_t i, float (&v)[8])
{
    if (DT == DQ_F32) {
        load4<DT, PASSING>(p, i, v);
        load4<DT, PASSING>(p, i + 4, v + 4);
    } else {
        const u32x4_any *q = reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(p) + i);
        const u32x4_any a = PASSING ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
        for (int j = 0; j < 4; j++) unpack2<DT>(a[j], v[2 * j], v[2 * j + 1]);
    }
}

// the same as words, two elements of a 16-bit type in each, and element j of them
template <int DT, int WORDS> __device__ __forceinline__ void load_words(const void *p, int64_t i, uint32_t (&x)[WORDS])
{
    const char *q = static_cast<const char *>(p) + i * (DT == DQ_F32 ? 4 : 2);
#pragma unroll
    for (int k = 0; k < WORDS; k += 4) {
        const u32x4_any a = *reinterpret_cast<const u32x4_any *>(q + 4 * k);
#pragma unroll
        for (int j = 0; j < 4; j++) x[k + j] = a[j];
    }
}
template <int DT, int WORDS> __device__ __forceinline__ float word_value(const uint32_t (&x)[WORDS], int j)
{
    if (DT == DQ_F32) return __uint_as_float(x[j]);
    float v[2];
    unpack2<DT>(x[j / 2], v[0], v[1]);
    return v[j & 1];
}
// ... and the elements i .. of the n that a row of fewer than eight has, those past its end 0
template <int DT, int WORDS> __device__ __forceinline__ void load_words_part(const void *p, int64_t row, uint32_t i, uint32_t n, uint32_t (&x)[WORDS])
{
    constexpr int PER = 8 / WORDS;
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int64_t at = row + min(i + j, n - 1);
        e[j] = DT == DQ_F32 ? static_cast<const uint32_t *>(p)[at] : static_cast<const uint16_t *>(p)[at];
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (i + j >= n) e[j] = 0u;
#pragma unroll
    for (int w = 0; w < WORDS; w++) x[w] = PER == 1 ? e[w] : e[PER * w] | e[PER * w + PER - 1] << 16;
}

// N elements from i on of a vector of n (n > 0), those past its end 0.  (Every lane loads, the last element where there is none, so that the loads do not
// wait for one another.)
template <int DT, int N> __device__ __forceinline__ void load_part(const void *p, int64_t i, int64_t n, float *v)
{
#pragma unroll
    for (int j = 0; j < N; j++) v[j] = ElemIO<DT>::load(p, min(i + j, n - 1));
#pragma unroll
    for (int j = 0; j < N; j++)
        if (i + j >= n) v[j] = 0.0f;
}

template <int DT, bool PASSING = false> __device__ __forceinline__ void store4(void *p, int64_t i, const float *v)
{
    if (DT == DQ_F32) {
        const f32x4_any a = {v[0], v[1], v[2], v[3]};
        f32x4_any *q = reinterpret_cast<f32x4_any *>(static_cast<float *>(p) + i);
        if (PASSING)
            __builtin_nontemporal_store(a, q);
        else
            *q = a;
    } else {
        const u32x2_any a = {pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
        u32x2_any *q = reinterpret_cast<u32x2_any *>(static_cast<uint16_t *>(p) + i);
        if (PASSING)
            __builtin_nontemporal_store(a, q);
        else
            *q = a;
    }
}

template <int DT, bool PASSING = false> __device__ __forceinline__ void store8(void *p, int64_t i, const float (&v)[8])
{
    if (DT == DQ_F32) {
        store4<DT, PASSING>(p, i, v);
        store4<DT, PASSING>(p, i + 4, v + 4);
    } else {
        const u32x4_any a = {pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])};
        u32x4_any *q = reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(p) + i);
        if (PASSING)
            __builtin_nontemporal_store(a, q);
        else
            *q = a;
    }
}

template <int DT, int N> __device__ __forceinline__ void store_part(void *p, int64_t i, int count, const float *v)
{
#pragma unroll
    for (int j = 0; j < N; j++)
        if (j < count) ElemIO<DT>::store(p, i + j, v[j]);
}

// Workgroups go to the eight XCDs in turn: each gets a run of the count units of work that lie together, so that what its 32 CUs work on at a time shares its L2.
__device__ __forceinline__ uint32_t unit_of(uint32_t id, uint32_t count)
{
    const uint32_t xcd = id & 7;
    return xcd * (count >> 3) + min(xcd, count & 7) + (id >> 3);
}

// ---- the shared power of two ----

// the largest magnitude of a block, which four neighbouring lanes hold eight elements each of, as a bit pattern: magnitudes are ordered
// like their patterns, and infinities and NaN, which the maximum passes on, lie above every number
__device__ __forceinline__ uint32_t block_max(const float (&v)[8])
{
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) most = __builtin_elementwise_maximum(most, __builtin_fabsf(v[j]));
    uint32_t u = __float_as_uint(most) & 0x7fffffffu;
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0xB1, 0xf, 0xf, true)); // quad_perm [1,0,3,2]
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x4E, 0xf, 0xf, true)); // quad_perm [2,3,0,1]
    return u;
}

// the byte k + 127 for k = floor(log2 largest) - TOP, one more where the mantissa's 23 bits are above LIFT; 0 at the least (and for a
// block of zeros), 255 for a block that holds an infinity or NaN
template <int TOP, uint32_t LIFT> __device__ __forceinline__ uint32_t block_scale(uint32_t largest)
{
    const int k = (int)(largest >> 23) - TOP + ((largest & 0x7fffffu) > LIFT ? 1 : 0);
    return largest >= 0x7f800000u ? 255u : (uint32_t)max(k, 0);
}
// 2^-k, a normal number for every byte up to 253; 0 for 255
__device__ __forceinline__ float scale_down(uint32_t byte) { return __uint_as_float(byte == 255u ? 0u : (254u - byte) << 23); }
// 2^k (2^-127 is subnormal); NaN for 255
__device__ __forceinline__ float scale_up(uint32_t byte)
{
    const uint32_t bits = byte << 23;
    return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : bits);
}


// ---- activation checkpoints: eight E4M3 codes of a lane in two words, four neighbouring lanes hold a block ----

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// Rounded to nearest, ties to even, with the least k for which the block's largest is at most 448 2^k.  At the largest k that a type needs, 240 2^k is the last multiple within its
// range, and magnitudes beyond become that: what is finite stays so in its own type.  The scale is the same in the block's lanes; of a block that is not a number the codes mean nothing.
template <int DT> __device__ __forceinline__ u32x2_t encode_e4m3(const float (&v)[8], uint32_t &scale)
{
    constexpr uint32_t kLast = DT == DQ_F16 ? 127 + 8 : 127 + 120;
    scale = block_scale<8, 0x600000u>(block_max(v));
    const float down = scale_down(scale), most = scale == kLast ? 240.0f : 448.0f;
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = __builtin_amdgcn_fmed3f(v[j] * down, -most, most);
    u32x2_t w;
    w[0] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
    w[1] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false), true);
    return w;
}
__device__ __forceinline__ void decode_e4m3(u32x2_t w, uint32_t scale, float (&v)[8])
{
    const float up = scale_up(scale);
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(w[k], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w[k], true);
        v[4 * k] = a.x * up; v[4 * k + 1] = a.y * up; v[4 * k + 2] = b.x * up; v[4 * k + 3] = b.y * up;
    }
}

// a checkpoint's buffer: codes [rows][32 blocks], scales [rows][blocks]
template <class BYTE> struct CheckpointOf {
    BYTE *codes, *scales;
    uint32_t blocks;
    __host__ __device__ __forceinline__ CheckpointOf(BYTE *data, int64_t rows, uint32_t cols) : codes(data), scales(data + rows * ((cols + 31) >> 5) * 32), blocks((cols + 31) >> 5) {}
};

} // namespace dq
