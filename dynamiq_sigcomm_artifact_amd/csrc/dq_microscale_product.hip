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
    uint32_t tiles_n;
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

// ---- many rows: tiles through LDS --------------------------------------------------------------------------

// 16 (4) bytes a lane from base + offset to LDS, lane after lane from byte `to` on.  Written out: the compiler takes a read of any part of LDS for one of
// what is on its way there, and waits.  Whoever reads waits for vmcnt himself.
__device__ __forceinline__ void load_lds16(const uint8_t *base, uint32_t offset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(to));
}
__device__ __forceinline__ void load_lds4(const uint8_t *base, uint32_t offset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(base), "s"(to));
}

// Which tile a workgroup takes.  Workgroups go to the eight XCDs in turn; each XCD gets a run of tiles that lie together, four rows of tiles high, so that
// what its 32 CUs work on at a time shares operands in its L2.
__device__ __forceinline__ uint2 tile_of(uint32_t id, uint32_t tiles, uint32_t tiles_m, uint32_t tiles_n)
{
    const uint32_t xcd = id & 7, each = tiles >> 3, more = tiles & 7;
    const uint32_t k = xcd * each + min(xcd, more) + (id >> 3);
    const uint32_t band = k / (4 * tiles_n), in_band = k - band * 4 * tiles_n;
    const uint32_t high = min(4u, tiles_m - 4 * band);
    // (divided in vector registers, the same in every lane)
    return make_uint2(__builtin_amdgcn_readfirstlane(4 * band + in_band % high), __builtin_amdgcn_readfirstlane(in_band / high));
}

// A workgroup of four waves, 2 x 2, takes a tile of T x T, superchunk by superchunk: rows of 128 bytes of codes and 8 of scales, which lie in LDS twice, one
// being computed with while the next arrives.  Piece b of row r lies in slot b ^ (r / 2 % 8): the sixteen lanes that read at a time, one piece of sixteen rows,
// then find sixteen different groups of banks.  The operands of a step are read during the products of the step before; the waves meet before the last step
// of a superchunk, when everything of it is in registers.
template <int DT, int T> __global__ __launch_bounds__(256, T == 256 ? 1 : 2) void mx4_tile_kernel(ProductArgs p)
{
    constexpr int F = T / 64; // 32 x 32 products of a wave, each way
    constexpr int kCodes = T * 128, kScales = T * 8, kStage = 2 * (kCodes + kScales);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kStage];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), half = lane >> 5;
    const uint2 at = tile_of(blockIdx.x, gridDim.x, (uint32_t)((p.m + T - 1) / T), p.tiles_n);
    const int64_t i0 = (int64_t)at.x * T, j0 = (int64_t)at.y * T;
    const uint32_t pitch = p.superchunks * 128u, scale_pitch = p.superchunks * 8u;

    // what this lane fetches: pieces of 16 bytes, eight rows a wave and instruction; scale words, 32 rows likewise.  Rows past the end are the last one's.
    constexpr int kLoads = T / 32, kScaleLoads = T / 128;
    uint32_t from_a[kLoads], from_b[kLoads], scale_a[kScaleLoads], scale_b[kScaleLoads];
#pragma unroll
    for (int k = 0; k < kLoads; k++) {
        const int r = 8 * (4 * k + wave) + (lane >> 3);
        const uint32_t piece = ((lane & 7) ^ (r >> 1 & 7)) * 16;
        from_a[k] = (uint32_t)min((int64_t)r, p.m - 1 - i0) * pitch + piece;
        from_b[k] = (uint32_t)min((int64_t)r, p.n - 1 - j0) * pitch + piece;
    }
#pragma unroll
    for (int k = 0; k < kScaleLoads; k++) {
        const int r = 32 * (4 * k + wave) + (lane >> 1);
        scale_a[k] = (uint32_t)min((int64_t)r, p.m - 1 - i0) * scale_pitch + 4 * (lane & 1);
        scale_b[k] = (uint32_t)min((int64_t)r, p.n - 1 - j0) * scale_pitch + 4 * (lane & 1);
    }
    const uint8_t *a = p.a_codes + i0 * pitch, *b = p.b_codes + j0 * pitch;
    const uint8_t *as = p.a_scales + i0 * scale_pitch, *bs = p.b_scales + j0 * scale_pitch;
    const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    constexpr int kParts = 2 * (kLoads + kScaleLoads);
    auto fetch_part = [&](uint32_t stage, int part) {
        const uint32_t to = lds_at + stage;
        const int k = part >> 1;
        if (k < kLoads) {
            if (part & 1)
                load_lds16(b, from_b[k], to + kCodes + 1024 * (4 * k + wave));
            else
                load_lds16(a, from_a[k], to + 1024 * (4 * k + wave));
        } else {
            if (part & 1)
                load_lds4(bs, scale_b[k - kLoads], to + 2 * kCodes + kScales + 256 * (4 * (k - kLoads) + wave));
            else
                load_lds4(as, scale_a[k - kLoads], to + 2 * kCodes + 256 * (4 * (k - kLoads) + wave));
        }
    };
    auto fetched = [&] { a += 128, b += 128, as += 8, bs += 8; };
    auto fetch = [&](uint32_t stage) {
#pragma unroll
        for (int k = 0; k < kParts; k++) fetch_part(stage, k);
        fetched();
    };

    f32x16 acc[F][F] = {};
    uint4 x[2][F], y[2][F];
    int sa[F], sb[F], next_sa[F], next_sb[F];
    const int ra = (wave >> 1) * (T / 2) + (lane & 31), rb = (wave & 1) * (T / 2) + (lane & 31);
    const uint8_t *at_a = lds + ra * 128, *at_b = lds + kCodes + rb * 128, *at_sa = lds + 2 * kCodes + ra * 8 + 4 * half,
                  *at_sb = lds + 2 * kCodes + kScales + rb * 8 + 4 * half;
    uint32_t slot[4];
#pragma unroll
    for (int k = 0; k < 4; k++) slot[k] = ((4 * half + k) ^ (lane >> 1 & 7)) * 16;
    auto read = [&](int to, int step, uint32_t stage) {
#pragma unroll
        for (int f = 0; f < F; f++) {
            x[to][f] = *reinterpret_cast<const uint4 *>(at_a + stage + slot[step] + 4096 * f);
            y[to][f] = *reinterpret_cast<const uint4 *>(at_b + stage + slot[step] + 4096 * f);
        }
    };
    // every wave has what it fetched, and is done with what it read
    auto meet = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
#define DQ_PRODUCTS(FROM, S)                                                                                                                    \
    _Pragma("unroll") for (int f = 0; f < F; f++)                                                                                               \
        _Pragma("unroll") for (int h = 0; h < F; h++)                                                                                           \
            acc[f][h] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(y[FROM][h]), operand(x[FROM][f]), acc[f][h], 4, 4, S, sb[h], S, sa[f]);
    // one read, then as many products as there are to a read
#define DQ_INTERLEAVE(READS)                                                                                                                    \
    _Pragma("unroll") for (int k = 0; k < 2 * F; k++) {                                                                                         \
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);                                                                                  \
        __builtin_amdgcn_sched_group_barrier(0x008, F / 2, 0);                                                                                  \
    }                                                                                                                                           \
    __builtin_amdgcn_sched_barrier(0);
    fetch(0);
    meet();
    if (p.superchunks > 1) fetch(kStage);
    read(0, 0, 0);
#pragma unroll
    for (int f = 0; f < F; f++) {
        next_sa[f] = *reinterpret_cast<const int *>(at_sa + 256 * f);
        next_sb[f] = *reinterpret_cast<const int *>(at_sb + 256 * f);
    }
    uint32_t stage = 0;
    // (one block of code each, without a branch: products would wander behind it)
#define DQ_SUPERCHUNK(FETCH)                                                                                                                    \
    {                                                                                                                                           \
        _Pragma("unroll") for (int f = 0; f < F; f++) sa[f] = next_sa[f], sb[f] = next_sb[f];                                                   \
        read(1, 1, stage);                                                                                                                      \
        DQ_PRODUCTS(0, 0)                                                                                                                       \
        DQ_INTERLEAVE(1)                                                                                                                        \
        read(0, 2, stage);                                                                                                                      \
        DQ_PRODUCTS(1, 1)                                                                                                                       \
        DQ_INTERLEAVE(1)                                                                                                                        \
        read(1, 3, stage);                                                                                                                      \
        DQ_PRODUCTS(0, 2)                                                                                                                       \
        DQ_INTERLEAVE(1)                                                                                                                        \
        meet();                                                                                                                                 \
        const uint32_t free_stage = stage;                                                                                                      \
        stage = kStage - stage;                                                                                                                 \
        /* the first operands of the next superchunk, and what is fetched for the one after it, between the last products of this one */       \
        _Pragma("unroll") for (int f = 0; f < F; f++)                                                                                           \
        {                                                                                                                                       \
            x[0][f] = *reinterpret_cast<const uint4 *>(at_a + stage + slot[0] + 4096 * f);                                                      \
            y[0][f] = *reinterpret_cast<const uint4 *>(at_b + stage + slot[0] + 4096 * f);                                                      \
            next_sa[f] = *reinterpret_cast<const int *>(at_sa + stage + 256 * f);                                                               \
            next_sb[f] = *reinterpret_cast<const int *>(at_sb + stage + 256 * f);                                                               \
            _Pragma("unroll") for (int h = 0; h < F; h++)                                                                                       \
            {                                                                                                                                   \
                acc[f][h] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(y[1][h]), operand(x[1][f]), acc[f][h], 4, 4, 3, sb[h], 3, sa[f]); \
                if (FETCH) {                                                                                                                    \
                    _Pragma("unroll") for (int k = (F * f + h) * kParts / (F * F); k < (F * f + h + 1) * kParts / (F * F); k++) fetch_part(free_stage, k); \
                }                                                                                                                               \
                __builtin_amdgcn_sched_barrier(0);                                                                                              \
            }                                                                                                                                   \
        }                                                                                                                                       \
        if (FETCH) fetched();                                                                                                                   \
    }
    for (int s = 2; s < p.superchunks; s++) DQ_SUPERCHUNK(true)
    if (p.superchunks > 1) DQ_SUPERCHUNK(false)
    DQ_SUPERCHUNK(false) // (what it reads ahead is of the superchunk before, and not used)
#undef DQ_SUPERCHUNK
#undef DQ_PRODUCTS
#undef DQ_INTERLEAVE
    // The result leaves through LDS as runs of whole rows: 32 rows x T / 2 columns of a wave at a time.  (All waves have passed the last meeting: what lay there
    // is in registers.)  A lane writes four columns of a row; rows are 16 bytes further apart than long, so that sixteen of them use all banks.
    typedef typename ElemIO<DT>::storage Elem;
    constexpr int kRow = T / 2 * sizeof(Elem), kApart = kRow + 16, kPer = 16 / sizeof(Elem), kLanes = kRow / 16;
    static_assert(4 * 32 * kApart <= 2 * kStage, "the waves' rows fit");
    uint8_t *mine = lds + wave * 32 * kApart;
    const int64_t col0 = j0 + (wave & 1) * (T / 2) + lane % kLanes * kPer;
#pragma unroll
    for (int f = 0; f < F; f++) {
#pragma unroll
        for (int h = 0; h < F; h++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint8_t *to = mine + (lane & 31) * kApart + (32 * h + 8 * k + 4 * half) * sizeof(Elem);
                const f32x16 v = acc[f][h];
                if (DT == DQ_F32)
                    *reinterpret_cast<float4 *>(to) = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                else if (DT == DQ_BF16)
                    *reinterpret_cast<uint2 *>(to) = make_uint2(f32x2_to_bf16x2(v[4 * k], v[4 * k + 1]), f32x2_to_bf16x2(v[4 * k + 2], v[4 * k + 3]));
                else
                    *reinterpret_cast<uint2 *>(to) = make_uint2(f32_to_f16_bits(v[4 * k]) | f32_to_f16_bits(v[4 * k + 1]) << 16,
                                                                f32_to_f16_bits(v[4 * k + 2]) | f32_to_f16_bits(v[4 * k + 3]) << 16);
            }
        wave_lds_sync();
#pragma unroll
        for (int k = 0; k < 32 * kLanes / 64; k++) {
            const int r = 64 / kLanes * k + lane / kLanes;
            const int64_t i = i0 + (wave >> 1) * (T / 2) + 32 * f + r;
            const uint4 v = *reinterpret_cast<const uint4 *>(mine + r * kApart + lane % kLanes * 16);
            if (i < p.m) {
                Elem *to = static_cast<Elem *>(p.out) + i * p.n + col0;
                if (col0 + kPer <= p.n) {
                    const u32x4_any w = {v.x, v.y, v.z, v.w};
                    *reinterpret_cast<u32x4_any *>(to) = w;
                } else {
                    const Elem *e = reinterpret_cast<const Elem *>(&v);
#pragma unroll
                    for (int c = 0; c < kPer; c++)
                        if (col0 + c < p.n) to[c] = e[c];
                }
            }
        }
        wave_lds_sync();
    }
}

template <int DT> static hipError_t launch_product(ProductArgs p, hipStream_t stream)
{
    if (p.m > 64) {
        const int tile = 256;
        p.tiles_n = (uint32_t)((p.n + tile - 1) / tile);
        const dim3 grid((uint32_t)((p.m + tile - 1) / tile) * p.tiles_n);
        return launch_with(mx4_tile_kernel<DT, 256>, grid, dim3(256), stream, p);
    }
    const dim3 grid((uint32_t)((p.n + 31) >> 5), (uint32_t)((p.m + 31) >> 5));
    return launch_with(mx4_product_kernel<DT>, grid, dim3(64), stream, p);
}

hipError_t launch_mx4_product(const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes, const uint8_t *b_scales, void *out, int64_t m,
                              int64_t n, int64_t k, int dtype, hipStream_t stream)
{
    const ProductArgs p = {a_codes, a_scales, b_codes, b_scales, out, m, n, (int)((k + 255) >> 8), 0};
    return dtype == DQ_F32 ? launch_product<DQ_F32>(p, stream) : dtype == DQ_BF16 ? launch_product<DQ_BF16>(p, stream) : launch_product<DQ_F16>(p, stream);
}

} // namespace dq
