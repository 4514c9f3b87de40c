// Products of 4-bit microscaled matrices on the matrix cores.
#include "dq_launch.h"
#include "dq_microscale.cuh"

namespace dq {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct ProductArgs {
    const uint8_t *a_codes, *a_scales, *b_codes, *b_scales;
    void *out;
    int64_t m, n, out_pitch;
    int superchunks;
    uint32_t tiles_n;
};
struct NarrowArgs : ProductArgs {
    int dtype;
};

__device__ __forceinline__ i32x8 operand(uint4 v)
{
    i32x8 x = {(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
    return x;
}

// ---- few rows, or a small result: operands straight from memory -------------------------------------------------

// v_mfma_scale_f32_16x16x128_f8f6f4 on E2M1: lane l holds 32 consecutive elements, one block, of row l % 16, and its scale is byte S of its scale word.  The order of
// the contraction is free as long as both sides keep it: of a superchunk's eight blocks the lanes l / 16 = g take blocks 2 g and 2 g + 1, so that what a lane
// loads is 32 bytes of codes in a row and two of scales.
struct Rows16 {
    uint4 codes[2];
    int scales;
    __device__ __forceinline__ void load(const uint8_t *c, const uint8_t *s)
    {
        codes[0] = reinterpret_cast<const uint4 *>(c)[0];
        codes[1] = reinterpret_cast<const uint4 *>(c)[1];
        scales = *reinterpret_cast<const uint16_t *>(s);
    }
};

// A workgroup takes 16 MF x 16 NF of the result; its waves share the superchunks out, one after the other, and add their sums up in LDS, in the order of the
// waves.  Bound by memory, or by the time to the first byte: every wave has U superchunks on their way at a time.  1 x 14336 x 4096: 31 MB of codes and scales in 8.4 us,
// 3.7 TB/s, some 3 of it the launch and the first load; 1 x 4096 x 4096 in 5.1.
template <int MF, int NF, int W, int U> __global__ __launch_bounds__(64 * W) void mx4_narrow_kernel(NarrowArgs p)
{
    __shared__ __attribute__((aligned(16))) float sums[W][MF * NF][64][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, group = lane >> 4;
    const int64_t i0 = (int64_t)(blockIdx.x / p.tiles_n) * (16 * MF), j0 = (int64_t)(blockIdx.x % p.tiles_n) * (16 * NF);
    const uint8_t *a[MF], *as[MF], *b[NF], *bs[NF];
#pragma unroll
    for (int f = 0; f < MF; f++) {
        const int64_t at = min(i0 + 16 * f + row, p.m - 1) * p.superchunks + wave;
        a[f] = p.a_codes + at * 128 + group * 32;
        as[f] = p.a_scales + at * 8 + group * 2;
    }
#pragma unroll
    for (int h = 0; h < NF; h++) {
        const int64_t at = min(j0 + 16 * h + row, p.n - 1) * p.superchunks + wave;
        b[h] = p.b_codes + at * 128 + group * 32;
        bs[h] = p.b_scales + at * 8 + group * 2;
    }
    f32x4 acc[MF][NF] = {};
    auto products = [&](const Rows16 (&x)[MF], const Rows16 (&y)[NF]) {
#pragma unroll
        for (int f = 0; f < MF; f++)
#pragma unroll
            for (int h = 0; h < NF; h++) {
                acc[f][h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(y[h].codes[0]), operand(x[f].codes[0]), acc[f][h], 4, 4, 0, y[h].scales, 0, x[f].scales);
                acc[f][h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(y[h].codes[1]), operand(x[f].codes[1]), acc[f][h], 4, 4, 1, y[h].scales, 1, x[f].scales);
            }
    };
    int s = wave;
    for (; s + (U - 1) * W < p.superchunks; s += U * W) {
        Rows16 x[U][MF], y[U][NF];
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int h = 0; h < NF; h++) y[u][h].load(b[h] + u * W * 128, bs[h] + u * W * 8);
#pragma unroll
            for (int f = 0; f < MF; f++) x[u][f].load(a[f] + u * W * 128, as[f] + u * W * 8);
        }
#pragma unroll
        for (int u = 0; u < U; u++) products(x[u], y[u]);
#pragma unroll
        for (int h = 0; h < NF; h++) b[h] += U * W * 128, bs[h] += U * W * 8;
#pragma unroll
        for (int f = 0; f < MF; f++) a[f] += U * W * 128, as[f] += U * W * 8;
    }
    for (; s < p.superchunks; s += W) {
        Rows16 x[MF], y[NF];
#pragma unroll
        for (int h = 0; h < NF; h++) {
            y[h].load(b[h], bs[h]);
            b[h] += W * 128, bs[h] += W * 8;
        }
#pragma unroll
        for (int f = 0; f < MF; f++) {
            x[f].load(a[f], as[f]);
            a[f] += W * 128, as[f] += W * 8;
        }
        products(x, y);
    }
#pragma unroll
    for (int f = 0; f < MF; f++)
#pragma unroll
        for (int h = 0; h < NF; h++) *reinterpret_cast<f32x4 *>(sums[wave][f * NF + h][lane]) = acc[f][h];
    __syncthreads();
    // b is the left operand: what a lane holds are four consecutive columns of a row of the result
#pragma unroll
    for (int k = 0; k < (MF * NF + W - 1) / W; k++) {
        const int block = k * W + wave;
        if (MF * NF % W != 0 && block >= MF * NF) continue;
        f32x4 v = *reinterpret_cast<const f32x4 *>(sums[0][block][lane]);
#pragma unroll
        for (int w = 1; w < W; w++) v += *reinterpret_cast<const f32x4 *>(sums[w][block][lane]);
        const int64_t i = i0 + 16 * (block / NF) + row, j = j0 + 16 * (block % NF) + 4 * group;
        if (i >= p.m) continue;
        const int64_t to = i * p.n + j;
        if (j + 4 <= p.n) {
            if (p.dtype == DQ_F32) {
                *reinterpret_cast<f32x4_any *>(static_cast<float *>(p.out) + to) = v;
            } else {
                typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
                u32x2_any w;
                if (p.dtype == DQ_BF16)
                    w = u32x2_any{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
                else
                    w = u32x2_any{f32_to_f16_bits(v[0]) | f32_to_f16_bits(v[1]) << 16, f32_to_f16_bits(v[2]) | f32_to_f16_bits(v[3]) << 16};
                *reinterpret_cast<u32x2_any *>(static_cast<uint16_t *>(p.out) + to) = w;
            }
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (j + c < p.n) {
                    if (p.dtype == DQ_F32)
                        ElemIO<DQ_F32>::store(p.out, to + c, v[c]);
                    else if (p.dtype == DQ_BF16)
                        ElemIO<DQ_BF16>::store(p.out, to + c, v[c]);
                    else
                        ElemIO<DQ_F16>::store(p.out, to + c, v[c]);
                }
        }
    }
}

// ---- many rows: tiles through LDS --------------------------------------------------------------------------

// 16 bytes a lane from base + offset to LDS, lane after lane from byte `to` on.  Written out: the compiler takes a read of any part of LDS for one of
// what is on its way there, and waits.  Whoever reads waits for vmcnt himself.
__device__ __forceinline__ void load_lds16(const uint8_t *base, uint32_t offset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(to) : "m0");
}

// Which tile a workgroup takes: an XCD's run of tiles is four rows of them high.
__device__ __forceinline__ uint2 tile_of(uint32_t id, uint32_t tiles, uint32_t tiles_m, uint32_t tiles_n)
{
    const uint32_t k = unit_of(id, tiles);
    const uint32_t band = k / (4 * tiles_n), in_band = k - band * 4 * tiles_n;
    const uint32_t high = min(4u, tiles_m - 4 * band);
    // (divided in vector registers, the same in every lane)
    return make_uint2(__builtin_amdgcn_readfirstlane(4 * band + in_band % high), __builtin_amdgcn_readfirstlane(in_band / high));
}

// A workgroup of four waves, 2 x 2, takes a tile of T x T, superchunk by superchunk: rows of 128 bytes of codes, which lie in LDS twice, one being computed with
// while the next arrives.  Piece b of row r lies in slot b ^ (r / 2 % 8): the sixteen lanes that read at a time, one piece of sixteen rows, then find sixteen
// different groups of banks.  The operands of a step are read during the products of the step before; the waves meet before the last step of a superchunk,
// when everything of it is in registers.  Scales come for four superchunks at a time, 32 bytes a row.
// A wave does 16 products of 32 x 32 x 64 per step, 512 cycles, and spends 800, 535, 535 and 800 on the four steps and 120 on the meeting: 4.4 PFLOP/s at 4096 x 4096 x 14336, at
// the 1.8 to 2.0 GHz that the power limit leaves (products alone, from registers, reach 6.0 to 6.5 on such data).  8192 x 14336 x 4096 in 252 us, 3.8 PFLOP/s: of a tile's
// 36 us some 2 are its first fetch and 4 its stores.  A workgroup that goes on to the next tile while it stores one gains 2 % there and loses 5 % with short contractions.
template <int DT, int T> __global__ __launch_bounds__(256, T == 256 ? 1 : 2) void mx4_tile_kernel(ProductArgs p)
{
    constexpr int F = T / 64; // 32 x 32 products of a wave, each way
    constexpr int kCodes = T * 128, kStage = 2 * kCodes, kScales = T * 32, kScaleGroup = 2 * kScales;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * (kStage + kScaleGroup)];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), half = lane >> 5;
    const uint2 at = tile_of(blockIdx.x, gridDim.x, (uint32_t)((p.m + T - 1) / T), p.tiles_n);
    const int64_t i0 = (int64_t)at.x * T, j0 = (int64_t)at.y * T;
    const uint32_t pitch = p.superchunks * 128u, scale_pitch = p.superchunks * 8u;

    // what this lane fetches: pieces of 16 bytes, eight rows a wave and instruction.  Rows past the end are the last one's.
    constexpr int kLoads = T / 32, kParts = 2 * kLoads;
    uint32_t from_a[kLoads], from_b[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; k++) {
        const int r = 8 * (4 * k + wave) + (lane >> 3);
        const uint32_t piece = ((lane & 7) ^ (r >> 1 & 7)) * 16;
        from_a[k] = (uint32_t)min((int64_t)r, p.m - 1 - i0) * pitch + piece;
        from_b[k] = (uint32_t)min((int64_t)r, p.n - 1 - j0) * pitch + piece;
    }
    const uint8_t *a = p.a_codes + i0 * pitch, *b = p.b_codes + j0 * pitch;
    const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    auto fetch_part = [&](uint32_t stage, int part) {
        const uint32_t to = lds_at + stage;
        const int k = part >> 1;
        if (part & 1)
            load_lds16(b, from_b[k], to + kCodes + 1024 * (4 * k + wave));
        else
            load_lds16(a, from_a[k], to + 1024 * (4 * k + wave));
    };
    auto fetched = [&] { a += 128, b += 128; };
    // Part j of the scales of superchunks 4 g .. 4 g + 3: 32 rows a wave and instruction, two lanes a row.  A row's last piece may reach into the next row; the last
    // row's begins eight bytes earlier instead.
    constexpr int kScaleParts = T / 64;
    auto fetch_scales = [&](uint32_t g, uint32_t j) {
        const bool of_b = j & 1;
        const uint32_t k = 4 * (j >> 1 & (kScaleParts / 2 - 1)) + wave, last = (uint32_t)(of_b ? p.n : p.m) - 1;
        const uint32_t row = min((uint32_t)(of_b ? j0 : i0) + 32 * k + (lane >> 1), last);
        load_lds16(of_b ? p.b_scales : p.a_scales, min(row * scale_pitch + 32 * g + 16 * (lane & 1), (last + 1) * scale_pitch - 16),
                   lds_at + 2 * kStage + (g & 1) * kScaleGroup + (of_b ? kScales : 0) + 1024 * k);
    };

    f32x16 acc[F][F] = {};
    uint4 x[2][F], y[2][F];
    int sa[F], sb[F], next_sa[F], next_sb[F];
    const int ra = (wave >> 1) * (T / 2) + (lane & 31), rb = (wave & 1) * (T / 2) + (lane & 31);
    const uint8_t *at_a = lds + ra * 128, *at_b = lds + kCodes + rb * 128, *at_sa = lds + 2 * kStage + ra * 32 + 4 * half, *at_sb = lds + 2 * kStage + kScales + rb * 32 + 4 * half;
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
    // the scales of superchunk s; last: s is the last one, and odd numbers of them end in half a piece
    auto read_scales = [&](int f, uint32_t s, bool last) {
        const uint32_t from = (s >> 2 & 1) * kScaleGroup + 8 * (s & 3) + 1024 * f;
        const bool odd = last && p.superchunks & 1;
        next_sa[f] = *reinterpret_cast<const int *>(at_sa + from + (odd && i0 + ra + 32 * f >= p.m - 1 ? 8 : 0));
        next_sb[f] = *reinterpret_cast<const int *>(at_sb + from + (odd && j0 + rb + 32 * f >= p.n - 1 ? 8 : 0));
    };
    // every wave has what it fetched, and is done with what it read
    auto meet = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // Products of step S from operands FROM, the next step's operands read between them, and parts LOW .. HIGH of what is fetched to stage TO
#define DQ_STEP(S, FROM, NEXT, STAGE, GO, TO, LOW, HIGH, MORE)                                                                                  \
    _Pragma("unroll") for (int f = 0; f < F; f++)                                                                                               \
    {                                                                                                                                           \
        x[1 - FROM][f] = *reinterpret_cast<const uint4 *>(at_a + STAGE + slot[NEXT] + 4096 * f);                                                \
        y[1 - FROM][f] = *reinterpret_cast<const uint4 *>(at_b + STAGE + slot[NEXT] + 4096 * f);                                                \
        MORE;                                                                                                                                   \
        _Pragma("unroll") for (int h = 0; h < F; h++)                                                                                           \
        {                                                                                                                                       \
            acc[f][h] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(y[FROM][h]), operand(x[FROM][f]), acc[f][h], 4, 4, S, sb[h], S, sa[f]); \
            if (GO) {                                                                                                                           \
                _Pragma("unroll") for (int k = (LOW) + (F * f + h) * ((HIGH) - (LOW)) / (F * F); k < (LOW) + (F * f + h + 1) * ((HIGH) - (LOW)) / (F * F); k++) \
                    fetch_part(TO, k);                                                                                                          \
            }                                                                                                                                   \
            __builtin_amdgcn_sched_barrier(0);                                                                                                  \
        }                                                                                                                                       \
    }
#define DQ_PRODUCTS(FROM, S)                                                                                                                    \
    _Pragma("unroll") for (int f = 0; f < F; f++)                                                                                               \
        _Pragma("unroll") for (int h = 0; h < F; h++)                                                                                           \
            acc[f][h] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(y[FROM][h]), operand(x[FROM][f]), acc[f][h], 4, 4, S, sb[h], S, sa[f]);
    // one read, then as many products as there are to a read
#define DQ_INTERLEAVE                                                                                                                           \
    _Pragma("unroll") for (int k = 0; k < 2 * F; k++) {                                                                                         \
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                                                                      \
        __builtin_amdgcn_sched_group_barrier(0x008, F / 2, 0);                                                                                  \
    }                                                                                                                                           \
    __builtin_amdgcn_sched_barrier(0);
    // A fetching instruction keeps a wave for 64 cycles, the time of two products (the four waves share 64 bytes a cycle), and waits for its turn: twenty in one
    // step, scales among them, took 1280 cycles where its products take 512.  So the fetches for superchunk s + 2 begin behind the meeting of s, in its last
    // step, and end in the first step of s + 1, and scales, as dear by the row as codes, come once in four superchunks: 4096 x 4096 x 14336 in 110 us instead of 126.
    constexpr int kFirst = kParts / 2;
    const int n = p.superchunks;
#pragma unroll
    for (int k = 0; k < kParts; k++) fetch_part(0, k);
    fetched();
#pragma unroll
    for (int j = 0; j < kScaleParts; j++) fetch_scales(0, j);
    fetch_scales(1, 0);
    meet();
    if (n > 1) {
#pragma unroll
        for (int k = 0; k < kFirst; k++) fetch_part(kStage, k);
    }
    read(0, 0, 0);
#pragma unroll
    for (int f = 0; f < F; f++) read_scales(f, 0, n == 1);
    uint32_t stage = 0;
    // (one block of code each, without a branch: products would wander behind it)
#define DQ_SUPERCHUNK(REST, FETCH)                                                                                                              \
    {                                                                                                                                           \
        _Pragma("unroll") for (int f = 0; f < F; f++) sa[f] = next_sa[f], sb[f] = next_sb[f];                                                   \
        const uint32_t other = kStage - stage;                                                                                                  \
        DQ_STEP(0, 0, 1, stage, REST, other, kFirst, kParts, )                                                                                  \
        if (REST) fetched();                                                                                                                    \
        read(0, 2, stage);                                                                                                                      \
        DQ_PRODUCTS(1, 1)                                                                                                                       \
        DQ_INTERLEAVE                                                                                                                           \
        read(1, 3, stage);                                                                                                                      \
        DQ_PRODUCTS(0, 2)                                                                                                                       \
        DQ_INTERLEAVE                                                                                                                           \
        meet();                                                                                                                                 \
        if (FETCH) fetch_scales((s + 1) / 4 + 1, s + 1);                                                                                        \
        DQ_STEP(3, 1, 0, other, FETCH, stage, 0, kFirst, read_scales(f, s + 1, !(FETCH)))                                                       \
        stage = other;                                                                                                                          \
    }
    int s = 0;
    for (; s < n - 2; s++) DQ_SUPERCHUNK(true, true)
    if (n > 1) {
        DQ_SUPERCHUNK(true, false)
        s++;
    }
    DQ_SUPERCHUNK(false, false) // (what it reads ahead is of the superchunk before, and not used)
#undef DQ_SUPERCHUNK
#undef DQ_STEP
#undef DQ_PRODUCTS
#undef DQ_INTERLEAVE
    // The result leaves through LDS as runs of whole rows: 32 rows x T / 2 columns of a wave at a time.  (All waves have passed the last meeting: what lay there
    // is in registers.)  A lane writes four columns of a row; rows are 16 bytes further apart than long, so that sixteen of them use all banks.
    typedef typename ElemIO<DT>::storage Elem;
    constexpr int kRow = T / 2 * sizeof(Elem), kApart = kRow + 16, kPer = 16 / sizeof(Elem), kLanes = kRow / 16;
    static_assert(4 * 32 * kApart <= 2 * (kStage + kScaleGroup), "the waves' rows fit");
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
                Elem *to = static_cast<Elem *>(p.out) + i * p.out_pitch + col0;
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

template <int MF, int NF, int W, int U> static hipError_t launch_narrow(const ProductArgs &p, int dtype, hipStream_t stream)
{
    NarrowArgs a;
    static_cast<ProductArgs &>(a) = p;
    a.dtype = dtype;
    a.tiles_n = (uint32_t)((p.n + 16 * NF - 1) / (16 * NF));
    return launch_with(mx4_narrow_kernel<MF, NF, W, U>, dim3((uint32_t)((p.m + 16 * MF - 1) / (16 * MF)) * a.tiles_n), dim3(64 * W), stream, a);
}

template <int DT, int T> static hipError_t launch_tiles(ProductArgs p, hipStream_t stream)
{
    p.tiles_n = (uint32_t)((p.n + T - 1) / T);
    return launch_with(mx4_tile_kernel<DT, T>, dim3((uint32_t)((p.m + T - 1) / T) * p.tiles_n), dim3(256), stream, p);
}

template <int T> static hipError_t launch_tiles_of(const ProductArgs &p, int dtype, hipStream_t stream)
{
    return dtype == DQ_F32 ? launch_tiles<DQ_F32, T>(p, stream) : dtype == DQ_BF16 ? launch_tiles<DQ_BF16, T>(p, stream) : launch_tiles<DQ_F16, T>(p, stream);
}

// Which kernel.  Two tiles of 128 x 128 share a CU, and 512 of them run at a time; tiles of 256 x 256 fetch half as much per product, but one takes a CU.  Where 512
// suffice they are the faster (2048 x 4096 x 4096, 512 tiles: 24.0 us, tiles of 256: 29.7), and slower beyond (2304 x 4096 x 4096, 576 tiles: 34.3 and 29.1 us).
// Below 40 tiles of 128 the contraction is shared out among the waves of a workgroup instead (256 x 3000 x 4096, 48 tiles: 12.6 us, shared out 20.2; 128 x 4096 x 4096,
// 32 tiles: 10.8 and 11.2; 128 x 2048 x 4096, 16 tiles: 10.7 and 7.9), with less than four superchunks, which a tile's two barriers and stores outlast, below 96
// (776 x 1000 x 333, 56 tiles: 6.4 and 4.8; 1024 x 1024 x 1024, 64 tiles: 5.4 and 6.6), in the largest blocks that leave 192 workgroups: with fewer, CUs have nothing to do
// (16 x 4096 x 4096, blocks of 16 x 16: 5.4 us, 16 x 64: 9.2), with more the operands are read more often (16 x 14336 x 4096: 13.3 and 9.6 us; 1 x 14336 x 4096: 9.3 and
// 8.4).  No block is twice as high or wide as it need be.
template <int MF, int NF, int U> static bool try_narrow(const ProductArgs &p, bool last, int dtype, hipStream_t stream, hipError_t &e)
{
    const int64_t blocks = ((p.m + 16 * MF - 1) / (16 * MF)) * ((p.n + 16 * NF - 1) / (16 * NF));
    if (!last && (blocks < 192 || (MF > 1 && 8 * MF >= p.m) || (NF > 1 && 8 * NF >= p.n))) return false;
    e = launch_narrow<MF, NF, 8, U>(p, dtype, stream);
    return true;
}

hipError_t launch_mx4_product(const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes, const uint8_t *b_scales, void *out, int64_t m,
                              int64_t n, int64_t k, int dtype, hipStream_t stream)
{
    const ProductArgs p = {a_codes, a_scales, b_codes, b_scales, out, m, n, n, (int)((k + 255) >> 8), 0};
    const auto tiles = [&](int64_t t) { return ((m + t - 1) / t) * ((n + t - 1) / t); };
    if (m > 64 && n > 64 && tiles(128) > 512) {
        // A last round of tiles of 256 in which less than half of the CUs have work takes as long as a full one; the same in tiles of 128, two to a CU, two thirds of
        // that.  So the longer side is cut where whole rounds end, and the rest is a launch of its own (3000 x 6000 x 4096, 288 tiles: 51 us instead of 62; 4352 x 4352 x 8192,
        // 289: 87 for 100; with half a round left, 4096 x 14336 x 4096, 138 for 140).  Short contractions do not make up for the launch.
        const bool along_n = n >= m;
        const int64_t side = ((along_n ? n : m) + 255) / 256, across = ((along_n ? m : n) + 255) / 256, whole = side * across / 256 * 256 / across;
        if (p.superchunks >= 8 && whole > 0 && (side - whole) * across <= 128 && whole < side) {
            ProductArgs first = p, rest = p;
            const int64_t cut = whole * 256;
            const int64_t row = (int64_t)p.superchunks;
            if (along_n) {
                first.n = cut;
                rest.n = n - cut;
                rest.b_codes += cut * row * 128;
                rest.b_scales += cut * row * 8;
                rest.out = static_cast<char *>(out) + cut * (dtype == DQ_F32 ? 4 : 2);
            } else {
                first.m = cut;
                rest.m = m - cut;
                rest.a_codes += cut * row * 128;
                rest.a_scales += cut * row * 8;
                rest.out = static_cast<char *>(out) + cut * n * (dtype == DQ_F32 ? 4 : 2);
            }
            const hipError_t e = launch_tiles_of<256>(first, dtype, stream);
            return e != hipSuccess ? e : launch_tiles_of<128>(rest, dtype, stream);
        }
        return launch_tiles_of<256>(p, dtype, stream);
    }
    if (m > 64 && n > 64 && tiles(128) >= (p.superchunks < 4 ? 96 : 40))
        return launch_tiles_of<128>(p, dtype, stream);
    hipError_t e = hipSuccess;
    (void)(try_narrow<4, 4, 1>(p, false, dtype, stream, e) || try_narrow<2, 4, 1>(p, false, dtype, stream, e) || try_narrow<2, 2, 1>(p, false, dtype, stream, e) ||
           try_narrow<1, 4, 1>(p, false, dtype, stream, e) || try_narrow<1, 2, 2>(p, false, dtype, stream, e) || try_narrow<1, 1, 2>(p, true, dtype, stream, e));
    return e;
}

} // namespace dq
