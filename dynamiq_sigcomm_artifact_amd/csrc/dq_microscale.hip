// 4-bit microscaled matrices: quantised along the rows or the columns, and their values.
//
// Both quantisers give a block of 32 elements to four neighbouring lanes, eight each: its largest magnitude and the last two stages of its
// rotation are two exchanges within the quad, and a lane's eight codes are one word.
#include "dq_launch.h"
#include "dq_microscale.cuh"

namespace dq {

// n / by for n below 2^27: (n mul) >> shift with mul = ceil(2^shift / by) and shift = 27 + ceil(log2 by), whose excess is less than n 2^-shift
struct Division {
    uint32_t by, mul, shift;
    Division() = default;
    explicit Division(uint32_t by_) : by(by_), shift(27)
    {
        while (((uint64_t)1 << (shift - 27)) < by) shift++;
        mul = (uint32_t)((((uint64_t)1 << shift) + by - 1) / by);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (uint32_t)((uint64_t)n * mul >> shift); }
};

enum { kNearest = -1, kPhilox = -2 }; // otherwise the element type of the pool

template <int CTRL> __device__ __forceinline__ float quad_f32(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// H (s x) of the quad's 32 elements, in place (1 / sqrt(32) is encode_block's); word: the sign bits of the block.  Stages of stride 1, 2, 4 lie within a lane, 8 and 16
// between lanes.  Every sum is one of two numbers, whichever lane takes it: the result does not depend on the layout.
__device__ __forceinline__ void rotate_block(float (&v)[8], uint32_t word, int g)
{
#pragma unroll
    for (int j = 0; j < 8; j++) // v ^ (its sign bit, shifted up, & the sign's place)
        v[j] = __uint_as_float(__builtin_amdgcn_bitop3_b32(__float_as_uint(v[j]), (word >> 8 * g) << (31 - j), 0x80000000u, 0x78));
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
        v[j] = g & 2 ? b - v[j] : v[j] + b;
    }
}

// the eight uniform values of elements e .. e + 7 of the result (e a multiple of 8)
template <int RAND> __device__ __forceinline__ void uniform8(const QuantizeArgs &a, int64_t e, float (&u)[8])
{
    if constexpr (RAND >= 0) {
        load8<RAND>(a.pool, e, u);
    } else if constexpr (RAND == kPhilox) {
        uint32_t w[4];
        const RandKey key = {a.key.seed, a.key.step + (a.step_dev ? *a.step_dev : 0)};
        chunk_uniform_words(key, e >> 4, w);
        const uint32_t lo = e & 8 ? w[2] : w[0], hi = e & 8 ? w[3] : w[1];
#pragma unroll
        for (int j = 0; j < 8; j++) u[j] = (float)(((j < 4 ? lo : hi) >> (8 * (j & 3)) & 0xffu) | 1u) * 0.00390625f;
    }
}

// eight codes in a word, the first in the lowest bits, and the block's scale byte (the same in the quad's lanes).  ROTATE: of v / sqrt(32), with one product for an
// element where there would be two.  (Finite sums are below 2^128, so that down is at least 2^-123 and its product with 1 / sqrt(32) a normal number.)
template <int RAND, bool ROTATE, uint32_t LIFT = 0> __device__ __forceinline__ uint32_t encode_block(const float (&v)[8], const float (&u)[8], uint32_t &scale)
{
    constexpr float kUnit = ROTATE ? 0.17677669529663687f : 1.0f;
    uint32_t largest = block_max(v);
    if (ROTATE) largest = __float_as_uint(__uint_as_float(largest) * kUnit);
    scale = RAND == kNearest ? block_scale<2, 0x7fffffu>(largest) : block_scale<2, 0x400000u>(largest);
    const float down = scale_down(scale) * kUnit;
    if (LIFT) scale = min(scale + LIFT, 255u); // (255 where it was, and beyond the largest scale)
    uint32_t word = 0;
    if constexpr (RAND == kNearest) {
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0] * down, v[1] * down, 1.0f, 0);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2] * down, v[3] * down, 1.0f, 1);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4] * down, v[5] * down, 1.0f, 2);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6] * down, v[7] * down, 1.0f, 3);
    } else {
        // With 2^e the power of two at or below max(y, 1), codes are 2^e / 2 apart and t = 2 y / 2^e counts them from 2 e on (below 1: from 0 on).  The exponent's bits
        // carry 127 along, twice: 254 in each place of the word, taken off at the end.
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float y = __builtin_fabsf(v[j]) * down;
            const uint32_t power = __float_as_uint(__builtin_fmaxf(y, 1.0f)) & 0x7f800000u;
            const float t = y * __uint_as_float(0x7f800000u - power);
            const uint32_t code = (uint32_t)t + (power >> 22) + (u[j] < __builtin_amdgcn_fractf(t) ? 1u : 0u);
            word += code << 4 * j;
        }
        // the signs: the highest bytes of four elements in a word
        uint32_t even, odd;
        {
            const auto top = [](float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0703u); };
            even = __builtin_amdgcn_perm(top(v[4], v[6]), top(v[0], v[2]), 0x05040100u);
            odd = __builtin_amdgcn_perm(top(v[5], v[7]), top(v[1], v[3]), 0x05040100u);
        }
        word = (word - 254u * 0x11111111u) | (even >> 4 & 0x08080808u) | (odd & 0x80808080u);
    }
    return word;
}

// Sums of 32 elements from 2^123 on may pass 2^128, and nothing of their block is finite then.  So a rotated block whose scale has become 255 is taken once more, 2^-6 of it, with its
// scale raised by 6: v are its elements as they were.  It is 255 still if it holds an infinity or NaN, or is beyond the largest scale.  (Half precision never gets there.)
template <int RAND> __device__ __forceinline__ uint32_t encode_lowered(float (&v)[8], const float (&u)[8], uint32_t sign, int g, uint32_t &scale)
{
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] *= 0x1p-6f;
    rotate_block(v, sign, g);
    return encode_block<RAND, true, 6>(v, u, scale);
}

// ---- along the rows ----------------------------------------------------------------------------------------

// unit: eight elements of the result, padding included
template <int DT, int RAND, bool ROTATE> __device__ __forceinline__ void quantize_rows(const QuantizeArgs &a, const Division &superchunks, uint32_t unit)
{
    const int g = threadIdx.x & 3;
    const uint32_t row = superchunks(unit >> 5), col = (unit - row * superchunks.by * 32) * 8;
    float v[8], u[8];
    const int64_t at = (int64_t)row * a.stride + col;
    const auto load = [&] {
        if (col + 8 <= (uint32_t)a.cols)
            load8<DT>(a.x, at, v);
        else
            load_part<DT, 8>(a.x, at, row * a.stride + a.cols, v);
    };
    const uint32_t sign = ROTATE ? a.sign[col >> 5] : 0u;
    load();
    uniform8<RAND>(a, (int64_t)unit * 8, u);
    if (ROTATE) rotate_block(v, sign, g);
    const auto put = [&](uint32_t word, uint32_t scale) {
        reinterpret_cast<uint32_t *>(a.codes)[unit] = word;
        if (g == 0) a.scales[unit >> 2] = (uint8_t)scale;
    };
    uint32_t scale;
    const uint32_t word = encode_block<RAND, ROTATE>(v, u, scale);
    put(word, scale);
    if (ROTATE && DT != DQ_F16 && DQ_UNLIKELY(scale == 255u)) { // (in all four lanes of a block)
        load();
        const uint32_t again = encode_lowered<RAND>(v, u, sign, g, scale);
        put(again, scale);
    }
}

// Bound by memory: 14336 x 4096 bf16 to the nearest in 27 us (5.5 TB/s), rotated and stochastic with a bf16 pool 4096 x 14336 in 47 to 56 (up to 5.7 TB/s).  With the random stream
// made in the kernel it is the arithmetic of the stream: 40 us for the latter's 149 MB, rotated 46 (30 at a copy's rate); along the columns, rotated, 50.  A lane takes half of the
// sixteen numbers that a call of the stream gives.
template <int DT, int RAND, bool ROTATE> __global__ __launch_bounds__(256) void mx4_rows_kernel(QuantizeArgs a, Division superchunks, uint32_t units)
{
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    if (unit < units) quantize_rows<DT, RAND, ROTATE>(a, superchunks, unit);
}

// ---- along the columns -------------------------------------------------------------------------------------

// A workgroup takes 256 rows x 128 columns: one superchunk of 128 rows of the result.  A wave takes 32 of the rows, a lane 8 rows x 8 columns, and a
// column's block lies in a quad as it does above.  The codes leave through LDS, as whole lines.  Elements of 16 bits stay packed until their column's turn: three
// workgroups on a CU instead of two (14336 x 4096 bf16, rotated, to the nearest in 28 us, 5.3 TB/s; unpacked 33).  8192 x 14336 with a bf16 pool takes 116 us behind its like
// (4.6 TB/s), 132 behind other work (with the XCDs' workgroups strewn 8 % more, 8000 x 5000 40 for 35), where the pool's runs of 64 bytes keep it from more: neither all of the pool asked for at once nor fewer
// instructions change it.  Half as wide a tile, with runs of 128 bytes of x, takes half as long again to the nearest.  Blocks that have to be lowered are looked for while their columns
// are encoded and taken behind the loop, where nothing else needs registers (in it: 2 to 6 % for every matrix); to the nearest four workgroups share a CU, which 65 registers would not let them.
struct ColumnsLds {
    __attribute__((aligned(16))) uint8_t tile[128 * 128];
    __attribute__((aligned(8))) uint8_t scales[128 * 8];
};
template <int DT, int RAND, bool ROTATE>
__device__ __forceinline__ void quantize_columns(const QuantizeArgs &a, uint32_t superchunks, const Division &tiles, uint32_t id, ColumnsLds &lds)
{
    uint8_t *tile = lds.tile, *tile_scales = lds.scales;
    const int lane = threadIdx.x & 63, block = threadIdx.x >> 6, g = lane & 3;
    const uint32_t superchunk = tiles(id), col0 = (id - superchunk * tiles.by) * 128, col = col0 + 8 * (lane >> 2), all_cols = (uint32_t)a.cols, last_row = (uint32_t)a.rows - 1;
    const uint32_t row0 = superchunk * 256 + 32 * block, row = row0 + 8 * g;
    constexpr int WORDS = DT == DQ_F32 ? 8 : 4;
    uint32_t x[8][WORDS]; // [row][column], as they are in memory
    if (all_cols >= 8) {
        // a lane whose eight columns reach past the end loads the last eight, and moves them up
        const uint32_t from = min(col, all_cols - 8), up = col - from;
#pragma unroll
        for (int j = 0; j < 8; j++) load_words<DT>(a.x, (int64_t)min(row + j, last_row) * a.stride + from, x[j]);
        if (up) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (WORDS == 4 && up & 1)
#pragma unroll
                    for (int w = 0; w < WORDS; w++) x[j][w] = __builtin_amdgcn_alignbit(x[j][min(w + 1, WORDS - 1)], x[j][w], 16);
#pragma unroll
                for (int k = 1; k < WORDS; k *= 2)
                    if (up & (8 / WORDS) * k)
#pragma unroll
                        for (int w = 0; w + k < WORDS; w++) x[j][w] = x[j][w + k];
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) load_words_part<DT>(a.x, (int64_t)min(row + j, last_row) * a.stride, col, all_cols, x[j]);
    }
    if (row + 8 > last_row + 1) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (row + j > last_row) {
#pragma unroll
                for (int w = 0; w < WORDS; w++) x[j][w] = 0u;
            }
    }
    const uint32_t sign = ROTATE ? a.sign[row0 >> 5] : 0u, first = col * superchunks + superchunk, most = (all_cols - 1) * superchunks + superchunk;
    // (what becomes of columns past the end is not stored)
    const auto draw = [&](int c, float (&u)[8]) { uniform8<RAND>(a, (int64_t)min(first + c * superchunks, most) * 256 + 32 * block + 8 * g, u); };
    const auto put = [&](int c, uint32_t word, uint32_t scale) {
        const int line = 8 * (lane >> 2) + c;
        *reinterpret_cast<uint32_t *>(tile + line * 128 + ((block ^ (line >> 3 & 7)) << 4) + 4 * g) = word;
        if (g == 0) tile_scales[line * 8 + block] = (uint8_t)scale;
    };
    bool beyond = false;
#pragma unroll
    for (int c = 0; c < 8; c++) {
        float v[8], u[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = word_value<DT>(x[j], c);
        draw(c, u);
        if (ROTATE) rotate_block(v, sign, g);
        uint32_t scale;
        const uint32_t word = encode_block<RAND, ROTATE>(v, u, scale);
        put(c, word, scale);
        beyond |= scale == 255u;
    }
    if (ROTATE && DT != DQ_F16 && DQ_UNLIKELY(__builtin_amdgcn_ballot_w64(beyond) != 0)) {
#pragma unroll 1
        for (int c = 0; c < 8; c++) { // what nobody holds any more, element by element
            float v[8], u[8];
            uint32_t scale;
            const auto load = [&] {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    v[j] = ElemIO<DT>::load(a.x, (int64_t)min(row + j, last_row) * a.stride + min(col + c, all_cols - 1));
                    if (row + j > last_row) v[j] = 0.0f;
                }
            };
            load();
            draw(c, u);
            rotate_block(v, sign, g);
            (void)encode_block<RAND, true>(v, u, scale);
            if (scale == 255u) {
                load();
                const uint32_t word = encode_lowered<RAND>(v, u, sign, g, scale);
                put(c, word, scale);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int s = threadIdx.x + 512 * k, line = s >> 3, piece = s & 7;
        if (col0 + line < all_cols)
            reinterpret_cast<uint4 *>(a.codes)[((int64_t)(col0 + line) * superchunks + superchunk) * 8 + piece] =
                *reinterpret_cast<const uint4 *>(tile + line * 128 + ((piece ^ (line >> 3 & 7)) << 4));
    }
    if (threadIdx.x < 128 && col0 + threadIdx.x < all_cols)
        reinterpret_cast<uint2 *>(a.scales)[(int64_t)(col0 + threadIdx.x) * superchunks + superchunk] = reinterpret_cast<const uint2 *>(tile_scales)[threadIdx.x];
}

template <int DT, int RAND, bool ROTATE>
__global__ __launch_bounds__(512, DT == DQ_F32 ? 4 : RAND == kNearest && ROTATE ? 8 : 6) void mx4_columns_kernel(QuantizeArgs a, uint32_t superchunks, Division tiles)
{
    __shared__ ColumnsLds lds;
    quantize_columns<DT, RAND, ROTATE>(a, superchunks, tiles, unit_of(blockIdx.x, gridDim.x), lds);
}

template <int DT, int RAND> static hipError_t launch_quantize(const QuantizeArgs &a, bool columns, hipStream_t stream)
{
    const uint32_t superchunks = (uint32_t)(((columns ? a.rows : a.cols) + 255) >> 8);
    if (columns) {
        const Division tiles((uint32_t)((a.cols + 127) >> 7));
        const dim3 grid(tiles.by * superchunks);
        if (a.sign)
            mx4_columns_kernel<DT, RAND, true><<<grid, 512, 0, stream>>>(a, superchunks, tiles);
        else
            mx4_columns_kernel<DT, RAND, false><<<grid, 512, 0, stream>>>(a, superchunks, tiles);
    } else {
        const uint32_t units = (uint32_t)(a.rows * superchunks * 32);
        const dim3 grid((units + 255) / 256);
        if (a.sign)
            mx4_rows_kernel<DT, RAND, true><<<grid, 256, 0, stream>>>(a, Division(superchunks), units);
        else
            mx4_rows_kernel<DT, RAND, false><<<grid, 256, 0, stream>>>(a, Division(superchunks), units);
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

// ---- several small matrices at once -------------------------------------------------------------------------

// Up to four matrices of one element type, along either axis and rounded in any way: a workgroup takes 4096 elements along the rows or a tile along the columns.  A small
// one leaves most CUs without work and costs a launch all the same: a linear layer's step of 333 x 776 x 1000, in a graph, takes 28 us with two such launches where six
// quantisers of their own made it 44, of 2048 x 2048 x 2048 56 for 66, of 4096 x 4096 x 4096 171 for 177.  What shares a launch has 4096 workgroups at most: 4096 x 14336 x 4096,
// whose last three matrices have just those, takes 534 us for 542 alone, 6000 x 6000 x 6000 500 for 512.  Without that limit, with the largest ones in kernels that hold
// less than they could, they are back at 541 and 513, and 8192 x 14336 x 4096 takes 980 us for 973.
struct QuantizeJob {
    QuantizeArgs a;
    Division by; // superchunks of a row, or tiles of 128 columns
    uint32_t superchunks, units, first; // first: of its workgroups
    int32_t kind;
};
constexpr int kJobs = 4, kJobBlocks = 4096;
struct QuantizeJobs {
    QuantizeJob job[kJobs];
};

template <int DT, int RAND, bool ROTATE> __device__ __forceinline__ void do_job(const QuantizeJob &j, bool columns, uint32_t id, ColumnsLds &lds)
{
    if (columns)
        quantize_columns<DT, RAND, ROTATE>(j.a, j.superchunks, j.by, id, lds);
    else if (id * 512 + threadIdx.x < j.units)
        quantize_rows<DT, RAND, ROTATE>(j.a, j.by, id * 512 + threadIdx.x);
}

template <int DT> __global__ __launch_bounds__(512, DT == DQ_F32 ? 4 : 6) void mx4_jobs_kernel(QuantizeJobs jobs)
{
    __shared__ ColumnsLds lds;
    int k = 0;
#pragma unroll
    for (int i = 1; i < kJobs; i++) k += blockIdx.x >= jobs.job[i].first ? 1 : 0;
    const QuantizeJob j = jobs.job[k];
    const uint32_t id = blockIdx.x - j.first;
    const bool columns = j.kind & 16;
    switch (j.kind & 15) {
    case 0: return do_job<DT, kNearest, false>(j, columns, id, lds);
    case 1: return do_job<DT, kNearest, true>(j, columns, id, lds);
    case 2: return do_job<DT, kPhilox, false>(j, columns, id, lds);
    case 3: return do_job<DT, kPhilox, true>(j, columns, id, lds);
    case 4: return do_job<DT, DQ_F16, false>(j, columns, id, lds);
    case 5: return do_job<DT, DQ_F16, true>(j, columns, id, lds);
    case 6: return do_job<DT, DQ_BF16, false>(j, columns, id, lds);
    case 7: return do_job<DT, DQ_BF16, true>(j, columns, id, lds);
    case 8: return do_job<DT, DQ_F32, false>(j, columns, id, lds);
    default: return do_job<DT, DQ_F32, true>(j, columns, id, lds);
    }
}

hipError_t launch_mx4_quantize_list(const QuantizeOne *list, int count, hipStream_t stream)
{
    const auto blocks_of = [](const QuantizeOne &q) {
        return q.columns ? ((q.a.cols + 127) >> 7) * ((q.a.rows + 255) >> 8) : (q.a.rows * ((q.a.cols + 255) >> 8) + 15) >> 4;
    };
    for (int next = 0; next < count;) {
        int take = 0;
        int64_t blocks = 0;
        while (take < kJobs && next + take < count && list[next + take].dtype == list[next].dtype && blocks + blocks_of(list[next + take]) <= kJobBlocks)
            blocks += blocks_of(list[next + take++]);
        hipError_t e;
        if (take < 2) {
            const QuantizeOne &q = list[next++];
            e = launch_mx4_quantize(q.a, q.dtype, q.columns, q.stochastic, q.pool_dtype, stream);
        } else {
            QuantizeJobs jobs = {};
            uint32_t first = 0;
            for (int k = 0; k < kJobs; k++) {
                QuantizeJob &j = jobs.job[k];
                j.first = k < take ? first : 0xffffffffu;
                j.by = Division(1);
                if (k >= take) continue;
                const QuantizeOne &q = list[next + k];
                j.a = q.a;
                j.superchunks = (uint32_t)(((q.columns ? q.a.rows : q.a.cols) + 255) >> 8);
                j.by = Division(q.columns ? (uint32_t)((q.a.cols + 127) >> 7) : j.superchunks);
                j.units = (uint32_t)(q.a.rows * j.superchunks * 32);
                j.kind = (q.columns ? 16 : 0) + (!q.stochastic ? 0 : !q.a.pool ? 2 : 4 + 2 * q.pool_dtype) + (q.a.sign ? 1 : 0);
                first += (uint32_t)blocks_of(q);
            }
            const dim3 grid((uint32_t)blocks), block(512);
            e = list[next].dtype == DQ_F32 ? launch_with(mx4_jobs_kernel<DQ_F32>, grid, block, stream, jobs)
              : list[next].dtype == DQ_BF16 ? launch_with(mx4_jobs_kernel<DQ_BF16>, grid, block, stream, jobs)
                                            : launch_with(mx4_jobs_kernel<DQ_F16>, grid, block, stream, jobs);
            next += take;
        }
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// ---- and back ----------------------------------------------------------------------------------------------

// bound by memory: 117 million elements to bf16 in 60 us, 5.0 TB/s
template <int DT>
__global__ __launch_bounds__(256) void mx4_values_kernel(const uint32_t *__restrict__ codes, const uint8_t *__restrict__ scales, void *__restrict__ out, uint32_t cols,
                                                        Division superchunks, uint32_t units)
{
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    if (unit >= units) return;
    const uint32_t row = superchunks(unit >> 5), col = (unit - row * superchunks.by * 32) * 8;
    if (col >= cols) return;
    const uint32_t word = codes[unit];
    const float up = scale_up(scales[unit >> 2]);
    float v[8];
    const f32x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 1);
    const f32x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 3);
    v[0] = p0.x * up; v[1] = p0.y * up; v[2] = p1.x * up; v[3] = p1.y * up;
    v[4] = p2.x * up; v[5] = p2.y * up; v[6] = p3.x * up; v[7] = p3.y * up;
    const int64_t at = (int64_t)row * cols + col;
    if (col + 8 <= cols)
        store8<DT>(out, at, v);
    else
        store_part<DT, 8>(out, at, (int)(cols - col), v);
}

hipError_t launch_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, void *out, int64_t rows, int64_t cols, int dtype, hipStream_t stream)
{
    const Division superchunks((uint32_t)((cols + 255) >> 8));
    const uint32_t units = (uint32_t)(rows * superchunks.by * 32);
    const dim3 grid((units + 255) / 256);
    const uint32_t *words = reinterpret_cast<const uint32_t *>(codes);
    if (dtype == DQ_F32)
        mx4_values_kernel<DQ_F32><<<grid, 256, 0, stream>>>(words, scales, out, (uint32_t)cols, superchunks, units);
    else if (dtype == DQ_BF16)
        mx4_values_kernel<DQ_BF16><<<grid, 256, 0, stream>>>(words, scales, out, (uint32_t)cols, superchunks, units);
    else
        mx4_values_kernel<DQ_F16><<<grid, 256, 0, stream>>>(words, scales, out, (uint32_t)cols, superchunks, units);
    return hipGetLastError();
}

} // namespace dq
