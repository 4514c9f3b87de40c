// The norms around a block: launches, and the sums over rows that end a backward pass.
#include "dq_launch.h"
#include "dq_microscale.cuh"

namespace dq {

// Threads of a row that lies in registers: eight elements each as far as 1024 of them go, then twice eight.
static uint32_t norm_threads(uint32_t cols)
{
    const uint32_t vectors = (cols + 7) >> 3;
    const uint32_t each = vectors <= 1024 ? 1 : 2;
    return std::min(((vectors + each - 1) / each + 63) & ~63u, 1024u);
}

// Rows of which a thread would have more than its registers hold: in LDS forward, and read twice backward.  2048 x 14336 bf16 with both norms and a gate, forward 63 us and backward 139
// (registers that spill 90 and 344), 1000 x 32768 with one norm 50 and 80 (118 and 281); 4096 x 8192 with both norms and a gate would take 150 backward in place of 96.
// With a residual alone registers are the better place as far as they go, though they spill 52 to 140 values of fp32, and of a 32-bit stream with a bias: both passes over 2048 x 14336 bf16
// 100 us (113 read twice), with a 32-bit stream 177 (187), fp32 228 (247), 4096 x 8200 with a 32-bit stream and a bias 241 (260); that form alone is slower in the widest, 208 for 193.
static bool norm_wide(uint32_t cols, bool between) { return cols > 16384 || (between && cols > 8192); }

// Whether a pass' arrays, four or so, are more than half of the 256 MB cache: then its loads carry the hint that nothing of them is wanted again soon.
static bool norm_passing(int64_t rows, uint32_t cols, int dtype) { return rows * cols * 4 * (dtype == DQ_F32 ? 4 : 2) > (int64_t)128 << 20; }

hipError_t launch_norm(BlockNormArgs a, int dtype, bool stream32, hipStream_t stream)
{
    a.flags |= norm_threads(a.cols) << 16;
    if (norm_passing(a.rows, a.cols, dtype)) a.flags |= kNormPassing;
    // workgroups that the chip holds at once, sixteen waves a CU, with as many rows each
    const bool halves = a.cols <= 16384 && norm_wide(a.cols, a.gate || a.flags & kNormAfter); // half a CU's LDS each
    const uint32_t held = 256 * (halves ? 2 : 1024 / norm_threads(a.cols)), turns = (a.rows + held - 1) / held;
    a.grid = (a.rows + turns - 1) / turns;
    return dtype == DQ_F32 ? launch_norm_f32(a, stream32, stream) : dtype == DQ_BF16 ? launch_norm_bf16(a, stream32, stream) : launch_norm_f16(a, stream32, stream);
}

// How a backward pass shares its rows out.  As many workgroups as the chip holds at once, two a CU, or one of a thousand threads (1024 x 8192 in 20 us, with two in turn 26); more
// would leave more sums to add up, fewer take longer than what that saves (with at least 4, 8 or 16 rows each 1024 x 4096 takes 1 % less, 7 and 60 % more).  Teams of as many threads as
// a row takes, or the 64 of a tile of a wide one, up to 512 together in a workgroup, have runs of `run` rows -- `parts` of them (the last ones shorter) to the rows of a gate, all of a
// workgroup's of the same one, or one of whole gates (then up to twice as many workgroups).  A gate that would be two runs or less is one: shared out among all of a workgroup's teams it
// would take a workgroup, most of whose teams had nothing to do (both passes over 8190 x 512 with 3 rows a gate 31 us, 83 shared out, with 2 rows 28; 12288 x 256 with 4 rows 30 and 66;
// 4096 x 14336 with 32 rows 397 and 454; nothing measured is slower).  At three runs 8190 x 512 with 5 rows would gain as well (59 to 31), but 30000 x 64 with 24 lose (52 to 65).
NormShares norm_shares(int64_t rows, int64_t per, uint32_t cols, bool between)
{
    NormShares s;
    s.wide = norm_wide(cols, between);
    const uint32_t threads = s.wide ? 64 : norm_threads(cols), tiles = s.wide ? (cols + 511) / 512 : 1;
    s.teams = std::max(1u, 512 / threads);
    const int64_t runs = std::max(1u, (threads > 512 ? 256 : 512) / tiles) * (int64_t)s.teams;
    int64_t run = (rows + runs - 1) / runs;
    if (per == 0 || per <= run || (s.teams > 2 && per <= 2 * run)) {
        if (per) run = std::max(run / per, (int64_t)1) * per;
        s.parts = 1;
        s.grid = (uint32_t)((rows + run * s.teams - 1) / (run * s.teams));
    } else {
        s.parts = (uint32_t)((per + run - 1) / run);
        s.parts = (s.parts + s.teams - 1) / s.teams * s.teams;
        run = (per + s.parts - 1) / s.parts;
        s.grid = (uint32_t)(rows / per * (s.parts / s.teams));
    }
    s.run = (uint32_t)run;
    return s;
}

struct ColumnSums {
    const float *work;
    uint32_t grid, cols, count, tiles;
    struct One {
        void *out;
        uint32_t segments, parts, dtype;
    } one[5];
};

// out[s][c]: the sum of `parts` rows of work, which lie one behind the other.  Sixteen threads share a column's rows, in an order that does not change: 512 rows of 4096 in 4 us (with four
// threads 7).
__global__ __launch_bounds__(1024) void column_sums_kernel(ColumnSums a)
{
    __shared__ float part[16][64];
    uint32_t id = blockIdx.x / a.tiles, k = 0;
    const uint32_t col = (blockIdx.x - id * a.tiles) * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6, at = min(col, a.cols - 1);
    while (id >= a.one[k].segments) id -= a.one[k++].segments;
    const ColumnSums::One o = a.one[k];
    const float *from = a.work + ((int64_t)k * a.grid + (int64_t)id * o.parts) * a.cols + at;
    float sum = 0.0f;
    uint32_t p = slice;
    for (; p + 112 < o.parts; p += 128) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = from[(int64_t)(p + 16 * j) * a.cols];
        sum += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    for (; p < o.parts; p += 16) sum += from[(int64_t)p * a.cols];
    part[slice][threadIdx.x & 63] = sum;
    __syncthreads();
    if (slice || col >= a.cols) return;
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; j += 4) sum += (part[j][threadIdx.x] + part[j + 1][threadIdx.x]) + (part[j + 2][threadIdx.x] + part[j + 3][threadIdx.x]);
    const int64_t to = (int64_t)id * a.cols + col;
    if (o.dtype == DQ_F32)
        ElemIO<DQ_F32>::store(o.out, to, sum);
    else if (o.dtype == DQ_BF16)
        ElemIO<DQ_BF16>::store(o.out, to, sum);
    else
        ElemIO<DQ_F16>::store(o.out, to, sum);
}

hipError_t launch_norm_backward(BlockNormBackArgs a, const NormSum (&sums)[5], int dtype, bool stream32, hipStream_t stream)
{
    const NormShares s = norm_shares(a.rows, a.gate ? a.per : 0, a.cols, a.gate || a.flags & kNormAfter);
    a.flags |= (s.wide ? 64 : norm_threads(a.cols)) << 16;
    a.means = s.wide ? a.work : nullptr;
    a.work += s.wide ? 4 * (int64_t)a.rows : 0;
    if (norm_passing(a.rows, a.cols, dtype)) a.flags |= kNormPassing;
    a.grid = s.grid;
    a.teams = s.teams;
    a.run = s.run;
    a.parts = s.parts;
    a.sums = 0;
    a.dgate = nullptr;
    ColumnSums c = {a.work, s.grid, a.cols, 0, (a.cols + 63) / 64, {}};
    uint32_t segments = 0;
    for (int k = 0; k < 5; k++) {
        if (!sums[k].out) continue;
        a.sums |= 1u << k;
        if (k == 2 && s.parts == 1) { // a gate's rows lie within one workgroup
            a.dgate = sums[k].out;
            continue;
        }
        c.one[c.count++] = {sums[k].out, k == 2 ? a.rows / a.per : 1, k == 2 ? s.parts / s.teams : s.grid, (uint32_t)sums[k].dtype};
        segments += c.one[c.count - 1].segments;
    }
    const hipError_t e = dtype == DQ_F32 ? launch_norm_backward_f32(a, stream32, stream)
                       : dtype == DQ_BF16 ? launch_norm_backward_bf16(a, stream32, stream) : launch_norm_backward_f16(a, stream32, stream);
    if (e != hipSuccess || !segments) return e;
    return launch_with(column_sums_kernel, dim3(segments * c.tiles), dim3(1024), stream, c);
}

} // namespace dq
