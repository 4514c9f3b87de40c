// The norms around a block, its gate and the residual: kernels for one type of activations (dq_residual_norm_*.hip have one each).
//
//   z = norm(y; after_weight, after_bias) or y,   r = residual_scale residual + block_scale gate z,   h = norm(r; weight, bias)
//
// A workgroup takes a row (64 to 1024 threads, eight elements of a thread together, from 8192 columns on twice, from 16384 four times), holds it in registers from the loads to the
// stores, and reduces through LDS: every array moves once.  Backward it takes a run of rows and keeps what the weights' and the gate's gradients add up to in registers; what
// workgroups have of the same columns is added in the order of the rows by a second launch.
//
// All arithmetic is in binary32, sums included; h, r and the gradients are rounded once, where they are stored, h from the r that is not rounded yet.
#pragma once

#include "dq_launch.h"
#include "dq_microscale.cuh"

namespace dq {

template <int DT> constexpr int kWords = DT == DQ_F32 ? 8 : 4; // of eight elements

// the sum over 16 lanes, and over a wave, in every lane
__device__ __forceinline__ float row16_sum(float v)
{
    v += dpp_f32<0xB1>(v);  // quad_perm [1,0,3,2]
    v += dpp_f32<0x4E>(v);  // quad_perm [2,3,0,1]
    v += dpp_f32<0x141>(v); // row_half_mirror
    v += dpp_f32<0x140>(v); // row_mirror
    return v;
}
__device__ __forceinline__ float wave_sum_f32(float v)
{
    const int u = __float_as_int(row16_sum(v));
    return (__int_as_float(__builtin_amdgcn_readlane(u, 0)) + __int_as_float(__builtin_amdgcn_readlane(u, 16))) +
           (__int_as_float(__builtin_amdgcn_readlane(u, 32)) + __int_as_float(__builtin_amdgcn_readlane(u, 48)));
}

// the elements that a lane has of a row, and zeros in place of the others
__device__ __forceinline__ int lanes_own(uint32_t col, uint32_t cols) { return (int)min(cols - min(col, cols), 8u); }
__device__ __forceinline__ void clip(float (&v)[8], int own)
{
    if (own < 8) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = j < own ? v[j] : 0.0f;
    }
}

// Sums over a workgroup's threads, in every one of them: a wave's, and then 16 lanes add what up to 16 waves have left.  Two buffers in turn: who writes one for the second time has
// met, in the sum between, everybody who still read it.
struct GroupSums {
    f32x2_t (*part)[16];
    uint32_t waves, first; // of those that share a row
    int turn = 0;
    __device__ __forceinline__ void operator()(float &a, float &b)
    {
        a = wave_sum_f32(a);
        b = wave_sum_f32(b);
        if (waves == 1) return;
        f32x2_t *at = part[turn];
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = f32x2_t{a, b};
        __syncthreads();
        const uint32_t w = threadIdx.x & 15;
        const f32x2_t v = at[first + min(w, waves - 1)];
        a = row16_sum(w < waves ? v.x : 0.0f);
        b = row16_sum(w < waves ? v.y : 0.0f);
    }
    // The mean of a row of cols elements and the sum of the squares of what lies between them and it, where every thread has eight neighbours (0 behind the last one): each wave
    // takes its own mean off first, and waves meet once: sum of squares = sum over the waves of (theirs + their count (their mean - the mean)^2).
    __device__ __forceinline__ void moments(const float (&x)[8], int own, uint32_t cols, float &mean, float &squares)
    {
        const uint32_t wave = (threadIdx.x >> 6) - first;
        const auto count = [&](uint32_t w) { return (float)min(cols - min(cols, 512 * w), 512u); };
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) s += x[j];
        s = wave_sum_f32(s);
        const float mine = s / fmaxf(count(wave), 1.0f);
        float d[8], q = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) d[j] = x[j] - mine;
        clip(d, own);
#pragma unroll
        for (int j = 0; j < 8; j++) q += d[j] * d[j];
        q = wave_sum_f32(q);
        mean = mine;
        squares = q;
        if (waves == 1) return;
        f32x2_t *at = part[turn];
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = f32x2_t{s, q};
        __syncthreads();
        const uint32_t w = threadIdx.x & 15;
        const f32x2_t v = at[first + min(w, waves - 1)];
        const float n = count(w);
        mean = row16_sum(w < waves ? v.x : 0.0f) / (float)cols;
        const float off = v.x / fmaxf(n, 1.0f) - mean;
        squares = row16_sum(w < waves ? v.y + n * (off * off) : 0.0f);
    }
};

// 1 / sqrt(x) to the last place but for one in thousands: a step in 64 bits from an estimate that is good to 2^-22
__device__ __forceinline__ float inverse_root(float x)
{
    const double y = __builtin_amdgcn_rsqf(x), rest = 1.0 - (double)x * y * y;
    return (float)(y + 0.5 * y * rest);
}

// where a row of elements begins, the same for every lane
template <int DT> __device__ __forceinline__ const char *row_of(const void *p, int64_t element) { return static_cast<const char *>(p) + element * (DT == DQ_F32 ? 4 : 2); }
template <int DT> __device__ __forceinline__ char *row_of(void *p, int64_t element) { return static_cast<char *>(p) + element * (DT == DQ_F32 ? 4 : 2); }

// Eight elements of a row as words.  A lane whose eight reach past the end loads the last eight of the row, and moves them up when they are used (settle), with zeros behind the
// last column: no lane loads less or apart (columns are eight at least), and no load is waited for before the next is on its way.
template <int DT, bool PASSING = false> __device__ __forceinline__ void load_row(const char *row, uint32_t col, uint32_t cols, uint32_t (&x)[kWords<DT>])
{
    constexpr int N = kWords<DT>;
    const uint32_t from = min(col, cols - 8);
    const char *q = row + from * (uint32_t)(DT == DQ_F32 ? 4 : 2);
#pragma unroll
    for (int k = 0; k < N; k += 4) {
        const u32x4_any *at = reinterpret_cast<const u32x4_any *>(q + 4 * k);
        const u32x4_any w = PASSING ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
        for (int j = 0; j < 4; j++) x[k + j] = w[j];
    }
}
template <int DT> __device__ __forceinline__ void settle(uint32_t col, uint32_t cols, uint32_t (&x)[kWords<DT>])
{
    constexpr int N = kWords<DT>;
    const uint32_t up = min(col - min(col, cols - 8), 8u);
    if (up) {
        if (N == 4 && up & 1) {
#pragma unroll
            for (int w = 0; w < N; w++) x[w] = w + 1 < N ? __builtin_amdgcn_alignbit(x[(w + 1) % N], x[w], 16) : x[w] >> 16;
        }
#pragma unroll
        for (int k = 1; k <= N; k *= 2)
            if (up & (8 / N) * k) {
#pragma unroll
                for (int w = 0; w < N; w++) x[w] = w + k < N ? x[(w + k) % N] : 0u;
            }
    }
}
template <int DT> __device__ __forceinline__ void row_values(uint32_t (&x)[kWords<DT>], uint32_t col, uint32_t cols, float (&v)[8])
{
    settle<DT>(col, cols, x);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = word_value<DT>(x, j);
}
// eight elements of a weight, a bias or a gate, which are of the activations' type or float32; 0 behind the last column
template <int DT> __device__ __forceinline__ void load_columns(const void *p, bool in32, int64_t base, uint32_t col, uint32_t cols, float (&v)[8])
{
    if (DT == DQ_F32 || in32) {
        uint32_t x[8];
        load_row<DQ_F32>(row_of<DQ_F32>(p, base), col, cols, x);
        row_values<DQ_F32>(x, col, cols, v);
    } else {
        uint32_t x[kWords<DT>];
        load_row<DT>(row_of<DT>(p, base), col, cols, x);
        row_values<DT>(x, col, cols, v);
    }
}
template <int DT, bool PASSING = false> __device__ __forceinline__ void store_row(char *row, uint32_t col, uint32_t cols, const float (&v)[8])
{
    if (col + 8 <= cols)
        store8<DT, PASSING>(row, col, v);
    else if (col < cols)
        store_part<DT, 8>(row, col, (int)(cols - col), v);
}

// eight elements of a row into a checkpoint (four neighbouring lanes together; those past the last column are 0)
template <int DT> __device__ __forceinline__ void keep_row(uint8_t *data, int64_t rows, uint32_t row, uint32_t col, uint32_t cols, const float (&v)[8])
{
    const CheckpointOf<uint8_t> c(data, rows, cols);
    if (col >= 32 * c.blocks) return;
    uint32_t scale;
    const u32x2_t w = encode_e4m3<DT>(v, scale);
    *reinterpret_cast<u32x2_t *>(c.codes + (int64_t)row * 32 * c.blocks + col) = w;
    if ((threadIdx.x & 3) == 0) c.scales[(int64_t)row * c.blocks + (col >> 5)] = (uint8_t)scale;
}

// What the columns are multiplied by, or added to them: words, and when they have all been asked for values (`none` where there is no such vector, 0 behind the last column).
template <int DT> struct Columns {
    uint32_t x[8];
    float v[8];
    __device__ __forceinline__ void ask(const void *p, bool in32, int64_t base, uint32_t col, uint32_t cols)
    {
        if (!p) return;
        if (DT == DQ_F32 || in32) {
            load_row<DQ_F32>(row_of<DQ_F32>(p, base), col, cols, x);
        } else {
            uint32_t y[kWords<DT>];
            load_row<DT>(row_of<DT>(p, base), col, cols, y);
#pragma unroll
            for (int w = 0; w < kWords<DT>; w++) x[w] = y[w];
        }
    }
    __device__ __forceinline__ void take(const void *p, bool in32, uint32_t col, uint32_t cols, float none)
    {
        if (!p) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = none;
            clip(v, lanes_own(col, cols));
        } else if (DT == DQ_F32 || in32) {
            row_values<DQ_F32>(x, col, cols, v);
        } else {
            uint32_t y[kWords<DT>];
#pragma unroll
            for (int w = 0; w < kWords<DT>; w++) y[w] = x[w];
            row_values<DT>(y, col, cols, v);
        }
    }
};

// FULL: there is a norm after the block, or a gate.  Rows up to 8192 wide, without these up to 16384, are taken in turn by as many workgroups as the chip holds, which keep the vectors and ask for a row
// before they work on the one in front of it.  Bound by memory: 8192 x 4096 bf16 with the checkpoints of h and r in 55 us (6.1 TB/s; a workgroup for each row, which loads the weight
// again, 60), with a norm after the block and gates, without checkpoints, 56 (4.8 TB/s; 65); 2048 x 14336 in 48 (4.9 TB/s; with the weight loaded again 94); 1 x 4096 in 2.7, a launch.
// Twice or four times as many workgroups as fit at once take up to 10 % longer.
template <int DT, int RT, int V, int THREADS, bool FULL, bool PASSING> __global__ __launch_bounds__(THREADS, 4) void residual_norm_kernel(BlockNormArgs a)
{
    constexpr bool HELD = V == 1 || (V == 2 && !FULL);
    __shared__ f32x2_t part[2][16];
    const uint32_t threads = a.flags >> 16, cols = a.cols;
    const bool center = a.flags & kNormCenter, after = FULL && a.flags & kNormAfter, before = a.flags & kNormBefore;
    GroupSums sums = {part, threads >> 6, 0};
    // mean and 1 / sqrt(var + eps) of a row, whose elements past the last column are 0
    const auto statistics = [&](const float (&x)[V][8], float &mean, float &rs) {
        float s = 0.0f, none = 0.0f;
        mean = 0.0f;
        if (V == 1 && center) {
            sums.moments(x[0], lanes_own(8 * threadIdx.x, cols), cols, mean, s);
            rs = inverse_root(s / (float)cols + a.eps);
            return;
        }
        if (center) {
#pragma unroll
            for (int k = 0; k < V; k++)
#pragma unroll
                for (int j = 0; j < 8; j++) s += x[k][j];
            sums(s, none);
            mean = s / (float)cols;
            s = none = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < V; k++) {
            float d[8];
#pragma unroll
            for (int j = 0; j < 8; j++) d[j] = x[k][j] - mean;
            clip(d, lanes_own(8 * (threadIdx.x + k * threads), cols));
#pragma unroll
            for (int j = 0; j < 8; j++) s += d[j] * d[j];
        }
        sums(s, none);
        rs = inverse_root(s / (float)cols + a.eps);
    };
    Columns<DT> weight[HELD ? V : 1], bias[HELD ? V : 1], after_weight, after_bias, gate;
    const auto ask_gate = [&](uint32_t row, uint32_t col) { gate.ask(a.gate, a.flags & kNormGate32, (int64_t)(row / a.per) * cols, col, cols); };
    const auto take_gate = [&](uint32_t col) { gate.take(a.gate, a.flags & kNormGate32, col, cols, 1.0f); };
    const auto ask_after = [&](uint32_t col) {
        after_weight.ask(a.after_weight, a.flags & kNormAfterWeight32, 0, col, cols);
        after_bias.ask(a.after_bias, a.flags & kNormAfterBias32, 0, col, cols);
    };
    const auto take_after = [&](uint32_t col) {
        after_weight.take(a.after_weight, a.flags & kNormAfterWeight32, col, cols, 1.0f);
        after_bias.take(a.after_bias, a.flags & kNormAfterBias32, col, cols, 0.0f);
    };
    const auto ask_before = [&](int k, uint32_t col) {
        weight[k].ask(a.weight, a.flags & kNormWeight32, 0, col, cols);
        bias[k].ask(a.bias, a.flags & kNormBias32, 0, col, cols);
    };
    const auto take_before = [&](int k, uint32_t col) {
        weight[k].take(a.weight, a.flags & kNormWeight32, col, cols, 1.0f);
        bias[k].take(a.bias, a.flags & kNormBias32, col, cols, 0.0f);
    };
    struct Raw {
        uint32_t y[V][kWords<DT>], residual[V][kWords<RT>];
    };
    const auto load = [&](Raw &raw, uint32_t row) {
        const int64_t base = (int64_t)row * cols;
#pragma unroll
        for (int k = 0; k < V; k++) load_row<DT, PASSING>(row_of<DT>(a.y, base), 8 * (threadIdx.x + k * threads), cols, raw.y[k]);
        if (a.residual) {
#pragma unroll
            for (int k = 0; k < V; k++) load_row<RT, PASSING>(row_of<RT>(a.residual, base), 8 * (threadIdx.x + k * threads), cols, raw.residual[k]);
        }
    };
    uint32_t gated = blockIdx.x / a.per; // the gate that is held
    const auto step = [&](Raw &now, Raw &next, uint32_t row) {
        const int64_t base = (int64_t)row * cols;
        if (HELD && row + a.grid < a.rows) load(next, row + a.grid);
        if (!HELD) load(now, row);
        float x[V][8], mean_y = 0.0f, rs_y = 1.0f;
#pragma unroll
        for (int k = 0; k < V; k++) row_values<DT>(now.y[k], 8 * (threadIdx.x + k * threads), cols, x[k]);
        if (a.flags & kNormKeepY) {
            uint8_t *data = a.kept + (a.flags & kNormKeepR ? (((int64_t)a.rows * ((cols + 31) >> 5) * 33 + 15) & ~(int64_t)15) : 0);
#pragma unroll
            for (int k = 0; k < V; k++) keep_row<DT>(data, a.rows, row, 8 * (threadIdx.x + k * threads), cols, x[k]);
        }
        if (after) statistics(x, mean_y, rs_y);
        if (FULL && HELD && a.gate && row / a.per != gated) {
            gated = row / a.per;
            ask_gate(row, 8 * threadIdx.x);
            take_gate(8 * threadIdx.x);
        }
#pragma unroll
        for (int k = 0; k < V; k++) {
            const uint32_t col = 8 * (threadIdx.x + k * threads);
            if (after) {
                if (!HELD) {
                    ask_after(col);
                    take_after(col);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] = (x[k][j] - mean_y) * rs_y * after_weight.v[j] + after_bias.v[j];
            }
            if (FULL && a.gate) {
                if (!HELD) {
                    ask_gate(row, col);
                    take_gate(col);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] *= gate.v[j];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) x[k][j] *= a.block_scale;
            if (a.residual) {
                float v[8];
                row_values<RT>(now.residual[k], col, cols, v);
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] = v[j] * a.residual_scale + x[k][j];
            }
            if (a.r) store_row<RT>(row_of<RT>(a.r, base), col, cols, x[k]);
            if (a.flags & kNormKeepR) { // of r as it is stored
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = ElemIO<RT>::round(x[k][j]);
                keep_row<RT>(a.kept, a.rows, row, col, cols, v);
            }
        }
        float mean = 0.0f, rs = 1.0f;
        if (before) {
            statistics(x, mean, rs);
#pragma unroll
            for (int k = 0; k < V; k++) {
                const uint32_t col = 8 * (threadIdx.x + k * threads);
                if (!HELD) {
                    ask_before(0, col);
                    take_before(0, col);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] = ElemIO<DT>::round((x[k][j] - mean) * rs * weight[HELD ? k : 0].v[j] + bias[HELD ? k : 0].v[j]);
                store_row<DT>(row_of<DT>(a.h, base), col, cols, x[k]);
                if (a.h8) keep_row<DT>(a.h8, a.rows, row, col, cols, x[k]);
            }
        }
        if (a.stats && threadIdx.x == 0) reinterpret_cast<float4 *>(a.stats)[row] = make_float4(mean, rs, mean_y, rs_y);
    };
    Raw one, other;
    if (HELD) {
        const uint32_t col = 8 * threadIdx.x;
        load(one, blockIdx.x);
        if (FULL) {
            ask_after(col);
            ask_gate(blockIdx.x, col);
        }
#pragma unroll
        for (int k = 0; k < V; k++) ask_before(k, col + 8 * k * threads);
        if (FULL) {
            take_after(col);
            take_gate(col);
        }
#pragma unroll
        for (int k = 0; k < V; k++) take_before(k, col + 8 * k * threads);
        for (uint32_t row = blockIdx.x; row < a.rows; row += 2 * a.grid) {
            step(one, other, row);
            if (row + a.grid < a.rows) step(other, one, row + a.grid);
        }
    } else {
        for (uint32_t row = blockIdx.x; row < a.rows; row += a.grid) step(one, one, row);
    }
}

// ---- backward ----------------------------------------------------------------------------------------------
//
//   xhat = (r - mean) rs, g = dh weight:   dr = rs (g - [mean g] - xhat mean(g xhat)) + the gradient of r itself
//   dresidual = residual_scale dr, t = block_scale dr, dgate = sum t z, t gate through the norm of y likewise: dy
//   dweight = sum dh xhat, dbias = sum dh, and of the norm of y with t gate in dh's place
//
// Bound by memory where few sums are kept: 8192 x 4096 bf16, weight's gradient, r in 8 bits, 44 us (5.3 TB/s): a row is asked for while the one in front of it is worked on (without
// that 53 at three workgroups a CU, 59 at two), with the hint that nothing of it is wanted again (52 without; what the cache holds is loaded without it, 15.0 us for 17 at 4095 x 768).  With a norm after the
// block and a gate, whose vectors, sums and arrays fill the 128 registers of two workgroups a CU, 76 us (5.3 TB/s; 121 at one workgroup a CU, with more registers each).  A checkpoint's
// codes and the two-byte forms are kernels of their own (EIGHT): one kernel for both waited for each load where the two ways met, 103 us.
//
// SUMS: which of them registers are kept for, at least those that are wanted.  Narrow rows are shared by fewer threads than a workgroup has: those that share one, a team, have a
// run of rows each, and add up what they have of the columns before it leaves.
enum { kSumWeight = 1, kSumBias = 2, kSumGate = 4, kSumAfterWeight = 8, kSumAfterBias = 16 };

template <int DT, int RT, int V, int THREADS, int SUMS, bool EIGHT, bool PASSING> __global__ __launch_bounds__(THREADS, 4) void residual_norm_backward_kernel(BlockNormBackArgs a)
{
    constexpr bool AHEAD = V == 1 && !(SUMS & ~(kSumWeight | kSumBias));
    constexpr bool AFTER = SUMS & (kSumAfterWeight | kSumAfterBias), BETWEEN = SUMS & ~(kSumWeight | kSumBias);
    __shared__ f32x2_t part[2][16];
    const uint32_t threads = a.flags >> 16, cols = a.cols;
    const bool center = a.flags & kNormCenter, after = AFTER && a.flags & kNormAfter;
    const uint32_t team = V == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / threads) : 0, lane = threadIdx.x - team * threads;
    GroupSums sums = {part, threads >> 6, team * (threads >> 6)};
    const float share = 1.0f / (float)cols;
    float acc[5][V][8];
    const auto clear = [&](int s) {
#pragma unroll
        for (int k = 0; k < V; k++)
#pragma unroll
            for (int j = 0; j < 8; j++) acc[s][k][j] = 0.0f;
    };
#pragma unroll
    for (int s = 0; s < 5; s++)
        if (SUMS >> s & 1) clear(s);
    // a team's rows: of one gate, or of whole ones
    const uint32_t id = blockIdx.x * a.teams + team, of = a.parts > 1 ? id / a.parts : 0;
    const uint32_t start = a.parts > 1 ? of * a.per + (id - of * a.parts) * a.run : id * a.run;
    const uint32_t end = min(start + a.run, a.parts > 1 ? (of + 1) * a.per : a.rows);
    uint32_t left = a.per;
    // What the columns are multiplied by, in registers where they hold it all along (1 where there is no weight; 0 behind the last column, where nothing else need be).
    constexpr bool HELD = V == 1 || (V == 2 && !BETWEEN);
    float weight[V][8], after_weight[V][8], gate[V][8];
    const auto load_weight = [&](const void *p, bool in32, int64_t base, uint32_t col, float (&v)[8]) {
        if (p) {
            load_columns<DT>(p, in32, base, col, cols, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = 1.0f;
            clip(v, lanes_own(col, cols));
        }
    };
    if (HELD) {
#pragma unroll
        for (int k = 0; k < V; k++) load_weight(a.weight, a.flags & kNormWeight32, 0, 8 * (lane + k * threads), weight[k]);
        if (AFTER) load_weight(a.after_weight, a.flags & kNormAfterWeight32, 0, 8 * lane, after_weight[0]);
        if (BETWEEN && a.gate) load_columns<DT>(a.gate, a.flags & kNormGate32, (int64_t)(min(start, a.rows - 1) / a.per) * cols, 8 * lane, cols, gate[0]); // (a team may have no rows)
    }
    const auto load_kept = [&](const void *p, auto &x, uint32_t row, uint32_t col, auto type) {
        constexpr int T = decltype(type)::value;
        if (EIGHT) {
            const CheckpointOf<const uint8_t> c(static_cast<const uint8_t *>(p), a.rows, cols);
            const uint32_t from = min(col, 32 * c.blocks - 8);
            const u32x2_t *at = reinterpret_cast<const u32x2_t *>(c.codes + (int64_t)row * 32 * c.blocks + from), w = PASSING ? __builtin_nontemporal_load(at) : *at;
            x[0] = w[0];
            x[1] = w[1];
            x[2] = (c.scales + (int64_t)row * c.blocks)[from >> 5];
        } else {
            load_row<T, PASSING>(row_of<T>(p, (int64_t)row * cols), col, cols, x);
        }
    };
    const auto kept_values = [&](auto &x, uint32_t col, float (&v)[8], auto type) {
        constexpr int T = decltype(type)::value;
        if (EIGHT) {
            const u32x2_t w = {x[0], x[1]};
            decode_e4m3(w, x[2], v);
        } else {
            row_values<T>(x, col, cols, v);
        }
    };
    typedef std::integral_constant<int, DT> Y;
    typedef std::integral_constant<int, RT> R;
    // a row as it comes from memory
    struct Raw {
        uint32_t dh[V][kWords<DT>], dr[V][kWords<RT>], r[V][kWords<RT>], y[V][kWords<DT>];
        float4 stats;
    };
    const auto load = [&](Raw &x, uint32_t row) {
        const int64_t base = (int64_t)row * cols;
#pragma unroll
        for (int k = 0; k < V; k++) {
            const uint32_t col = 8 * (lane + k * threads);
            if (a.dh) {
                load_row<DT, PASSING>(row_of<DT>(a.dh, base), col, cols, x.dh[k]);
                load_kept(a.r, x.r[k], row, col, R());
            }
            if (a.dr) load_row<RT, PASSING>(row_of<RT>(a.dr, base), col, cols, x.dr[k]);
            if (BETWEEN && a.y) load_kept(a.y, x.y[k], row, col, Y());
        }
        x.stats = reinterpret_cast<const float4 *>(a.stats)[row];
    };
    // what becomes of row start + i (as many for every team: they meet), while `next` is on its way
    const auto step = [&](Raw &now, Raw &next, uint32_t i) {
        const uint32_t row = start + i;
        const bool there = row < end;
        const int64_t base = (int64_t)row * cols;
        if (AHEAD) {
            if (row + 1 < end) load(next, row + 1);
        } else if (there) {
            load(now, row);
        }
        if (!there) { // a row of zeros, which adds nothing
#pragma unroll
            for (int k = 0; k < V; k++) {
#pragma unroll
                for (int w = 0; w < kWords<DT>; w++) now.dh[k][w] = now.y[k][w] = 0u;
#pragma unroll
                for (int w = 0; w < kWords<RT>; w++) now.dr[k][w] = now.r[k][w] = 0u;
            }
            now.stats = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        const float4 stats = now.stats;
        float t[V][8];
        if (a.dh) {
            float xhat[V][8], first = 0.0f, second = 0.0f;
#pragma unroll
            for (int k = 0; k < V; k++) {
                kept_values(now.r[k], 8 * (lane + k * threads), xhat[k], R());
                row_values<DT>(now.dh[k], 8 * (lane + k * threads), cols, t[k]);
                if (!HELD) load_weight(a.weight, a.flags & kNormWeight32, 0, 8 * (lane + k * threads), weight[k]);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    xhat[k][j] = (xhat[k][j] - stats.x) * stats.y;
                    if (SUMS & kSumWeight) acc[0][k][j] += t[k][j] * xhat[k][j];
                    if (SUMS & kSumBias) acc[1][k][j] += t[k][j];
                    t[k][j] *= weight[k][j];
                    first += t[k][j];
                    second += t[k][j] * xhat[k][j];
                }
            }
            sums(first, second);
            first = center ? first * share : 0.0f;
            second *= share;
#pragma unroll
            for (int k = 0; k < V; k++)
#pragma unroll
                for (int j = 0; j < 8; j++) t[k][j] = (t[k][j] - first - xhat[k][j] * second) * stats.y;
        } else {
#pragma unroll
            for (int k = 0; k < V; k++)
#pragma unroll
                for (int j = 0; j < 8; j++) t[k][j] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < V; k++) {
            const uint32_t col = 8 * (lane + k * threads);
            float v[8];
            if (a.dr) {
                row_values<RT>(now.dr[k], col, cols, v);
#pragma unroll
                for (int j = 0; j < 8; j++) t[k][j] += v[j];
            }
            if (a.dresidual && there) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = t[k][j] * a.residual_scale;
                store_row<RT>(row_of<RT>(a.dresidual, base), col, cols, v);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) t[k][j] *= a.block_scale;
        }
        if (BETWEEN) {
            float yhat[V][8], first = 0.0f, second = 0.0f;
#pragma unroll
            for (int k = 0; k < V; k++) {
                const uint32_t col = 8 * (lane + k * threads);
                if (a.y) {
                    kept_values(now.y[k], col, yhat[k], Y());
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) yhat[k][j] = 0.0f;
                }
                if (after) {
#pragma unroll
                    for (int j = 0; j < 8; j++) yhat[k][j] = (yhat[k][j] - stats.z) * stats.w;
                    if (!HELD) load_weight(a.after_weight, a.flags & kNormAfterWeight32, 0, col, after_weight[k]);
                }
                if (SUMS & kSumGate) {
#pragma unroll
                    for (int j = 0; j < 8; j++) acc[2][k][j] += t[k][j] * (after ? yhat[k][j] * after_weight[k][j] : yhat[k][j]);
                    if (after && a.after_bias) {
                        float v[8];
                        load_columns<DT>(a.after_bias, a.flags & kNormAfterBias32, 0, col, cols, v);
#pragma unroll
                        for (int j = 0; j < 8; j++) acc[2][k][j] += t[k][j] * v[j];
                    }
                }
                if (a.gate) {
                    if (!HELD) load_columns<DT>(a.gate, a.flags & kNormGate32, (int64_t)(min(row, a.rows - 1) / a.per) * cols, col, cols, gate[k]);
#pragma unroll
                    for (int j = 0; j < 8; j++) t[k][j] *= gate[k][j];
                }
                if (after) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        if (SUMS & kSumAfterWeight) acc[3][k][j] += t[k][j] * yhat[k][j];
                        if (SUMS & kSumAfterBias) acc[4][k][j] += t[k][j];
                        t[k][j] *= after_weight[k][j];
                        first += t[k][j];
                        second += t[k][j] * yhat[k][j];
                    }
                }
            }
            if (after) {
                sums(first, second);
                first = center ? first * share : 0.0f;
                second *= share;
#pragma unroll
                for (int k = 0; k < V; k++)
#pragma unroll
                    for (int j = 0; j < 8; j++) t[k][j] = (t[k][j] - first - yhat[k][j] * second) * stats.w;
            }
        }
        if (a.dy && there) {
#pragma unroll
            for (int k = 0; k < V; k++) store_row<DT>(row_of<DT>(a.dy, base), 8 * (lane + k * threads), cols, t[k]);
        }
        if (SUMS & kSumGate && a.gate && --left == 0) { // the last row of a gate; where all of its rows are this team's, its gradient is whole
            left = a.per;
            if (a.dgate && there) {
                const int64_t to = (int64_t)(row / a.per) * cols;
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const uint32_t col = 8 * (lane + k * threads);
                    if (DT == DQ_F32 || a.flags & kNormGate32)
                        store_row<DQ_F32>(row_of<DQ_F32>(a.dgate, to), col, cols, acc[2][k]);
                    else
                        store_row<DT>(row_of<DT>(a.dgate, to), col, cols, acc[2][k]);
                }
                clear(2);
            }
            if (HELD && row + 1 < end) load_columns<DT>(a.gate, a.flags & kNormGate32, (int64_t)((row + 1) / a.per) * cols, 8 * lane, cols, gate[0]);
        }
    };
    Raw one, other;
    if (AHEAD) {
        if (start < end) load(one, start);
        for (uint32_t i = 0; i < a.run; i += 2) {
            step(one, other, i);
            if (i + 1 < a.run) step(other, one, i + 1);
        }
    } else {
        for (uint32_t i = 0; i < a.run; i++) step(one, one, i);
    }
    uint32_t slot = 0;
#pragma unroll
    for (int s = 0; s < 5; s++) {
        if (!(SUMS >> s & 1) || !(a.sums >> s & 1) || (s == 2 && a.dgate)) continue;
        char *to = row_of<DQ_F32>(a.work, ((int64_t)slot++ * a.grid + blockIdx.x) * cols);
        if constexpr (V == 1 && THREADS == 512) {
            if (a.teams > 1) {
                __shared__ float4 both[2][512];
                __syncthreads();
                both[0][threadIdx.x] = make_float4(acc[s][0][0], acc[s][0][1], acc[s][0][2], acc[s][0][3]);
                both[1][threadIdx.x] = make_float4(acc[s][0][4], acc[s][0][5], acc[s][0][6], acc[s][0][7]);
                __syncthreads();
                if (team == 0) {
                    for (uint32_t m = 1; m < a.teams; m++) {
                        const float4 x = both[0][m * threads + lane], y = both[1][m * threads + lane];
                        acc[s][0][0] += x.x; acc[s][0][1] += x.y; acc[s][0][2] += x.z; acc[s][0][3] += x.w;
                        acc[s][0][4] += y.x; acc[s][0][5] += y.y; acc[s][0][6] += y.z; acc[s][0][7] += y.w;
                    }
                }
            }
        }
        if (team == 0) {
#pragma unroll
            for (int k = 0; k < V; k++) store_row<DQ_F32>(to, 8 * (lane + k * threads), cols, acc[s][k]);
        }
    }
}

// ---- launches for one type of activations --------------------------------------------------------------------

template <int DT, int RT> static hipError_t launch_norm_of(const BlockNormArgs &a, hipStream_t stream)
{
    const uint32_t threads = a.flags >> 16;
    const dim3 grid(a.grid), block(threads);
    const bool full = a.gate || a.flags & kNormAfter, passing = a.flags & kNormPassing;
    if (a.cols > 16384) return launch_with(residual_norm_kernel<DT, RT, 4, 1024, true, false>, grid, block, stream, a);
    if (a.cols > 8192)
        return full ? launch_with(residual_norm_kernel<DT, RT, 2, 1024, true, false>, grid, block, stream, a) : launch_with(residual_norm_kernel<DT, RT, 2, 1024, false, true>, grid, block, stream, a);
    if (threads > 512)
        return full ? passing ? launch_with(residual_norm_kernel<DT, RT, 1, 1024, true, true>, grid, block, stream, a) : launch_with(residual_norm_kernel<DT, RT, 1, 1024, true, false>, grid, block, stream, a)
                    : passing ? launch_with(residual_norm_kernel<DT, RT, 1, 1024, false, true>, grid, block, stream, a) : launch_with(residual_norm_kernel<DT, RT, 1, 1024, false, false>, grid, block, stream, a);
    return full ? passing ? launch_with(residual_norm_kernel<DT, RT, 1, 512, true, true>, grid, block, stream, a) : launch_with(residual_norm_kernel<DT, RT, 1, 512, true, false>, grid, block, stream, a)
                : passing ? launch_with(residual_norm_kernel<DT, RT, 1, 512, false, true>, grid, block, stream, a) : launch_with(residual_norm_kernel<DT, RT, 1, 512, false, false>, grid, block, stream, a);
}

template <int DT, int RT, int V, int THREADS, int SUMS> static hipError_t launch_norm_backward_with(const BlockNormBackArgs &a, hipStream_t stream)
{
    const dim3 grid(a.grid), block((a.flags >> 16) * a.teams);
    if constexpr (V == 1) {
        if (a.flags & kNormPassing)
            return a.flags & kNormEight ? launch_with(residual_norm_backward_kernel<DT, RT, V, THREADS, SUMS, true, true>, grid, block, stream, a)
                                        : launch_with(residual_norm_backward_kernel<DT, RT, V, THREADS, SUMS, false, true>, grid, block, stream, a);
    }
    return a.flags & kNormEight ? launch_with(residual_norm_backward_kernel<DT, RT, V, THREADS, SUMS, true, false>, grid, block, stream, a)
                                : launch_with(residual_norm_backward_kernel<DT, RT, V, THREADS, SUMS, false, false>, grid, block, stream, a);
}
template <int DT, int RT> static hipError_t launch_norm_backward_of(const BlockNormBackArgs &a, hipStream_t stream)
{
    // the block between r and y takes part only in kernels that keep sums of it
    const uint32_t want = a.sums | (a.gate ? kSumGate : 0) | (a.flags & kNormAfter ? kSumAfterWeight : 0);
    const auto within = [&](uint32_t of) { return !(want & ~of); };
    if (a.cols > 16384) return within(3) ? launch_norm_backward_with<DT, RT, 4, 1024, 3>(a, stream) : launch_norm_backward_with<DT, RT, 4, 1024, 31>(a, stream);
    if (a.cols > 8192)
        return within(1) ? launch_norm_backward_with<DT, RT, 2, 1024, 1>(a, stream)
             : within(3) ? launch_norm_backward_with<DT, RT, 2, 1024, 3>(a, stream) : launch_norm_backward_with<DT, RT, 2, 1024, 31>(a, stream);
    if (a.cols > 4096)
        return within(3) ? launch_norm_backward_with<DT, RT, 1, 1024, 3>(a, stream)
             : within(13) ? launch_norm_backward_with<DT, RT, 1, 1024, 13>(a, stream) : launch_norm_backward_with<DT, RT, 1, 1024, 31>(a, stream);
    if (within(1)) return launch_norm_backward_with<DT, RT, 1, 512, 1>(a, stream);
    if (within(3)) return launch_norm_backward_with<DT, RT, 1, 512, 3>(a, stream);
    if (within(7)) return launch_norm_backward_with<DT, RT, 1, 512, 7>(a, stream);
    if (within(13)) return launch_norm_backward_with<DT, RT, 1, 512, 13>(a, stream);
    return launch_norm_backward_with<DT, RT, 1, 512, 31>(a, stream);
}

template <int DT> static hipError_t launch_norm_in(const BlockNormArgs &a, bool stream32, hipStream_t stream)
{
    if (DT == DQ_F32 || stream32) return launch_norm_of<DT, DQ_F32>(a, stream);
    return launch_norm_of<DT, DT>(a, stream);
}
template <int DT> static hipError_t launch_norm_backward_in(const BlockNormBackArgs &a, bool stream32, hipStream_t stream)
{
    if (DT == DQ_F32 || stream32) return launch_norm_backward_of<DT, DQ_F32>(a, stream);
    return launch_norm_backward_of<DT, DT>(a, stream);
}

} // namespace dq
