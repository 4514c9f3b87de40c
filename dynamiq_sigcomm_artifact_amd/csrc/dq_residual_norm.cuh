// The norms around a block, its gate and the residual: kernels for one type of activations (dq_residual_norm_*.hip have one each).
//
//   z = norm(y; after_weight, after_bias) or y,   r = residual_scale residual + block_scale gate z,   h = norm(r; weight, bias)
//
// A workgroup takes a row (64 to 1024 threads, eight elements of a thread together, from 8192 columns on twice), holds it in registers from the loads to the stores, and reduces
// through LDS: every array moves once.  Backward it takes a run of rows and keeps what the weights' and the gate's gradients add up to in registers; what workgroups have of the same
// columns is added in the order of the rows by a second launch.  Rows beyond 16384, or beyond 8192 with more than a residual between y and r, have kernels of their own.
//
// Column numbers are made afresh from the thread's where a loop over rows would spill (an empty asm): what follows from them alone, addresses and the shifts of a row's end, is else
// kept from row to row for every array.  2048 x 14336 bf16 with a binary32 residual 73 us forward, 196 with it kept; all five sums of 4096 x 4096 77 backward, and 99; where
// registers are left, keeping it is 2 % faster.
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

// FULL: there is a norm after the block, or a gate.  Rows are taken in turn by as many workgroups as the chip holds, which keep the vectors and ask for a row before they work on the
// one in front of it.  Bound by memory: 8192 x 4096 bf16 with the checkpoints of h and r in 55 us (6.1 TB/s; a workgroup for each row, which loads the weight again, 60), with a norm
// after the block and gates, without checkpoints, 56 (4.8 TB/s; 65); 2048 x 14336 in 46 (5.1 TB/s; in LDS 55); 1 x 4096 in 2.7, a launch.  Twice or four times as many workgroups as
// fit at once take up to 10 % longer.
template <int DT, int RT, int V, int THREADS, bool FULL, bool PASSING> __global__ __launch_bounds__(THREADS, 4) void residual_norm_kernel(BlockNormArgs a)
{
    static_assert(V == 1 || !FULL, "the vectors between r and y are held of eight columns");
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
    Columns<DT> weight[V], bias[V], after_weight, after_bias, gate;
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
    const auto col_of = [&](int k) {
        uint32_t thread = threadIdx.x;
        if (V > 1) asm volatile("" : "+v"(thread));
        return 8 * (thread + k * threads);
    };
    const auto load = [&](Raw &raw, uint32_t row) {
        const int64_t base = (int64_t)row * cols;
#pragma unroll
        for (int k = 0; k < V; k++) load_row<DT, PASSING>(row_of<DT>(a.y, base), col_of(k), cols, raw.y[k]);
        if (a.residual) {
#pragma unroll
            for (int k = 0; k < V; k++) load_row<RT, PASSING>(row_of<RT>(a.residual, base), col_of(k), cols, raw.residual[k]);
        }
    };
    uint32_t gated = blockIdx.x / a.per; // the gate that is held
    const auto step = [&](Raw &now, Raw &next, uint32_t row) {
        const int64_t base = (int64_t)row * cols;
        if (row + a.grid < a.rows) load(next, row + a.grid);
        float x[V][8], mean_y = 0.0f, rs_y = 1.0f;
#pragma unroll
        for (int k = 0; k < V; k++) row_values<DT>(now.y[k], col_of(k), cols, x[k]);
        if (a.flags & kNormKeepY) {
            uint8_t *data = a.kept + (a.flags & kNormKeepR ? (((int64_t)a.rows * ((cols + 31) >> 5) * 33 + 15) & ~(int64_t)15) : 0);
#pragma unroll
            for (int k = 0; k < V; k++) keep_row<DT>(data, a.rows, row, col_of(k), cols, x[k]);
        }
        if (after) statistics(x, mean_y, rs_y);
        if (FULL && a.gate && row / a.per != gated) {
            gated = row / a.per;
            ask_gate(row, 8 * threadIdx.x);
            take_gate(8 * threadIdx.x);
        }
#pragma unroll
        for (int k = 0; k < V; k++) {
            const uint32_t col = col_of(k);
            if (after) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] = (x[k][j] - mean_y) * rs_y * after_weight.v[j] + after_bias.v[j];
            }
            if (FULL && a.gate) {
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
                const uint32_t col = col_of(k);
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] = ElemIO<DT>::round((x[k][j] - mean) * rs * weight[k].v[j] + bias[k].v[j]);
                store_row<DT>(row_of<DT>(a.h, base), col, cols, x[k]);
                if (a.h8) keep_row<DT>(a.h8, a.rows, row, col, cols, x[k]);
            }
        }
        if (a.stats && threadIdx.x == 0) reinterpret_cast<float4 *>(a.stats)[row] = make_float4(mean, rs, mean_y, rs_y);
    };
    Raw one, other;
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
}

// Wider rows lie in LDS, each thread's own columns of them, from the loads of y to the stores of h; two workgroups a CU, or one beyond 16384.  Bound by vector instructions and LDS beside
// memory: 2048 x 14336 bf16 with both norms and a gate 63 us (3.7 TB/s), 1000 x 32768 with one norm 50 (5.2 TB/s).
template <int DT, int RT, int THREADS> __global__ __launch_bounds__(THREADS, 4) void residual_norm_wide_kernel(BlockNormArgs a)
{
    constexpr int V = 4;
    __shared__ f32x2_t part[2][16];
    __shared__ float4 held[2 * V][THREADS];
    const uint32_t cols = a.cols;
    const bool center = a.flags & kNormCenter, after = a.flags & kNormAfter, before = a.flags & kNormBefore;
    GroupSums sums = {part, THREADS / 64, 0};
    const auto col_of = [](int k) { // afresh
        uint32_t thread = threadIdx.x;
        asm volatile("" : "+v"(thread));
        return 8 * (thread + k * THREADS);
    };
    const auto hold = [&](int k, const float (&v)[8]) {
        held[2 * k][threadIdx.x] = make_float4(v[0], v[1], v[2], v[3]);
        held[2 * k + 1][threadIdx.x] = make_float4(v[4], v[5], v[6], v[7]);
    };
    const auto look = [&](int k, float (&v)[8]) {
        const float4 x = held[2 * k][threadIdx.x], y = held[2 * k + 1][threadIdx.x];
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
    };
    // mean and 1 / sqrt(var + eps) of what is held, from the sum of it, or of its squares
    const auto statistics = [&](float s, float &mean, float &rs) {
        float none = 0.0f;
        sums(s, none);
        mean = 0.0f;
        if (center) {
            mean = s / (float)cols;
            s = none = 0.0f;
#pragma unroll
            for (int k = 0; k < V; k++) {
                if (8 * k * THREADS >= cols) break;
                float v[8];
                look(k, v);
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] -= mean;
                clip(v, lanes_own(col_of(k), cols));
#pragma unroll
                for (int j = 0; j < 8; j++) s += v[j] * v[j];
            }
            sums(s, none);
        }
        rs = inverse_root(s / (float)cols + a.eps);
    };
    const auto add_up = [&](const float (&v)[8], float &s) {
#pragma unroll
        for (int j = 0; j < 8; j++) s += center ? v[j] : v[j] * v[j];
    };
    for (uint32_t row = blockIdx.x; row < a.rows; row += a.grid) {
        const int64_t base = (int64_t)row * cols;
        uint32_t y[V][kWords<DT>], residual[V][kWords<RT>];
#pragma unroll
        for (int k = 0; k < V; k++) load_row<DT, true>(row_of<DT>(a.y, base), col_of(k), cols, y[k]);
        if (a.residual) {
#pragma unroll
            for (int k = 0; k < V; k++) load_row<RT, true>(row_of<RT>(a.residual, base), col_of(k), cols, residual[k]);
        }
        float mean_y = 0.0f, rs_y = 1.0f, mean = 0.0f, rs = 1.0f, s = 0.0f;
        uint8_t *data = a.kept + (a.flags & kNormKeepR ? (((int64_t)a.rows * ((cols + 31) >> 5) * 33 + 15) & ~(int64_t)15) : 0);
#pragma unroll
        for (int k = 0; k < V; k++) {
            if (8 * k * THREADS >= cols) break;
            float v[8];
            const uint32_t col = col_of(k);
            row_values<DT>(y[k], col, cols, v);
            if (a.flags & kNormKeepY) keep_row<DT>(data, a.rows, row, col, cols, v);
            hold(k, v);
            add_up(v, s);
        }
        if (after) statistics(s, mean_y, rs_y);
        s = 0.0f;
#pragma unroll
        for (int k = 0; k < V; k++) {
            if (8 * k * THREADS >= cols) break;
            const uint32_t col = col_of(k);
            float x[8];
            Columns<DT> weight, bias, gate;
            if (after) {
                weight.ask(a.after_weight, a.flags & kNormAfterWeight32, 0, col, cols);
                bias.ask(a.after_bias, a.flags & kNormAfterBias32, 0, col, cols);
            }
            gate.ask(a.gate, a.flags & kNormGate32, (int64_t)(row / a.per) * cols, col, cols);
            look(k, x);
            if (after) {
                weight.take(a.after_weight, a.flags & kNormAfterWeight32, col, cols, 1.0f);
                bias.take(a.after_bias, a.flags & kNormAfterBias32, col, cols, 0.0f);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = (x[j] - mean_y) * rs_y * weight.v[j] + bias.v[j];
            }
            if (a.gate) {
                gate.take(a.gate, a.flags & kNormGate32, col, cols, 1.0f);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] *= gate.v[j];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] *= a.block_scale;
            if (a.residual) {
                float v[8];
                row_values<RT>(residual[k], col, cols, v);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = v[j] * a.residual_scale + x[j];
            }
            if (a.r) store_row<RT>(row_of<RT>(a.r, base), col, cols, x);
            if (a.flags & kNormKeepR) { // of r as it is stored
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = ElemIO<RT>::round(x[j]);
                keep_row<RT>(a.kept, a.rows, row, col, cols, v);
            }
            hold(k, x);
            add_up(x, s);
        }
        if (before) {
            statistics(s, mean, rs);
#pragma unroll
            for (int k = 0; k < V; k++) {
                if (8 * k * THREADS >= cols) break;
                const uint32_t col = col_of(k);
                float x[8];
                Columns<DT> weight, bias;
                weight.ask(a.weight, a.flags & kNormWeight32, 0, col, cols);
                bias.ask(a.bias, a.flags & kNormBias32, 0, col, cols);
                look(k, x);
                weight.take(a.weight, a.flags & kNormWeight32, col, cols, 1.0f);
                bias.take(a.bias, a.flags & kNormBias32, col, cols, 0.0f);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = ElemIO<DT>::round((x[j] - mean) * rs * weight.v[j] + bias.v[j]);
                store_row<DT>(row_of<DT>(a.h, base), col, cols, x);
                if (a.h8) keep_row<DT>(a.h8, a.rows, row, col, cols, x);
            }
        }
        if (a.stats && threadIdx.x == 0) reinterpret_cast<float4 *>(a.stats)[row] = make_float4(mean, rs, mean_y, rs_y);
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
struct RowMeans { // of g and g xhat, and of the norm of y likewise
    float mean, mean_xhat, mean_after, mean_yhat;
};
enum { kSumWeight = 1, kSumBias = 2, kSumGate = 4, kSumAfterWeight = 8, kSumAfterBias = 16 };

template <int DT, int RT, int V, int THREADS, int SUMS, bool EIGHT, bool PASSING, bool WIDE> __global__ __launch_bounds__(THREADS, 4) void residual_norm_backward_kernel(BlockNormBackArgs a)
{
    constexpr bool AHEAD = V == 1 && !(SUMS & ~(kSumWeight | kSumBias));
    constexpr bool AFTER = SUMS & (kSumAfterWeight | kSumAfterBias), BETWEEN = SUMS & ~(kSumWeight | kSumBias);
    __shared__ f32x2_t part[2][16];
    const uint32_t threads = a.flags >> 16, cols = a.cols;
    const bool center = a.flags & kNormCenter, after = AFTER && a.flags & kNormAfter;
    const uint32_t team = V == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / threads) : 0, lane = threadIdx.x - team * threads + (WIDE ? blockIdx.x * threads : 0);
    const uint32_t workgroup = WIDE ? blockIdx.y : blockIdx.x; // of those that share the rows
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
    const uint32_t id = workgroup * a.teams + team, of = a.parts > 1 ? id / a.parts : 0;
    const uint32_t start = a.parts > 1 ? of * a.per + (id - of * a.parts) * a.run : id * a.run;
    const uint32_t end = min(start + a.run, a.parts > 1 ? (of + 1) * a.per : a.rows);
    uint32_t left = a.per;
    // What the columns are multiplied by, in registers all along (1 where there is no weight; 0 behind the last column, where nothing else need be).
    static_assert(V == 1 || !BETWEEN, "the vectors between r and y are held of eight columns");
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
#pragma unroll
    for (int k = 0; k < V; k++) load_weight(a.weight, a.flags & kNormWeight32, 0, 8 * (lane + k * threads), weight[k]);
    if (AFTER) load_weight(a.after_weight, a.flags & kNormAfterWeight32, 0, 8 * lane, after_weight[0]);
    if (BETWEEN && a.gate) load_columns<DT>(a.gate, a.flags & kNormGate32, (int64_t)(min(start, a.rows - 1) / a.per) * cols, 8 * lane, cols, gate[0]); // (a team may have no rows)
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
        RowMeans means;
    };
    const auto col_of = [&](int k) {
        uint32_t mine = lane;
        if (V > 1 || SUMS == 31 || (AFTER && RT == DQ_F32)) asm volatile("" : "+v"(mine));
        return 8 * (mine + k * threads);
    };
    const auto load = [&](Raw &x, uint32_t row) {
        const int64_t base = (int64_t)row * cols;
#pragma unroll
        for (int k = 0; k < V; k++) {
            const uint32_t col = col_of(k);
            if (a.dh) {
                load_row<DT, PASSING>(row_of<DT>(a.dh, base), col, cols, x.dh[k]);
                load_kept(a.r, x.r[k], row, col, R());
            }
            if (a.dr) load_row<RT, PASSING>(row_of<RT>(a.dr, base), col, cols, x.dr[k]);
            if (BETWEEN && a.y) load_kept(a.y, x.y[k], row, col, Y());
        }
        x.stats = reinterpret_cast<const float4 *>(a.stats)[row];
        if (WIDE) x.means = reinterpret_cast<const RowMeans *>(a.means)[row];
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
            now.means = {0.0f, 0.0f, 0.0f, 0.0f};
        }
        const float4 stats = now.stats;
        float t[V][8];
        if (a.dh) {
            float xhat[V][8], first = 0.0f, second = 0.0f;
#pragma unroll
            for (int k = 0; k < V; k++) {
                kept_values(now.r[k], col_of(k), xhat[k], R());
                row_values<DT>(now.dh[k], col_of(k), cols, t[k]);
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
            if (WIDE) {
                first = now.means.mean;
                second = now.means.mean_xhat;
            } else {
                sums(first, second);
                first = center ? first * share : 0.0f;
                second *= share;
            }
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
            const uint32_t col = col_of(k);
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
                const uint32_t col = col_of(k);
                if (a.y) {
                    kept_values(now.y[k], col, yhat[k], Y());
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) yhat[k][j] = 0.0f;
                }
                if (after) {
#pragma unroll
                    for (int j = 0; j < 8; j++) yhat[k][j] = (yhat[k][j] - stats.z) * stats.w;
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
                if (WIDE) {
                    first = now.means.mean_after;
                    second = now.means.mean_yhat;
                } else {
                    sums(first, second);
                    first = center ? first * share : 0.0f;
                    second *= share;
                }
#pragma unroll
                for (int k = 0; k < V; k++)
#pragma unroll
                    for (int j = 0; j < 8; j++) t[k][j] = (t[k][j] - first - yhat[k][j] * second) * stats.w;
            }
        }
        if (a.dy && there) {
#pragma unroll
            for (int k = 0; k < V; k++) store_row<DT>(row_of<DT>(a.dy, base), col_of(k), cols, t[k]);
        }
        if (SUMS & kSumGate && a.gate && --left == 0) { // the last row of a gate; where all of its rows are this team's, its gradient is whole
            left = a.per;
            if (a.dgate && there) {
                const int64_t to = (int64_t)(row / a.per) * cols;
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const uint32_t col = col_of(k);
                    if (DT == DQ_F32 || a.flags & kNormGate32)
                        store_row<DQ_F32>(row_of<DQ_F32>(a.dgate, to), col, cols, acc[2][k]);
                    else
                        store_row<DT>(row_of<DT>(a.dgate, to), col, cols, acc[2][k]);
                }
                clear(2);
            }
            if (row + 1 < end) load_columns<DT>(a.gate, a.flags & kNormGate32, (int64_t)((row + 1) / a.per) * cols, 8 * lane, cols, gate[0]);
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
        char *to = row_of<DQ_F32>(a.work, ((int64_t)slot++ * a.grid + workgroup) * cols);
        if constexpr (V == 1 && THREADS == 512) {
            if (a.teams > 1) {
                __shared__ float4 both[2][512];
                __syncthreads();
                both[0][threadIdx.x] = make_float4(acc[s][0][0], acc[s][0][1], acc[s][0][2], acc[s][0][3]);
                both[1][threadIdx.x] = make_float4(acc[s][0][4], acc[s][0][5], acc[s][0][6], acc[s][0][7]);
                __syncthreads();
                if (team == 0) {
                    for (uint32_t m = 1; m < a.teams; m++) {
                        const float4 x = both[0][m * threads + threadIdx.x], y = both[1][m * threads + threadIdx.x];
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

// The means of rows that are too wide for a thread to hold its part of all arrays and sums: a workgroup goes over a row, and with a norm after the block over it again, from the cache.
// Then the kernel above takes the columns in tiles of 512 (WIDE), a wave each with a run of rows: it meets nobody.  2048 x 14336 bf16 with both norms and a gate 72 us, bound by what
// each element has to be unpacked and multiplied with more than by memory (3.3 TB/s; the same at 8 to 24 waves a CU, with one vector or two at a time), and 62 us (5.7 TB/s).
constexpr uint32_t kMeansGrid = 1024; // as many as the chip holds, and as many again
template <int DT, int RT, bool EIGHT> __global__ __launch_bounds__(512, 4) void residual_norm_means_kernel(BlockNormBackArgs a)
{
    __shared__ f32x2_t part[2][16];
    const uint32_t cols = a.cols;
    const bool center = a.flags & kNormCenter, after = a.flags & kNormAfter;
    const float share = 1.0f / (float)cols;
    GroupSums sums = {part, 8, 0};
    typedef std::integral_constant<int, DT> Y;
    typedef std::integral_constant<int, RT> R;
    const auto load_kept = [&](const void *p, auto &x, uint32_t row, uint32_t col, auto type) {
        constexpr int T = decltype(type)::value;
        if (EIGHT) {
            const CheckpointOf<const uint8_t> c(static_cast<const uint8_t *>(p), a.rows, cols);
            const uint32_t from = min(col, 32 * c.blocks - 8);
            const u32x2_t w = *reinterpret_cast<const u32x2_t *>(c.codes + (int64_t)row * 32 * c.blocks + from);
            x[0] = w[0];
            x[1] = w[1];
            x[2] = (c.scales + (int64_t)row * c.blocks)[from >> 5];
        } else {
            load_row<T>(row_of<T>(p, (int64_t)row * cols), col, cols, x);
        }
    };
    const auto kept_values = [&](auto &x, uint32_t col, float (&v)[8], auto type) {
        constexpr int T = decltype(type)::value;
        if (EIGHT) {
            const u32x2_t w = {x[0], x[1]};
            decode_e4m3(w, x[2], v);
            clip(v, lanes_own(col, cols));
        } else {
            row_values<T>(x, col, cols, v);
        }
    };
    // 1 where there is no such vector, and 0 behind the last column
    const auto load_weight = [&](const void *p, bool in32, int64_t base, uint32_t col, float (&v)[8]) {
        if (p) {
            load_columns<DT>(p, in32, base, col, cols, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = 1.0f;
            clip(v, lanes_own(col, cols));
        }
    };
    for (uint32_t row = blockIdx.x; row < a.rows; row += kMeansGrid) {
        const int64_t base = (int64_t)row * cols;
        const float4 stats = reinterpret_cast<const float4 *>(a.stats)[row];
        RowMeans means = {0.0f, 0.0f, 0.0f, 0.0f};
        if (a.dh) {
            float first = 0.0f, second = 0.0f;
            for (uint32_t at = 8 * threadIdx.x; at < cols; at += 8192) {
                uint32_t dh[2][kWords<DT>], r[2][kWords<RT>];
                float weight[2][8];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    load_row<DT>(row_of<DT>(a.dh, base), at + 4096 * k, cols, dh[k]);
                    load_kept(a.r, r[k], row, at + 4096 * k, R());
                }
#pragma unroll
                for (int k = 0; k < 2; k++) load_weight(a.weight, a.flags & kNormWeight32, 0, at + 4096 * k, weight[k]);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    float g[8], xhat[8];
                    row_values<DT>(dh[k], at + 4096 * k, cols, g);
                    kept_values(r[k], at + 4096 * k, xhat, R());
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        g[j] *= weight[k][j];
                        first += g[j];
                        second += g[j] * ((xhat[j] - stats.x) * stats.y);
                    }
                }
            }
            sums(first, second);
            means.mean = center ? first * share : 0.0f;
            means.mean_xhat = second * share;
        }
        if (after) {
            float first = 0.0f, second = 0.0f;
            for (uint32_t at = 8 * threadIdx.x; at < cols; at += 8192) {
                uint32_t dh[2][kWords<DT>], r[2][kWords<RT>], dr[2][kWords<RT>], y[2][kWords<DT>];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const uint32_t col = at + 4096 * k;
                    if (a.dh) {
                        load_row<DT>(row_of<DT>(a.dh, base), col, cols, dh[k]);
                        load_kept(a.r, r[k], row, col, R());
                    }
                    if (a.dr) load_row<RT>(row_of<RT>(a.dr, base), col, cols, dr[k]);
                    if (a.y) load_kept(a.y, y[k], row, col, Y());
                }
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const uint32_t col = at + 4096 * k;
                    float t[8], v[8];
                    if (a.dh) {
                        row_values<DT>(dh[k], col, cols, t);
                        kept_values(r[k], col, v, R());
                        float weight[8];
                        load_weight(a.weight, a.flags & kNormWeight32, 0, col, weight);
#pragma unroll
                        for (int j = 0; j < 8; j++) t[j] = (t[j] * weight[j] - means.mean - (v[j] - stats.x) * stats.y * means.mean_xhat) * stats.y;
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++) t[j] = 0.0f;
                    }
                    if (a.dr) {
                        row_values<RT>(dr[k], col, cols, v);
#pragma unroll
                        for (int j = 0; j < 8; j++) t[j] += v[j];
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++) t[j] *= a.block_scale;
                    if (a.gate) {
                        load_columns<DT>(a.gate, a.flags & kNormGate32, (int64_t)(row / a.per) * cols, col, cols, v);
#pragma unroll
                        for (int j = 0; j < 8; j++) t[j] *= v[j];
                    }
                    load_weight(a.after_weight, a.flags & kNormAfterWeight32, 0, col, v);
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        t[j] *= v[j]; // (0 behind the last column)
                        first += t[j];
                    }
                    if (a.y) {
                        kept_values(y[k], col, v, Y());
#pragma unroll
                        for (int j = 0; j < 8; j++) second += t[j] * ((v[j] - stats.z) * stats.w);
                    }
                }
            }
            sums(first, second);
            means.mean_after = center ? first * share : 0.0f;
            means.mean_yhat = second * share;
        }
        if (threadIdx.x == 0) reinterpret_cast<RowMeans *>(a.means)[row] = means;
    }
}

// ---- launches for one type of activations --------------------------------------------------------------------

template <int DT, int RT> static hipError_t launch_norm_of(const BlockNormArgs &a, hipStream_t stream)
{
    const uint32_t threads = a.flags >> 16;
    const dim3 grid(a.grid), block(threads);
    const bool full = a.gate || a.flags & kNormAfter, passing = a.flags & kNormPassing;
    if (a.cols > 16384) return launch_with(residual_norm_wide_kernel<DT, RT, 1024>, grid, dim3(1024), stream, a);
    if (a.cols > 8192 && full) return launch_with(residual_norm_wide_kernel<DT, RT, 512>, grid, dim3(512), stream, a);
    if (a.cols > 8192) return launch_with(residual_norm_kernel<DT, RT, 2, 1024, false, true>, grid, block, stream, a);
    if (threads > 512)
        return full ? passing ? launch_with(residual_norm_kernel<DT, RT, 1, 1024, true, true>, grid, block, stream, a) : launch_with(residual_norm_kernel<DT, RT, 1, 1024, true, false>, grid, block, stream, a)
                    : passing ? launch_with(residual_norm_kernel<DT, RT, 1, 1024, false, true>, grid, block, stream, a) : launch_with(residual_norm_kernel<DT, RT, 1, 1024, false, false>, grid, block, stream, a);
    return full ? passing ? launch_with(residual_norm_kernel<DT, RT, 1, 512, true, true>, grid, block, stream, a) : launch_with(residual_norm_kernel<DT, RT, 1, 512, true, false>, grid, block, stream, a)
                : passing ? launch_with(residual_norm_kernel<DT, RT, 1, 512, false, true>, grid, block, stream, a) : launch_with(residual_norm_kernel<DT, RT, 1, 512, false, false>, grid, block, stream, a);
}

template <int DT, int RT, int V, int THREADS, int SUMS, bool WIDE = false> static hipError_t launch_norm_backward_with(const BlockNormBackArgs &a, hipStream_t stream)
{
    const dim3 grid = WIDE ? dim3((a.cols + 511) / 512, a.grid) : dim3(a.grid), block((a.flags >> 16) * a.teams);
    if constexpr (V == 1) {
        if (a.flags & kNormPassing)
            return a.flags & kNormEight ? launch_with(residual_norm_backward_kernel<DT, RT, V, THREADS, SUMS, true, true, WIDE>, grid, block, stream, a)
                                        : launch_with(residual_norm_backward_kernel<DT, RT, V, THREADS, SUMS, false, true, WIDE>, grid, block, stream, a);
    }
    return a.flags & kNormEight ? launch_with(residual_norm_backward_kernel<DT, RT, V, THREADS, SUMS, true, false, WIDE>, grid, block, stream, a)
                                : launch_with(residual_norm_backward_kernel<DT, RT, V, THREADS, SUMS, false, false, WIDE>, grid, block, stream, a);
}
template <int DT, int RT> static hipError_t launch_norm_backward_of(const BlockNormBackArgs &a, hipStream_t stream)
{
    // the block between r and y takes part only in kernels that keep sums of it
    const uint32_t want = a.sums | (a.gate ? kSumGate : 0) | (a.flags & kNormAfter ? kSumAfterWeight : 0);
    const auto within = [&](uint32_t of) { return !(want & ~of); };
    if (a.means) {
        const dim3 grid(std::min(a.rows, kMeansGrid)), block(512);
        const hipError_t e = a.flags & kNormEight ? launch_with(residual_norm_means_kernel<DT, RT, true>, grid, block, stream, a) : launch_with(residual_norm_means_kernel<DT, RT, false>, grid, block, stream, a);
        if (e != hipSuccess) return e;
        return within(3) ? launch_norm_backward_with<DT, RT, 1, 512, 3, true>(a, stream)
             : within(13) ? launch_norm_backward_with<DT, RT, 1, 512, 13, true>(a, stream) : launch_norm_backward_with<DT, RT, 1, 512, 31, true>(a, stream);
    }
    if (a.cols > 8192) return within(1) ? launch_norm_backward_with<DT, RT, 2, 1024, 1>(a, stream) : launch_norm_backward_with<DT, RT, 2, 1024, 3>(a, stream);
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
