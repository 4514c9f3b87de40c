// The norms around a block, its gate and the residual: kernels for one type of activations (dq_residual_norm_*.hip have one each).
//
//   z = norm(y; after_weight, after_bias) or y,   r = residual_scale residual + block_scale gate z,   h = norm(r; weight, bias)
//
// A workgroup takes a row (64 to 1024 threads, eight elements of a thread together, up to four times), holds it in registers from the loads to the stores, and reduces through
// LDS: every array moves once.  Backward it takes a run of rows and keeps what the weights' and the gate's gradients add up to in registers; what workgroups have of the same
// columns is added in the order of the rows by a second launch.
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

// Sums over a workgroup's threads, in every one of them: a wave's, and then 16 lanes add what up to 16 waves have left.  Two buffers in turn: who writes one for the second time has
// met, in the sum between, everybody who still read it.
struct GroupSums {
    f32x2_t (*part)[16];
    uint32_t waves;
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
        const f32x2_t v = at[min(w, waves - 1)];
        a = row16_sum(w < waves ? v.x : 0.0f);
        b = row16_sum(w < waves ? v.y : 0.0f);
    }
};

// 1 / sqrt(x) to the last place but for one in thousands: a step in 64 bits from an estimate that is good to 2^-22
__device__ __forceinline__ float inverse_root(float x)
{
    const double y = __builtin_amdgcn_rsqf(x), rest = 1.0 - (double)x * y * y;
    return (float)(y + 0.5 * y * rest);
}

// Eight elements of a row as words, 0 behind the last column.  A lane whose eight reach past the end loads the last eight of the row and moves them up: no lane loads less or
// apart (columns are eight at least).
template <int DT> __device__ __forceinline__ void load_row(const void *p, int64_t base, uint32_t col, uint32_t cols, uint32_t (&x)[kWords<DT>])
{
    const uint32_t from = min(col, cols - 8);
    load_words<DT>(p, base + from, x);
    const uint32_t up = min(col - from, 8u);
    if (up) {
        constexpr int N = kWords<DT>;
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
// the elements that a lane has of a row, and zeros in place of the others
__device__ __forceinline__ int lanes_own(uint32_t col, uint32_t cols) { return (int)min(cols - min(col, cols), 8u); }
__device__ __forceinline__ void clip(float (&v)[8], int own)
{
    if (own < 8) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = j < own ? v[j] : 0.0f;
    }
}
template <int DT> __device__ __forceinline__ void row_values(const uint32_t (&x)[kWords<DT>], float (&v)[8])
{
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = word_value<DT>(x, j);
}
// eight elements of a weight, a bias or a gate, which are of the activations' type or float32; 0 behind the last column
template <int DT> __device__ __forceinline__ void load_columns(const void *p, bool in32, int64_t base, uint32_t col, uint32_t cols, float (&v)[8])
{
    if (DT == DQ_F32 || in32) {
        uint32_t x[8];
        load_row<DQ_F32>(p, base, col, cols, x);
        row_values<DQ_F32>(x, v);
    } else {
        uint32_t x[kWords<DT>];
        load_row<DT>(p, base, col, cols, x);
        row_values<DT>(x, v);
    }
}
template <int DT> __device__ __forceinline__ void store_row(void *p, int64_t base, uint32_t col, uint32_t cols, const float (&v)[8])
{
    if (col + 8 <= cols)
        store8<DT>(p, base + col, v);
    else if (col < cols)
        store_part<DT, 8>(p, base + col, (int)(cols - col), v);
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

template <int DT, int RT, int V, int THREADS> __global__ __launch_bounds__(THREADS) void residual_norm_kernel(BlockNormArgs a)
{
    __shared__ f32x2_t part[2][16];
    const uint32_t threads = a.flags >> 16, cols = a.cols;
    const bool center = a.flags & kNormCenter, after = a.flags & kNormAfter, before = a.flags & kNormBefore;
    GroupSums sums = {part, threads >> 6};
    // mean and 1 / sqrt(var + eps) of a row, whose elements past the last column are 0
    const auto statistics = [&](const float (&x)[V][8], float &mean, float &rs) {
        float s = 0.0f, none = 0.0f;
        mean = 0.0f;
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
    const auto normalise = [&](float (&x)[8], float mean, float rs, const void *weight, bool weight32, const void *bias, bool bias32, uint32_t col) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = (x[j] - mean) * rs;
        if (weight) {
            load_columns<DT>(weight, weight32, 0, col, cols, v);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] *= v[j];
        }
        if (bias) {
            load_columns<DT>(bias, bias32, 0, col, cols, v);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] += v[j];
        }
        clip(x, lanes_own(col, cols));
    };
    for (uint32_t row = blockIdx.x; row < a.rows; row += a.grid) {
        const int64_t base = (int64_t)row * cols;
        uint32_t yw[V][kWords<DT>], rw[V][kWords<RT>];
#pragma unroll
        for (int k = 0; k < V; k++) load_row<DT>(a.y, base, 8 * (threadIdx.x + k * threads), cols, yw[k]);
        if (a.residual) {
#pragma unroll
            for (int k = 0; k < V; k++) load_row<RT>(a.residual, base, 8 * (threadIdx.x + k * threads), cols, rw[k]);
        }
        float x[V][8], mean_y = 0.0f, rs_y = 1.0f;
#pragma unroll
        for (int k = 0; k < V; k++) row_values<DT>(yw[k], x[k]);
        if (a.flags & kNormKeepY) {
            uint8_t *data = a.kept + (a.flags & kNormKeepR ? (((int64_t)a.rows * ((cols + 31) >> 5) * 33 + 15) & ~(int64_t)15) : 0);
#pragma unroll
            for (int k = 0; k < V; k++) keep_row<DT>(data, a.rows, row, 8 * (threadIdx.x + k * threads), cols, x[k]);
        }
        if (after) statistics(x, mean_y, rs_y);
#pragma unroll
        for (int k = 0; k < V; k++) {
            const uint32_t col = 8 * (threadIdx.x + k * threads);
            if (after) {
                normalise(x[k], mean_y, rs_y, a.after_weight, a.flags & kNormAfterWeight32, a.after_bias, a.flags & kNormAfterBias32, col);
            }
            if (a.gate) {
                float g[8];
                load_columns<DT>(a.gate, a.flags & kNormGate32, (int64_t)(row / a.per) * cols, col, cols, g);
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] *= g[j];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) x[k][j] *= a.block_scale;
            if (a.residual) {
                float v[8];
                row_values<RT>(rw[k], v);
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] = v[j] * a.residual_scale + x[k][j];
            }
            if (a.r) store_row<RT>(a.r, base, col, cols, x[k]);
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
                normalise(x[k], mean, rs, a.weight, a.flags & kNormWeight32, a.bias, a.flags & kNormBias32, col);
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] = ElemIO<DT>::round(x[k][j]);
                store_row<DT>(a.h, base, col, cols, x[k]);
                if (a.h8) keep_row<DT>(a.h8, a.rows, row, col, cols, x[k]);
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
// SUMS: which of them registers are kept for, at least those that are wanted.
enum { kSumWeight = 1, kSumBias = 2, kSumGate = 4, kSumAfterWeight = 8, kSumAfterBias = 16 };

template <int DT, int RT, int V, int THREADS, int SUMS> __global__ __launch_bounds__(THREADS) void residual_norm_backward_kernel(BlockNormBackArgs a)
{
    __shared__ f32x2_t part[2][16];
    const uint32_t threads = a.flags >> 16, cols = a.cols, sums_wanted = a.sums;
    const bool center = a.flags & kNormCenter, after = a.flags & kNormAfter, eight = a.flags & kNormEight;
    GroupSums sums = {part, threads >> 6};
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
    // the workgroup's rows: of one gate, or of whole ones
    const uint32_t of = a.parts > 1 ? blockIdx.x / a.parts : 0;
    const uint32_t start = a.parts > 1 ? of * a.per + (blockIdx.x - of * a.parts) * a.run : blockIdx.x * a.run;
    const uint32_t end = min(start + a.run, a.parts > 1 ? (of + 1) * a.per : a.rows);
    uint32_t left = a.per;
    const auto load_kept = [&](const void *p, auto &x, int64_t row, uint32_t col, auto type) {
        constexpr int T = decltype(type)::value;
        if (eight) {
            const CheckpointOf<const uint8_t> c(static_cast<const uint8_t *>(p), a.rows, cols);
            const uint32_t from = min(col, 32 * c.blocks - 8);
            const u32x2_t w = *reinterpret_cast<const u32x2_t *>(c.codes + row * 32 * c.blocks + from);
            x[0] = w[0];
            x[1] = w[1];
            x[2] = c.scales[row * c.blocks + (from >> 5)];
        } else {
            load_row<T>(p, row * cols, col, cols, x);
        }
    };
    const auto kept_values = [&](const auto &x, float (&v)[8], auto type) {
        constexpr int T = decltype(type)::value;
        if (eight) {
            const u32x2_t w = {x[0], x[1]};
            decode_e4m3(w, x[2], v);
        } else {
            row_values<T>(x, v);
        }
    };
    typedef std::integral_constant<int, DT> Y;
    typedef std::integral_constant<int, RT> R;
    for (uint32_t row = start; row < end; row++) {
        const int64_t base = (int64_t)row * cols;
        uint32_t dhw[V][kWords<DT>], drw[V][kWords<RT>], rw[V][kWords<RT>], yw[V][kWords<DT>];
#pragma unroll
        for (int k = 0; k < V; k++) {
            const uint32_t col = 8 * (threadIdx.x + k * threads);
            if (a.dh) {
                load_row<DT>(a.dh, base, col, cols, dhw[k]);
                load_kept(a.r, rw[k], row, col, R());
            }
            if (a.dr) load_row<RT>(a.dr, base, col, cols, drw[k]);
            if (a.y) load_kept(a.y, yw[k], row, col, Y());
        }
        const float4 stats = reinterpret_cast<const float4 *>(a.stats)[row];
        float t[V][8];
        if (a.dh) {
            float xhat[V][8], first = 0.0f, second = 0.0f;
#pragma unroll
            for (int k = 0; k < V; k++) {
                const uint32_t col = 8 * (threadIdx.x + k * threads);
                float w[8], v[8];
                kept_values(rw[k], v, R());
                row_values<DT>(dhw[k], t[k]);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    xhat[k][j] = (v[j] - stats.x) * stats.y;
                    if (SUMS & kSumWeight) acc[0][k][j] += t[k][j] * xhat[k][j];
                    if (SUMS & kSumBias) acc[1][k][j] += t[k][j];
                }
                if (a.weight) {
                    load_columns<DT>(a.weight, a.flags & kNormWeight32, 0, col, cols, w);
#pragma unroll
                    for (int j = 0; j < 8; j++) t[k][j] *= w[j];
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
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
            const uint32_t col = 8 * (threadIdx.x + k * threads);
            float v[8];
            if (a.dr) {
                row_values<RT>(drw[k], v);
#pragma unroll
                for (int j = 0; j < 8; j++) t[k][j] += v[j];
            }
            if (a.dresidual) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = t[k][j] * a.residual_scale;
                store_row<RT>(a.dresidual, base, col, cols, v);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) t[k][j] *= a.block_scale;
        }
        if (SUMS & (kSumGate | kSumAfterWeight | kSumAfterBias)) {
            if (a.y) {
                float yhat[V][8], first = 0.0f, second = 0.0f;
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const uint32_t col = 8 * (threadIdx.x + k * threads);
                    float w[8], v[8];
                    kept_values(yw[k], yhat[k], Y());
                    if (after) {
#pragma unroll
                        for (int j = 0; j < 8; j++) yhat[k][j] = (yhat[k][j] - stats.z) * stats.w;
                        clip(t[k], lanes_own(col, cols));
                    }
                    if (after && a.after_weight) {
                        load_columns<DT>(a.after_weight, a.flags & kNormAfterWeight32, 0, col, cols, w);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j++) w[j] = 1.0f;
                    }
                    if (SUMS & kSumGate && sums_wanted & kSumGate) {
#pragma unroll
                        for (int j = 0; j < 8; j++) acc[2][k][j] += t[k][j] * (yhat[k][j] * w[j]);
                        if (a.after_bias) {
                            load_columns<DT>(a.after_bias, a.flags & kNormAfterBias32, 0, col, cols, v);
#pragma unroll
                            for (int j = 0; j < 8; j++) acc[2][k][j] += t[k][j] * v[j];
                        }
                    }
                    if (a.gate) {
                        load_columns<DT>(a.gate, a.flags & kNormGate32, (int64_t)(row / a.per) * cols, col, cols, v);
#pragma unroll
                        for (int j = 0; j < 8; j++) t[k][j] *= v[j];
                    }
                    if (after) {
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            if (SUMS & kSumAfterWeight) acc[3][k][j] += t[k][j] * yhat[k][j];
                            if (SUMS & kSumAfterBias) acc[4][k][j] += t[k][j];
                            t[k][j] *= w[j];
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
            } else if (a.gate) {
#pragma unroll
                for (int k = 0; k < V; k++) {
                    float g[8];
                    load_columns<DT>(a.gate, a.flags & kNormGate32, (int64_t)(row / a.per) * cols, 8 * (threadIdx.x + k * threads), cols, g);
#pragma unroll
                    for (int j = 0; j < 8; j++) t[k][j] *= g[j];
                }
            }
        }
        if (a.dy) {
#pragma unroll
            for (int k = 0; k < V; k++) store_row<DT>(a.dy, base, 8 * (threadIdx.x + k * threads), cols, t[k]);
        }
        if (SUMS & kSumGate && a.dgate && --left == 0) { // the last row of a gate that no other workgroup has rows of
            left = a.per;
            const int64_t to = (int64_t)(row / a.per) * cols;
#pragma unroll
            for (int k = 0; k < V; k++) {
                const uint32_t col = 8 * (threadIdx.x + k * threads);
                if (DT == DQ_F32 || a.flags & kNormGate32)
                    store_row<DQ_F32>(a.dgate, to, col, cols, acc[2][k]);
                else
                    store_row<DT>(a.dgate, to, col, cols, acc[2][k]);
            }
            clear(2);
        }
    }
    uint32_t slot = 0;
#pragma unroll
    for (int s = 0; s < 5; s++) {
        if (!(SUMS >> s & 1) || !(sums_wanted >> s & 1) || (s == 2 && a.dgate)) continue;
        const int64_t to = ((int64_t)slot++ * a.grid + blockIdx.x) * cols;
#pragma unroll
        for (int k = 0; k < V; k++) store_row<DQ_F32>(a.work, to, 8 * (threadIdx.x + k * threads), cols, acc[s][k]);
    }
}

// ---- launches for one type of activations --------------------------------------------------------------------

template <int DT, int RT> static hipError_t launch_norm_of(const BlockNormArgs &a, hipStream_t stream)
{
    const uint32_t threads = a.flags >> 16;
    const dim3 grid(a.grid), block(threads);
    return a.cols > 16384 ? launch_with(residual_norm_kernel<DT, RT, 4, 1024>, grid, block, stream, a)
         : a.cols > 8192 ? launch_with(residual_norm_kernel<DT, RT, 2, 1024>, grid, block, stream, a)
         : threads > 256 ? launch_with(residual_norm_kernel<DT, RT, 1, 1024>, grid, block, stream, a) : launch_with(residual_norm_kernel<DT, RT, 1, 256>, grid, block, stream, a);
}

template <int DT, int RT, int SUMS> static hipError_t launch_norm_backward_with(const BlockNormBackArgs &a, hipStream_t stream)
{
    const uint32_t threads = a.flags >> 16;
    const dim3 grid(a.grid), block(threads);
    return a.cols > 16384 ? launch_with(residual_norm_backward_kernel<DT, RT, 4, 1024, SUMS>, grid, block, stream, a)
         : a.cols > 8192 ? launch_with(residual_norm_backward_kernel<DT, RT, 2, 1024, SUMS>, grid, block, stream, a)
         : threads > 512 ? launch_with(residual_norm_backward_kernel<DT, RT, 1, 1024, SUMS>, grid, block, stream, a)
                         : launch_with(residual_norm_backward_kernel<DT, RT, 1, 512, SUMS>, grid, block, stream, a);
}
template <int DT, int RT> static hipError_t launch_norm_backward_of(const BlockNormBackArgs &a, hipStream_t stream)
{
    // the block between r and y takes part only in kernels that keep sums of it
    const uint32_t want = a.sums | (a.gate ? kSumGate : 0) | (a.flags & kNormAfter ? kSumAfterWeight : 0);
    if (!(want & ~kSumWeight)) return launch_norm_backward_with<DT, RT, kSumWeight>(a, stream);
    if (!(want & ~(kSumWeight | kSumBias))) return launch_norm_backward_with<DT, RT, kSumWeight | kSumBias>(a, stream);
    if (!(want & ~(kSumWeight | kSumGate))) return launch_norm_backward_with<DT, RT, kSumWeight | kSumGate>(a, stream);
    if (!(want & ~(kSumWeight | kSumGate | kSumAfterWeight))) return launch_norm_backward_with<DT, RT, kSumWeight | kSumGate | kSumAfterWeight>(a, stream);
    return launch_norm_backward_with<DT, RT, 31>(a, stream);
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
