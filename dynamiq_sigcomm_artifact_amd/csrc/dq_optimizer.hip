// The end of a training step: the norm of all gradients with the factor that clips them, and the AdamW step over many tensors.
//
// Both stream their tensors once and are bound by memory.  A launch takes its tensors as kernel arguments and cuts each into tiles; a workgroup finds
// the tensor of its tile with a load or two per lane and a ballot.  Nothing about the tensors is kept between calls.
#include "dq_launch.h"
#include "dq_microscale.cuh"

namespace dq {

// the tensor that tile `tile` belongs to: the last one that starts at or before it
template <int TENSORS> __device__ __forceinline__ int tensor_of(const uint32_t (&first_tile)[TENSORS], uint32_t tile)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
#pragma unroll
    for (int k = 0; k < TENSORS; k += 64)
        before += __builtin_popcountll(__builtin_amdgcn_ballot_w64((TENSORS % 64 == 0 || k + lane < TENSORS) && first_tile[min(k + lane, TENSORS - 1)] <= tile));
    return __builtin_amdgcn_readfirstlane(before - 1);
}

// ---- the norm ---------------------------------------------------------------------------------------------

constexpr int kNormTile = 256 * 32;

__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// the sum over a workgroup's threads, in its first one
__device__ __forceinline__ double group_sum(double v)
{
    __shared__ double part[4];
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

__device__ __forceinline__ void put_norm(double sum, double max_norm, float *out)
{
    const double norm = __builtin_sqrt(sum), factor = __builtin_fmin(1.0, max_norm / (norm + 1e-6));
    out[0] = (float)norm;
    out[1] = __builtin_isfinite(norm) ? (float)factor : __builtin_nanf("");
}

// Squares are taken and added in 64 bits: a gradient beyond 2^64 or below 2^-63 has no square in 32, and a sum of 10^8 terms is as exact as
// its terms.  A workgroup adds its tiles up and leaves one number for grad_norm_end_kernel, which adds those.  (Workgroups that count themselves, the last of which
// adds, take longer than a second launch: 800 of them 27 us where the two launches take 9, an atomic on one address being some 30 ns.)  Bound by memory: 249 MB of
// bf16 in 148 tensors in 49.5 us, 5.0 TB/s; 26 MB in 8.3, of which the second launch takes 3.
template <int DT, int TENSORS> __global__ __launch_bounds__(256) void grad_norm_kernel(NormArgs<TENSORS> a)
{
    const int t = threadIdx.x;
    double sum = 0.0;
    for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        const int k = tensor_of(a.first_tile, tile);
        const void *p = a.data[k];
        const int64_t n = a.n[k], at = (int64_t)(tile - a.first_tile[k]) * kNormTile;
        constexpr int kPer = DT == DQ_F32 ? 4 : 8; // elements of 16 bytes
        float v[32 / kPer][8];
        if (at + kNormTile <= n) {
#pragma unroll
            for (int j = 0; j < 32 / kPer; j++) {
                const int64_t i = at + kPer * (256 * j + t);
                if (DT == DQ_F32)
                    load4<DT>(p, i, v[j]);
                else
                    load8<DT>(p, i, v[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32 / kPer; j++) {
                const int64_t i = at + kPer * (256 * j + t);
                if (i + kPer > n)
                    load_part<DT, kPer>(p, i, n, v[j]);
                else if (DT == DQ_F32)
                    load4<DT>(p, i, v[j]);
                else
                    load8<DT>(p, i, v[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 32 / kPer; j++)
#pragma unroll
            for (int e = 0; e < kPer; e++) sum = __builtin_fma((double)v[j][e], (double)v[j][e], sum);
    }
    sum = group_sum(sum);
    if (t == 0) {
        if (blockIdx.x < a.slots_before) sum += a.partial[blockIdx.x];
        a.partial[blockIdx.x] = sum;
        if (a.out) put_norm(sum, a.max_norm, a.out);
    }
}

__global__ __launch_bounds__(256) void grad_norm_end_kernel(NormEnd a)
{
    double v[kNormGrid / 256];
#pragma unroll
    for (int k = 0; k < kNormGrid / 256; k++) {
        const uint32_t s = 256 * k + threadIdx.x;
        v[k] = a.partial[min(s, a.slots - 1)];
        if (s >= a.slots) v[k] = 0.0;
    }
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kNormGrid / 256; k++) sum += v[k];
    sum = group_sum(sum);
    if (threadIdx.x == 0) put_norm(sum, a.max_norm, a.out);
}

struct NormCall {
    const dq_span_t *spans;
    int count, next;
    double *partial;
    double max_norm;
    float *out;
    uint32_t slots;
    hipStream_t stream;
};

// one launch: tensors of one element type, one after the other, from c.next on
template <int TENSORS> static hipError_t launch_norm(NormCall &c)
{
    NormArgs<TENSORS> a;
    const int dtype = c.spans[c.next].dtype;
    int take = 0;
    int64_t tiles = 0;
    const bool first = c.next == 0;
    for (; c.next < c.count && take < TENSORS && c.spans[c.next].dtype == dtype; c.next++) {
        const dq_span_t &x = c.spans[c.next];
        const int64_t more = (x.n + kNormTile - 1) / kNormTile;
        if (take && tiles + more > 0x7fffffff) break;
        if (more == 0) continue;
        a.first_tile[take] = (uint32_t)tiles;
        a.data[take] = x.data;
        a.n[take++] = x.n;
        tiles += more;
    }
    const bool alone = first && c.next == c.count && tiles <= 2; // the whole call is work for one workgroup
    if (tiles == 0 && !alone) return hipSuccess;
    for (int j = take; j < TENSORS; j++) a.first_tile[j] = 0xffffffffu;
    a.partial = c.partial;
    a.out = alone ? c.out : nullptr;
    a.max_norm = c.max_norm;
    a.tiles = (uint32_t)tiles;
    a.slots_before = c.slots;
    const uint32_t grid = alone ? 1 : (uint32_t)std::min<int64_t>(tiles, kNormGrid);
    c.slots = std::max(c.slots, grid);
    if (alone) c.out = nullptr;
    return dtype == DQ_F32 ? launch_with(grad_norm_kernel<DQ_F32, TENSORS>, dim3(grid), dim3(256), c.stream, a)
         : dtype == DQ_BF16 ? launch_with(grad_norm_kernel<DQ_BF16, TENSORS>, dim3(grid), dim3(256), c.stream, a)
                            : launch_with(grad_norm_kernel<DQ_F16, TENSORS>, dim3(grid), dim3(256), c.stream, a);
}

hipError_t launch_grad_norm(const dq_span_t *spans, int count, double max_norm, double *work, float *out, hipStream_t stream)
{
    const dq_span_t nothing = {nullptr, 0, DQ_F32, 0};
    NormCall c = {count ? spans : &nothing, std::max(count, 1), 0, work, max_norm, out, 0, stream};
    hipError_t e = hipSuccess;
    while (c.next < c.count && e == hipSuccess) e = c.count - c.next <= 8 ? launch_norm<8>(c) : launch_norm<192>(c);
    if (e != hipSuccess || !c.out) return e;
    if (c.slots == 0) { // several types, all of nothing
        c.next = c.count = 1;
        c.spans = &nothing;
        c.next = 0;
        return launch_norm<8>(c);
    }
    const NormEnd end = {work, out, max_norm, c.slots};
    return launch_with(grad_norm_end_kernel, dim3(1), dim3(256), stream, end);
}

// ---- AdamW ------------------------------------------------------------------------------------------------

constexpr int kStepTile = 256 * 8;

struct Coefficients {
    float keep, step, root; // 1 - lr decay; lr / (1 - beta1^t); 1 / sqrt(1 - beta2^t)
    uint32_t dither;        // t times its constant
};

constexpr uint32_t kDitherElement = 0x9E3779B9u, kDitherStep = 0xB504F333u;

// An 8-bit state is E4M3, whose codes are a sixteenth to an eighth apart; a moment that decays by a thousandth a step would never leave its code if it were
// rounded to nearest.  So what is cut away is added up over the steps instead: a dither of 20 bits, the fractions of i phi + t / sqrt 2, is added where the
// bits are cut, and over the steps of one element, and over the elements of one step, these fractions are spread evenly: the mean error goes to zero as
// 1 / steps.  v_cvt_sr_fp8_f32 adds the upper 20 bits of its seed in this way, at normal and at subnormal codes.
template <int J> __device__ __forceinline__ uint32_t cut_e4m3(float y, uint32_t seed, uint32_t word) { return __builtin_amdgcn_cvt_sr_fp8_f32(y, seed, word, J); }

__device__ __forceinline__ uint32_t cut4(const float (&y)[4], uint32_t seed, uint32_t flip)
{
    uint32_t w = 0;
    w = cut_e4m3<0>(y[0], seed ^ flip, w);
    w = cut_e4m3<1>(y[1], (seed + kDitherElement) ^ flip, w);
    w = cut_e4m3<2>(y[2], (seed + 2u * kDitherElement) ^ flip, w);
    return cut_e4m3<3>(y[3], (seed + 3u * kDitherElement) ^ flip, w);
}

// the largest magnitude of a block that eight neighbouring lanes hold four elements each of, as a bit pattern
__device__ __forceinline__ uint32_t block_max4(const float *v)
{
    uint32_t u = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) u = max(u, __float_as_uint(v[j]) & 0x7fffffffu);
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0xB1, 0xf, 0xf, true));  // quad_perm [1,0,3,2]
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x4E, 0xf, 0xf, true));  // quad_perm [2,3,0,1]
    u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x141, 0xf, 0xf, true)); // row_half_mirror
    return u;
}

template <bool PASSING> __device__ __forceinline__ uint32_t load_word(const uint8_t *p)
{
    const uint32_t *q = reinterpret_cast<const uint32_t *>(p);
    return PASSING ? __builtin_nontemporal_load(q) : *q;
}
template <bool PASSING> __device__ __forceinline__ void store_word(uint8_t *p, uint32_t w)
{
    uint32_t *q = reinterpret_cast<uint32_t *>(p);
    if (PASSING)
        __builtin_nontemporal_store(w, q);
    else
        *q = w;
}

// Square roots of eight numbers that are not negative.  Between 2^-100 and 2^120, and of 0: v / sqrt(v) from v_rsq_f32, corrected by half of what its square lacks times
// 1 / sqrt(v), which leaves it rounded to nearest (but for one in millions, whose two neighbours are all but equally near); 8 issue cycles an element where the
// compiler's root, which also handles what is outside, takes 17.  Anything outside takes that one, for the whole wave.
__device__ __forceinline__ void roots8(const float (&v)[8], float (&r)[8])
{
    uint32_t least = ~0u, most = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        least = min(least, __float_as_uint(v[j]) - 1u); // (0 is above all)
        most = max(most, __float_as_uint(v[j]));
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float s = __builtin_amdgcn_rsqf(__builtin_fmaxf(v[j], 0x1p-126f)), q = v[j] * s;
        r[j] = __builtin_fmaf(__builtin_fmaf(-q, q, v[j]), 0.5f * s, q);
    }
    if (DQ_UNLIKELY(__builtin_amdgcn_ballot_w64(least < 0x0d800000u - 1u || most >= 0x7b800000u) != 0)) {
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = __builtin_sqrtf(v[j]);
    }
}

// PASSING: a launch moves more than the 256 MB of cache in front of the memory hold, so that nothing of it is there at the next step.  (That goes by the launch: a step of several,
// each below that, runs without the hint even if together they are beyond it.)  With the hint that says so on every load and
// store 124,439,808 binary32 weights take 593 us with 32-bit states and 328 with 8-bit ones where they take 667 and 385 without it (5.9 and 6.1 TB/s for 5.2; in 148
// tensors at odd addresses 622 and 358 for 671 and 376; on the loads or the stores alone it gains little or loses).  A bucket of 6,553,600, whose 183 MB stay, takes
// 32 us without the hint and 39 with it.  Bound by memory, also with 8-bit states, since roots, quotients and the cut to E4M3 take few instructions (above; before, 375 us
// for the latter): a step of 218,112,000 bf16 weights with their masters and 32-bit states takes 1,076 us, 5.7 TB/s.
template <int PD, int GD, int BITS, bool MASTER, int TENSORS, bool PASSING> __global__ __launch_bounds__(256) void adamw_kernel(AdamwArgs<TENSORS> a)
{
    const float scale = a.grad_scale ? *a.grad_scale : 1.0f;
    if (!__builtin_isfinite(scale)) return;
    Coefficients c = {a.keep, a.step, a.root, a.dither};
    if (a.coefficients) {
        c.keep = a.coefficients[0];
        c.step = a.coefficients[1];
        c.root = a.coefficients[2];
        c.dither = __float_as_uint(a.coefficients[3]);
    }
    // A lane takes four elements in each half of the tile, so that what a wave loads or stores with an instruction lies together.
    const int k = tensor_of(a.first_tile, blockIdx.x);
    const int64_t n = a.n[k], i = (int64_t)(blockIdx.x - a.first_tile[k]) * kStepTile + 4 * threadIdx.x;
    const int64_t at = (int64_t)a.first_block[k] * kMxBlock + i;  // in the arenas
    const int64_t end = (n + kMxBlock - 1) & ~(int64_t)(kMxBlock - 1); // of its states
    int mine[2];                                                  // elements of the tensor; 0 or less in its padding and behind
    bool live[2];
    float g[8], p[8], m[8], v[8], r[8];
    uint8_t *codes = static_cast<uint8_t *>(a.state);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int64_t e = i + kStepTile / 2 * h, s = at + kStepTile / 2 * h;
        mine[h] = (int)max((int64_t)0, min((int64_t)4, n - e));
        live[h] = e < end;
        if (mine[h] == 4)
            load4<GD, PASSING>(a.grad[k], e, g + 4 * h);
        else
            load_part<GD, 4>(a.grad[k], e, n, g + 4 * h);
        if (!MASTER) {
            if (mine[h] == 4)
                load4<PD, PASSING>(a.param[k], e, p + 4 * h);
            else
                load_part<PD, 4>(a.param[k], e, n, p + 4 * h);
        }
        if (live[h]) {
            if (MASTER) load4<DQ_F32, PASSING>(a.master, s, p + 4 * h);
            if (BITS == 32) {
                load4<DQ_F32, PASSING>(a.state, s, m + 4 * h);
                load4<DQ_F32, PASSING>(a.state, a.total + s, v + 4 * h);
            } else {
                const uint32_t wm = load_word<PASSING>(codes + s), wr = load_word<PASSING>(codes + a.total + s);
                const float um = scale_up(a.scales[s >> 5]), ur = scale_up(a.scales[(a.total + s) >> 5]);
                const f32x2_t m0 = __builtin_amdgcn_cvt_pk_f32_fp8(wm, false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8(wm, true);
                const f32x2_t r0 = __builtin_amdgcn_cvt_pk_f32_fp8(wr, false), r1 = __builtin_amdgcn_cvt_pk_f32_fp8(wr, true);
                m[4 * h] = m0.x * um; m[4 * h + 1] = m0.y * um; m[4 * h + 2] = m1.x * um; m[4 * h + 3] = m1.y * um;
                r[4 * h] = r0.x * ur; r[4 * h + 1] = r0.y * ur; r[4 * h + 2] = r1.x * ur; r[4 * h + 3] = r1.y * ur;
            }
        } else {
#pragma unroll
            for (int j = 4 * h; j < 4 * h + 4; j++) p[j] = m[j] = v[j] = r[j] = 0.0f;
        }
    }
    if (BITS == 8) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = r[j] * r[j];
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float gj = g[j] * scale;
        m[j] = m[j] * a.beta1 + gj * a.rest1;
        v[j] = v[j] * a.beta2 + (gj * gj) * a.rest2;
    }
    roots8(v, r);
    // The quotient only moves the weight: by the reciprocal, good to 1 ulp, unless some divisor of the wave is subnormal, zero or so large that its reciprocal is.
    float q[8];
    uint32_t least = ~0u, most = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float under = r[j] * c.root + a.eps;
        least = min(least, __float_as_uint(under));
        most = max(most, __float_as_uint(under));
        q[j] = m[j] * __builtin_amdgcn_rcpf(under);
    }
    if (DQ_UNLIKELY(__builtin_amdgcn_ballot_w64(least < 0x00800000u || most >= 0x7e800000u) != 0)) {
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = m[j] / (r[j] * c.root + a.eps);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) p[j] = p[j] * c.keep - c.step * q[j];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int64_t e = i + kStepTile / 2 * h, s = at + kStepTile / 2 * h;
        if (mine[h] < 4) { // the padding is zero, whatever it was
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j >= mine[h]) p[4 * h + j] = m[4 * h + j] = v[4 * h + j] = r[4 * h + j] = 0.0f;
        }
        if (BITS == 8) { // (every lane: a block lies in eight of them)
            const uint32_t sm = block_scale<8, 0x600000u>(block_max4(m + 4 * h)), sr = block_scale<8, 0x600000u>(block_max4(r + 4 * h));
            const float dm = scale_down(sm), dr = scale_down(sr);
            const uint32_t seed = (uint32_t)e * kDitherElement + c.dither;
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = m[4 * h + j] * dm;
            const uint32_t wm = cut4(y, seed, 0);
            // A root above zero stays above zero, since a step divides by it: no less than 2^-9, the smallest code.  (Roots above zero are 2^-75 and more.)
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = __builtin_amdgcn_fmed3f(r[4 * h + j] * dr, 0x1p-9f, r[4 * h + j] * 0x1p127f);
            const uint32_t wr = cut4(y, seed, ~0u);
            if (live[h]) {
                store_word<PASSING>(codes + s, wm);
                store_word<PASSING>(codes + a.total + s, wr);
                if ((threadIdx.x & 7) == 0) {
                    a.scales[s >> 5] = (uint8_t)sm;
                    a.scales[(a.total + s) >> 5] = (uint8_t)sr;
                }
            }
        }
        if (live[h]) {
            if (BITS == 32) {
                store4<DQ_F32, PASSING>(a.state, s, m + 4 * h);
                store4<DQ_F32, PASSING>(a.state, a.total + s, v + 4 * h);
            }
            if (MASTER) store4<DQ_F32, PASSING>(a.master, s, p + 4 * h);
        }
        if (mine[h] == 4)
            store4<PD, PASSING>(a.param[k], e, p + 4 * h);
        else
            store_part<PD, 4>(a.param[k], e, mine[h], p + 4 * h);
    }
}

// what a step's kernels take from the step's number, where that number is in device memory: a recorded step counts on
__global__ void adamw_coefficients_kernel(AdamwCount a)
{
    if (a.grad_scale && !__builtin_isfinite(*a.grad_scale)) return;
    const int64_t t = *a.count + 1;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    *a.count = t;
    a.out[0] = (float)(1.0 - lr * a.weight_decay);
    a.out[1] = (float)(lr / (1.0 - pow(a.beta1, (double)t)));
    a.out[2] = (float)(1.0 / sqrt(1.0 - pow(a.beta2, (double)t)));
    a.out[3] = __uint_as_float((uint32_t)t * kDitherStep);
}

hipError_t launch_adamw_coefficients(const AdamwCount &a, hipStream_t stream)
{
    return launch_with(adamw_coefficients_kernel, dim3(1), dim3(1), stream, a);
}

template <int PD, int GD, bool MASTER, int TENSORS> static hipError_t launch_step_with(const AdamwArgs<TENSORS> &a, int bits, bool passing, uint32_t grid, hipStream_t stream)
{
    if (bits == 32)
        return passing ? launch_with(adamw_kernel<PD, GD, 32, MASTER, TENSORS, true>, dim3(grid), dim3(256), stream, a)
                       : launch_with(adamw_kernel<PD, GD, 32, MASTER, TENSORS, false>, dim3(grid), dim3(256), stream, a);
    return passing ? launch_with(adamw_kernel<PD, GD, 8, MASTER, TENSORS, true>, dim3(grid), dim3(256), stream, a)
                   : launch_with(adamw_kernel<PD, GD, 8, MASTER, TENSORS, false>, dim3(grid), dim3(256), stream, a);
}

template <int PD, int GD, int TENSORS> static hipError_t launch_step(const AdamwArgs<TENSORS> &a, int bits, bool passing, uint32_t grid, hipStream_t stream)
{
    if constexpr (PD != DQ_F32) {
        if (a.master) return launch_step_with<PD, GD, true>(a, bits, passing, grid, stream);
    }
    return launch_step_with<PD, GD, false>(a, bits, passing, grid, stream);
}

template <int PD, int TENSORS> static hipError_t launch_step_of(int grad, const AdamwArgs<TENSORS> &a, int bits, bool passing, uint32_t grid, hipStream_t stream)
{
    return grad == DQ_F32 ? launch_step<PD, DQ_F32>(a, bits, passing, grid, stream)
         : grad == DQ_BF16 ? launch_step<PD, DQ_BF16>(a, bits, passing, grid, stream) : launch_step<PD, DQ_F16>(a, bits, passing, grid, stream);
}

// one launch: tensors of the same element types, one after the other, from *next on
template <int TENSORS> static hipError_t launch_tensors(const dq_adamw_t &o, const dq_adamw_tensor_t *tensors, int count, int *next, hipStream_t stream)
{
    AdamwArgs<TENSORS> a;
    a.state = o.state;
    a.scales = o.scales;
    a.master = o.master;
    a.total = o.total;
    a.grad_scale = o.grad_scale;
    a.coefficients = o.coefficients;
    a.beta1 = (float)o.beta1;
    a.rest1 = (float)(1.0 - o.beta1);
    a.beta2 = (float)o.beta2;
    a.rest2 = (float)(1.0 - o.beta2);
    a.eps = (float)o.eps;
    a.keep = a.step = a.root = 0.0f;
    a.dither = 0;
    if (!o.coefficients) {
        a.keep = (float)(1.0 - o.lr * o.weight_decay);
        a.step = (float)(o.lr / (1.0 - pow(o.beta1, (double)o.step)));
        a.root = (float)(1.0 / sqrt(1.0 - pow(o.beta2, (double)o.step)));
        a.dither = (uint32_t)o.step * kDitherStep;
    }
    const int param = tensors[*next].param_dtype, grad = tensors[*next].grad_dtype;
    int take = 0;
    int64_t tiles = 0;
    for (; *next < count && take < TENSORS && tensors[*next].param_dtype == param && tensors[*next].grad_dtype == grad; ++*next) {
        const dq_adamw_tensor_t &x = tensors[*next];
        const int64_t more = (x.n + kStepTile - 1) / kStepTile;
        if (take && tiles + more > kMxMost / kStepTile - 1) break;
        if (more == 0) continue;
        a.first_tile[take] = (uint32_t)tiles;
        a.param[take] = x.param;
        a.grad[take] = x.grad;
        a.n[take] = x.n;
        a.first_block[take++] = (uint32_t)(x.start / kMxBlock);
        tiles += more;
    }
    if (tiles == 0) return hipSuccess;
    for (int j = take; j < TENSORS; j++) a.first_tile[j] = 0xffffffffu;
    const int64_t bytes = (o.master ? 4 : 0) + (param == DQ_F32 ? 4 : 2) + (grad == DQ_F32 ? 4 : 2) + (o.bits == 32 ? 8 : 2);
    const bool passing = tiles * kStepTile * bytes > (int64_t)256 << 20;
    return param == DQ_F32 ? launch_step_of<DQ_F32>(grad, a, o.bits, passing, (uint32_t)tiles, stream)
         : param == DQ_BF16 ? launch_step_of<DQ_BF16>(grad, a, o.bits, passing, (uint32_t)tiles, stream)
                            : launch_step_of<DQ_F16>(grad, a, o.bits, passing, (uint32_t)tiles, stream);
}

hipError_t launch_adamw(const dq_adamw_t &o, const dq_adamw_tensor_t *tensors, int count, hipStream_t stream)
{
    hipError_t e = hipSuccess;
    int next = 0;
    while (next < count && e == hipSuccess)
        e = count - next <= 32 ? launch_tensors<32>(o, tensors, count, &next, stream) : launch_tensors<112>(o, tensors, count, &next, stream);
    return e;
}

} // namespace dq
