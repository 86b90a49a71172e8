// Root-mean-square norm of rows with the residual's addition, an output in 8 bits, and the gradients.
//
//   sum = x + residual (rounded to the residual's type: what is stored is what is normalised)
//   y   = sum * rstd * weight,   rstd = 1 / sqrt(mean(sum^2) + eps)
//   8 bits: scale = max |y| / limit,  q = round(y / scale)
//   backwards, u = gy * weight, v = sum * rstd:  gx = rstd * (u - v * mean(u * v)) + gsum,  gweight = sum over rows of gy * v
//
// Memory bounds it: each tensor once. A row stays in the registers of one to sixteen waves, so that nothing is read twice. [32768, 2048] in
// bf16 with a float32 residual: 146 us forwards (805 MB, 5.5 TB/s), 215 backwards (1074 MB, 5.0 TB/s); [16384, 2049] in bf16 to 8 bits,
// where seven rows in eight begin inside a vector: 57 us from memory (235 MB, 4.1 TB/s), 47 to 53 where the caches hold some of it; 16 rows of
// 2048: 4 us, a launch and one trip to memory. Backwards the vectors lie where they fall: [32768, 2049] takes 452 us with both passes, 2048 365.
#pragma once

#include "ops_common.hpp"

namespace scanscam {

struct NormArgs {
    scanscam_norm a;
    int waves;    // of a row
    bool shifted; // see NormPlan
    float *part;  // backward: [workgroups][channels] sums of gy * v
};

// Elements of a lane's vector: 16 bytes of the widest tensor, so that an instruction of a wave covers one contiguous span of each.
// (With 8 elements beside a float32 residual, every other 16 bytes: 211 us for [32768, 2048] forwards, 145 so.)
template <typename ST, typename RT> constexpr int norm_vec() { return sizeof(ST) == 4 || sizeof(RT) == 4 ? 4 : 8; }

__device__ __forceinline__ float round_to(float v, const float *) { return v; }
template <typename T> __device__ __forceinline__ float round_to(float v, const T *) { return (float)(T)v; }

// The largest absolute value by its bits, which order as the values do and put a NaN above all.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t max_(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Over the wave on DPP row shifts and broadcasts, the last lane's value to all.
template <typename Join> __device__ __forceinline__ float over_wave(float v, Join join)
{
    v = join(v, dpp_move<0x111, 0xf>(0.0f, v));
    v = join(v, dpp_move<0x112, 0xf>(0.0f, v));
    v = join(v, dpp_move<0x114, 0xf>(0.0f, v));
    v = join(v, dpp_move<0x118, 0xf>(0.0f, v));
    v = join(v, dpp_move<0x142, 0xa>(0.0f, v));
    v = join(v, dpp_move<0x143, 0xc>(0.0f, v));
    return read_lane(v, 63);
}
__device__ __forceinline__ float add_(float a, float b) { return a + b; }
__device__ __forceinline__ float top_(float a, float b)
{
    return __builtin_bit_cast(float, max_(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)));
}

// Over the waves of a row, in order; `slots` has one word a wave.
template <typename Join> __device__ __forceinline__ float over_row(float v, int waves, float *slots, Join join)
{
    v = over_wave(v, join);
    if (waves == 1) return v;
    const int wave = threadIdx.x >> 6, first = wave / waves * waves;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slots[wave] = v;
    __syncthreads();
    v = slots[first];
    for (int w = 1; w < waves; w++) v = join(v, slots[first + w]);
    return v;
}

// A lane's vectors of a row: vector j of lane l of the row's wave w covers elements ((j * waves + w) * 64 + l) * VEC - shift on, where
// shift puts vectors of rows that begin inside one on its border. What reaches past the row's start or end is the VEC elements inside
// next to it instead; those that the neighbour has are not the lane's own: they count as nothing in sums and are stored
// twice, the same. So all vectors are whole and are loaded without a branch. Rows of less than VEC elements are loaded one by one.
// EXACT: rows are whole vectors.
template <int VEC, int NV, bool EXACT> struct Place {
    int at[NV];
    int from[EXACT ? 1 : NV], to[EXACT ? 1 : NV];  // its own elements of a vector
    bool there[NV];
    bool any[NV];                                  // of the wave's lanes
    int count;                                     // elements of a vector, below VEC in short rows
    __device__ __forceinline__ Place(int channels, int place, int waves, int shift)
    {
        count = EXACT || channels >= VEC ? VEC : channels;
        shift = EXACT || channels < VEC ? 0 : shift;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (j * waves * 64 + place) * VEC - shift, last = channels - count;
            there[j] = c < channels;
            any[j] = __builtin_amdgcn_readfirstlane((int)there[j]) != 0;
            at[j] = c < last ? c : last;
            if constexpr (!EXACT) {
                at[j] = at[j] < 0 ? 0 : at[j];
                from[j] = c < 0 ? 0 : c - at[j];
                to[j] = !there[j] ? 0 : c < 0 ? VEC + c : VEC;
            }
        }
    }
    __device__ __forceinline__ bool own(int j, int k) const
    {
        if constexpr (EXACT) return there[j];
        else return k >= from[j] && k < to[j];
    }
};

template <typename T, int VEC> struct VecOf {
    Elems<T, VEC> e;
    __device__ __forceinline__ void load(const T *p, int count)
    {
        if (count == VEC) {
            constexpr int PIECE = VEC * sizeof(T) < 16 ? VEC * (int)sizeof(T) : 16;
            using raw_t = typename RawT<PIECE / sizeof(T) * sizeof(T)>::type;
            typedef raw_t raw_unaligned_t __attribute__((aligned(sizeof(T))));
            struct Raw { raw_t r[VEC * sizeof(T) / PIECE]; } raw;
#pragma unroll
            for (int i = 0; i < (int)(VEC * sizeof(T) / PIECE); i++) raw.r[i] = reinterpret_cast<const raw_unaligned_t *>(p)[i];
            e = __builtin_bit_cast(decltype(e), raw);
        } else {
            for (int k = 0; k < VEC; k++) e.e[k] = k < count ? p[k] : (T)0.0f;
        }
    }
    __device__ __forceinline__ float operator[](int k) const { return (float)e.e[k]; }
};

// A vector of the weights, of whatever type: asked for as it is stored, taken apart where it is used.
template <int VEC> struct Weights {
    uint32_t raw[VEC];
    __device__ __forceinline__ void load(const scanscam_param &w, int64_t at, int count)
    {
        if (w.dtype == SCANSCAM_F32) {
            VecOf<float, VEC> v;
            v.load(static_cast<const float *>(w.p) + at, count);
            __builtin_memcpy(raw, &v, sizeof(v));
        } else {
            VecOf<_Float16, VEC> v;  // (either of the 16-bit types)
            v.load(static_cast<const _Float16 *>(w.p) + at, count);
            __builtin_memcpy(raw, &v, sizeof(v));
        }
    }
    __device__ __forceinline__ void get(int dtype, float (&f)[VEC]) const
    {
        if (dtype == SCANSCAM_F32) {
#pragma unroll
            for (int k = 0; k < VEC; k++) f[k] = __builtin_bit_cast(float, raw[k]);
        } else if (dtype == SCANSCAM_BF16) {
#pragma unroll
            for (int k = 0; k < VEC; k++) f[k] = __builtin_bit_cast(float, k % 2 == 0 ? raw[k / 2] << 16 : raw[k / 2] & 0xffff0000u);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; k++) f[k] = (float)__builtin_bit_cast(_Float16, (uint16_t)(k % 2 == 0 ? raw[k / 2] & 0xffffu : raw[k / 2] >> 16));
        }
    }
};

// Waves a SIMD at least: rows of 6 vectors of 8 that begin inside one take 132 registers and three waves if they may; in the 128 of four, three
// of them spilled, [16384, 2049] to 8 bits takes 53 us instead of 56 (whole vectors, [16384, 2048]: 47).
template <typename ST, typename RT, int NV, bool EXACT> constexpr int norm_fwd_least() { return !EXACT && NV == 6 && norm_vec<ST, RT>() == 8 ? 4 : 1; }

// A workgroup holds 4 waves, or the row's. RT: the residual's type (the activations' where there is none).
template <typename ST, typename RT, int NV, int THREADS, bool EXACT>
__global__ __launch_bounds__(THREADS, (norm_fwd_least<ST, RT, NV, EXACT>())) void norm_fwd_kernel(NormArgs args)
{
    constexpr int VEC = norm_vec<ST, RT>();
    const scanscam_norm &a = args.a;
    const int waves = args.waves;
    __shared__ float slots[16];
    const int wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / 64 / waves) + wave / waves;
    const bool there = row < a.rows;
    const int64_t r = there ? row : a.rows - 1, D = a.channels;
    const int place = (wave % waves) * 64 + (threadIdx.x & 63);
    const Place<VEC, NV, EXACT> at((int)D, place, waves, args.shifted ? (int)(r * D % VEC) : 0);
    const bool added = a.residual != nullptr;
    VecOf<ST, VEC> x[NV];
    VecOf<RT, VEC> more[NV];
#pragma unroll
    for (int j = 0; j < NV; j++)
        if (at.any[j]) x[j].load(static_cast<const ST *>(a.x) + r * a.x_stride + at.at[j], at.count);
    if (added) {
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (at.any[j]) more[j].load(static_cast<const RT *>(a.residual) + r * a.residual_stride + at.at[j], at.count);
    }
    Weights<VEC> weights[NV];
#pragma unroll
    for (int j = 0; j < NV; j++)
        if (at.any[j]) weights[j].load(a.weight, at.at[j], at.count);
    float v[NV][VEC], square = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if (!at.any[j]) continue;
#pragma unroll
        for (int k = 0; k < VEC; k++) v[j][k] = x[j][k];
        if (added) {
#pragma unroll
            for (int k = 0; k < VEC; k++) v[j][k] = round_to(v[j][k] + more[j][k], static_cast<const RT *>(nullptr));
            if (there && at.there[j]) store_some(static_cast<RT *>(a.sum) + r * D + at.at[j], at.count, v[j]);
        }
#pragma unroll
        for (int k = 0; k < VEC; k++) square = __builtin_fmaf(at.own(j, k) ? v[j][k] : 0.0f, v[j][k], square);
    }
    square = over_row(square, waves, slots, add_);
    const float rstd = 1.0f / __builtin_sqrtf(square / (float)D + a.eps);
    if (there && a.rstd != nullptr && place == 0) a.rstd[r] = rstd;
    const bool eight = a.out_dtype == SCANSCAM_I8 || a.out_dtype == SCANSCAM_F8;
    const float factor = eight ? 1.0f : rstd;  // (in 8 bits rstd is a factor of the scale alone: one rounding less on the way to y / scale)
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if (!at.any[j]) continue;
        float w[VEC];
        weights[j].get(a.weight.dtype, w);
#pragma unroll
        for (int k = 0; k < VEC; k++) {
            v[j][k] = v[j][k] * factor * w[k];
            top = max_(top, k < at.count ? abs_bits(v[j][k]) : 0u);
        }
        if (!eight && there && at.there[j]) store_some(static_cast<ST *>(a.y) + r * D + at.at[j], at.count, v[j]);
    }
    if (!eight) return;
    // y / scale = sum w limit / max |sum w|. Rows of tiny values are first raised, so that limit / max stays finite. A row that holds a
    // NaN or an infinity has no scale: all of it is NaN (integers: 0). Squares that overflow make rstd, and so y, 0.
    const float limit = a.out_dtype == SCANSCAM_I8 ? 127.0f : 448.0f;
    float most = over_row(__builtin_bit_cast(float, top), waves, slots, top_);
    const bool lost = !(most < __builtin_inff());
    if (rstd == 0.0f && !lost) most = 0.0f;
    const float raise = most < 0x1p-80f ? 0x1p100f : 1.0f, unit = most == 0.0f ? 0.0f : limit / (most * raise);
    if (there && place == 0) a.scale[r] = lost ? __builtin_nanf("") : most == 0.0f ? 1.0f : most * rstd / limit;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if (!at.there[j] || !there) continue;
        float q[VEC];
#pragma unroll
        for (int k = 0; k < VEC; k++) q[k] = __builtin_amdgcn_fmed3f(v[j][k] * raise * unit, -limit, limit);
        uint32_t packed[VEC / 4];
        if (a.out_dtype == SCANSCAM_F8) {
#pragma unroll
            for (int h = 0; h < VEC / 4; h++) {
                int p = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], 0, false);
                packed[h] = lost ? 0x7f7f7f7fu : (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], p, true);
            }
        } else {
#pragma unroll
            for (int h = 0; h < VEC / 4; h++) {
                uint32_t p = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) p |= ((uint32_t)(int)__builtin_rintf(q[4 * h + k]) & 0xffu) << (8 * k);
                packed[h] = lost ? 0u : p;
            }
        }
        uint8_t *to = static_cast<uint8_t *>(a.y) + r * D + at.at[j];
        if (at.count == VEC) {
            typedef typename RawT<VEC>::type bytes_t __attribute__((aligned(1)));
            struct Packed { uint32_t p[VEC / 4]; } all;
#pragma unroll
            for (int h = 0; h < VEC / 4; h++) all.p[h] = packed[h];
            *reinterpret_cast<bytes_t *>(to) = __builtin_bit_cast(typename RawT<VEC>::type, all);
        } else {
            for (int k = 0; k < at.count; k++) to[k] = (uint8_t)(packed[k / 4] >> (8 * (k % 4)));
        }
    }
}

// Every group of `waves` waves takes rows g, g + groups, ...; the sums of gy * v over its rows stay in registers, are added up over
// the workgroup's groups in order, and go out as one part a workgroup. All of a row is asked for before anything is waited for.
template <typename ST, typename RT, int NV, int THREADS, bool EXACT>
__global__ __launch_bounds__(THREADS) void norm_bwd_kernel(NormArgs args)
{
    constexpr int VEC = norm_vec<ST, RT>();
    const scanscam_norm &a = args.a;
    const int waves = args.waves;
    __shared__ float slots[16];
    extern __shared__ float part[];  // [channels] where a workgroup holds several rows at a time
    const int wave = threadIdx.x >> 6;
    const int here = blockDim.x / 64 / waves, mine = wave / waves;
    const int place = (wave % waves) * 64 + (threadIdx.x & 63);
    const int64_t D = a.channels, groups = (int64_t)gridDim.x * here;
    const Place<VEC, NV, EXACT> at((int)D, place, waves, 0);  // (the sums over rows need the same columns of every row)
    const bool added = a.residual != nullptr, onto = a.gsum != nullptr;
    const RT *sums = static_cast<const RT *>(added ? a.sum : a.x);
    const int64_t pitch = added ? D : a.x_stride;
    float gw[NV][VEC] = {};
    Weights<VEC> weights[NV];
#pragma unroll
    for (int j = 0; j < NV; j++)
        if (at.any[j]) weights[j].load(a.weight, at.at[j], at.count);
    // (every group of a workgroup goes through the loop as often as the others: it has barriers where a row has several waves)
    for (int64_t base = (int64_t)blockIdx.x * here; base < a.rows; base += groups) {
        const bool there = base + mine < a.rows;
        const int64_t r = there ? base + mine : a.rows - 1;
        VecOf<ST, VEC> gy[NV];
        VecOf<RT, VEC> sum[NV], gsum[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (!at.any[j]) continue;
            gy[j].load(static_cast<const ST *>(a.gy) + r * D + at.at[j], at.count);
            sum[j].load(sums + r * pitch + at.at[j], at.count);
        }
        if (onto) {
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (at.any[j]) gsum[j].load(static_cast<const RT *>(a.gsum) + r * D + at.at[j], at.count);
        }
        const float rstd = a.rstd[r], mine_of_it = there ? rstd : 0.0f;
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (!at.any[j]) continue;
            float w[VEC];
            weights[j].get(a.weight.dtype, w);
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                const float gv = at.own(j, k) ? gy[j][k] * sum[j][k] : 0.0f;
                gw[j][k] = __builtin_fmaf(gv, mine_of_it, gw[j][k]);
                dot = __builtin_fmaf(gv, w[k], dot);
            }
        }
        // (u . v / channels, v = sum * rstd; the rstd of v comes in once here and once below)
        const float mean = over_row(dot, waves, slots, add_) * rstd / (float)D;
        if (!there) continue;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (!at.there[j]) continue;
            float g[VEC], w[VEC];
            weights[j].get(a.weight.dtype, w);
#pragma unroll
            for (int k = 0; k < VEC; k++) g[k] = rstd * (gy[j][k] * w[k] - sum[j][k] * rstd * mean);
            if (onto) {
#pragma unroll
                for (int k = 0; k < VEC; k++) g[k] += gsum[j][k];
            }
            store_some(static_cast<ST *>(a.gx) + r * D + at.at[j], at.count, g);
            if (a.gresidual != nullptr) store_some(static_cast<RT *>(a.gresidual) + r * D + at.at[j], at.count, g);
        }
    }
    for (int g = 0; g < here; g++) {
        if (g == mine) {
#pragma unroll
            for (int j = 0; j < NV; j++) {
#pragma unroll
                for (int k = 0; k < VEC; k++)
                    if (at.own(j, k) && k < at.count) {
                        if (here == 1) args.part[(int64_t)blockIdx.x * D + at.at[j] + k] = gw[j][k];
                        else part[at.at[j] + k] = g == 0 ? gw[j][k] : part[at.at[j] + k] + gw[j][k];
                    }
            }
        }
        __syncthreads();
    }
    if (here == 1) return;
    for (int64_t c = threadIdx.x; c < D; c += blockDim.x) args.part[(int64_t)blockIdx.x * D + c] = part[c];
}

struct NormPlan {
    int waves, nv, groups;  // waves a row, vectors a lane, rows of a workgroup at a time
    bool shifted;           // the lanes have a vector more than the row, so that vectors may lie on their borders
};

// One per storage type of the activations, in a file of its own.
template <typename ST> hipError_t launch_norm(bool back, const NormPlan &plan, unsigned grid, size_t lds, hipStream_t stream, const NormArgs &args);

template <typename ST, typename RT, int THREADS, bool EXACT> void (*norm_kernel(bool back, int nv))(NormArgs)
{
    constexpr int MOST = norm_vec<ST, RT>() == 4 ? 8 : 6;
    return nv == 1   ? (back ? norm_bwd_kernel<ST, RT, 1, THREADS, EXACT> : norm_fwd_kernel<ST, RT, 1, THREADS, EXACT>)
           : nv == 2 ? (back ? norm_bwd_kernel<ST, RT, 2, THREADS, EXACT> : norm_fwd_kernel<ST, RT, 2, THREADS, EXACT>)
           : nv == 4 ? (back ? norm_bwd_kernel<ST, RT, 4, THREADS, EXACT> : norm_fwd_kernel<ST, RT, 4, THREADS, EXACT>)
                     : (back ? norm_bwd_kernel<ST, RT, MOST, THREADS, EXACT> : norm_fwd_kernel<ST, RT, MOST, THREADS, EXACT>);
}
// (workgroups of 256 threads may use more registers than the larger ones of long rows)
template <typename ST, typename RT> hipError_t launch_norm_with(bool back, const NormPlan &plan, unsigned grid, size_t lds, hipStream_t stream, const NormArgs &args)
{
    const int threads = 64 * plan.waves * plan.groups;
    const bool exact = args.a.channels % norm_vec<ST, RT>() == 0;
    auto kernel = threads <= 256 ? (exact ? norm_kernel<ST, RT, 256, true>(back, plan.nv) : norm_kernel<ST, RT, 256, false>(back, plan.nv))
                                 : (exact ? norm_kernel<ST, RT, 1024, true>(back, plan.nv) : norm_kernel<ST, RT, 1024, false>(back, plan.nv));
    return launch_op(kernel, dim3(grid), dim3((unsigned)threads), lds, stream, args);
}
#define SCANSCAM_DEFINE_NORM_LAUNCH(ST)                                                                                                                             \
    template <> hipError_t launch_norm<ST>(bool back, const NormPlan &plan, unsigned grid, size_t lds, hipStream_t stream, const NormArgs &args)                    \
    {                                                                                                                                                               \
        switch (args.a.residual != nullptr ? args.a.residual_dtype : args.a.dtype) {                                                                                \
        case SCANSCAM_F32: return launch_norm_with<ST, float>(back, plan, grid, lds, stream, args);                                                                 \
        case SCANSCAM_BF16: return launch_norm_with<ST, __bf16>(back, plan, grid, lds, stream, args);                                                               \
        default: return launch_norm_with<ST, _Float16>(back, plan, grid, lds, stream, args);                                                                        \
        }                                                                                                                                                           \
    }

}  // namespace scanscam
