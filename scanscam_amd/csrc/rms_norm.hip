// Root-mean-square norm of rows with the residual's addition, an output in 8 bits, and the gradients.
//
//   sum = x + residual (rounded to the residual's type: what is stored is what is normalised)
//   y   = sum * rstd * weight,   rstd = 1 / sqrt(mean(sum^2) + eps)
//   8 bits: scale = max |y| / limit,  q = round(y / scale)
//   backwards, u = gy * weight, v = sum * rstd:  gx = rstd * (u - v * mean(u * v)) + gsum,  gweight = sum over rows of gy * v
//
// Memory bounds it: each tensor once. A row stays in the registers of one to sixteen waves, so that nothing is read twice.
#include "ops_common.hpp"

namespace scanscam {

struct NormArgs {
    scanscam_norm a;
    float *part;  // backward: [workgroups][channels] sums of gy * v
};

constexpr int kNormVec = 8;  // elements of a lane's vector

__device__ __forceinline__ void load_any(const void *p, int dtype, int64_t i, int count, float (&f)[kNormVec])
{
    if (dtype == SCANSCAM_F32) load_part(static_cast<const float *>(p) + i, count, f);
    else if (dtype == SCANSCAM_BF16) load_part(static_cast<const __bf16 *>(p) + i, count, f);
    else load_part(static_cast<const _Float16 *>(p) + i, count, f);
}

__device__ __forceinline__ void store_any(void *p, int dtype, int64_t i, int count, const float (&f)[kNormVec])
{
    if (dtype == SCANSCAM_F32) store_some(static_cast<float *>(p) + i, count, f);
    else if (dtype == SCANSCAM_BF16) store_some(static_cast<__bf16 *>(p) + i, count, f);
    else store_some(static_cast<_Float16 *>(p) + i, count, f);
}

__device__ __forceinline__ float round_to(float v, int dtype)
{
    return dtype == SCANSCAM_F32 ? v : dtype == SCANSCAM_BF16 ? (float)(__bf16)v : (float)(_Float16)v;
}

// The largest absolute value by its bits, which order as the values do and put a NaN above all.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t max_(uint32_t a, uint32_t b) { return a > b ? a : b; }

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v = max_(v, (uint32_t)__shfl_xor((int)v, m));
    return v;
}

// The sum over the waves of a row; `slots` has one word a wave. Every wave adds in the same order.
template <typename T, typename Join>
__device__ __forceinline__ T across_waves(T v, int waves, T *slots, Join join)
{
    if (waves == 1) return v;
    const int wave = threadIdx.x >> 6, first = wave / waves * waves;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slots[wave] = v;
    __syncthreads();
    T all = slots[first];
    for (int w = 1; w < waves; w++) all = join(all, slots[first + w]);
    return all;
}

// `waves` waves a row, NV vectors a lane: vector j of lane l of the row's wave w covers elements ((j * waves + w) * 64 + l) * 8 on.
// A workgroup holds 4 waves, or the row's.
template <int NV>
__global__ __launch_bounds__(1024) void norm_fwd_kernel(NormArgs args, int waves)
{
    const scanscam_norm &a = args.a;
    __shared__ float sums[16];
    __shared__ uint32_t tops[16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / 64 / waves) + wave / waves;
    const bool there = row < a.rows;
    const int64_t r = there ? row : a.rows - 1;
    const int place = (wave % waves) * 64 + lane;
    const int64_t D = a.channels;
    float v[NV][kNormVec];
    float square = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int64_t c = ((int64_t)j * waves * 64 + place) * kNormVec;
        const int count = (int)clamp_(D - c, 0, kNormVec);
#pragma unroll
        for (int k = 0; k < kNormVec; k++) v[j][k] = 0.0f;
        if (count > 0) load_any(a.x, a.dtype, r * a.x_stride + c, count, v[j]);
        if (a.residual != nullptr && count > 0) {
            float o[kNormVec];
            load_any(a.residual, a.residual_dtype, r * a.residual_stride + c, count, o);
#pragma unroll
            for (int k = 0; k < kNormVec; k++) v[j][k] = round_to(v[j][k] + o[k], a.residual_dtype);
            if (there) store_any(a.sum, a.residual_dtype, r * D + c, count, v[j]);
        }
#pragma unroll
        for (int k = 0; k < kNormVec; k++) square = __builtin_fmaf(v[j][k], v[j][k], square);
    }
    square = across_waves(wave_sum(square), waves, sums, [](float p, float q) { return p + q; });
    const float rstd = 1.0f / __builtin_sqrtf(square / (float)D + a.eps);
    if (there && a.rstd != nullptr && place == 0) a.rstd[r] = rstd;
    const bool eight = a.out_dtype == SCANSCAM_I8 || a.out_dtype == SCANSCAM_F8;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int64_t c = ((int64_t)j * waves * 64 + place) * kNormVec;
        const int count = (int)clamp_(D - c, 0, kNormVec);
        if (count <= 0) continue;
        float w[kNormVec];
        load_any(a.weight.p, a.weight.dtype, c, count, w);
#pragma unroll
        for (int k = 0; k < kNormVec; k++) {
            // (in 8 bits rstd is a factor of the scale alone: one rounding less on the way to y / scale)
            v[j][k] = eight ? v[j][k] * w[k] : v[j][k] * rstd * w[k];
            top = max_(top, k < count ? abs_bits(v[j][k]) : 0u);
        }
        if (!eight && there) store_any(a.y, a.dtype, r * D + c, count, v[j]);
    }
    if (!eight) return;
    const float limit = a.out_dtype == SCANSCAM_I8 ? 127.0f : 448.0f;
    const float most = __builtin_bit_cast(float, across_waves(wave_max(top), waves, tops, max_));
    // y / scale = sum w limit / max |sum w|. Rows of tiny values are first raised, so that limit / max stays finite; where the row has a
    // NaN or an infinity, rstd or a product of it is NaN, and so is the scale.
    const float raise = most < 0x1p-80f ? 0x1p100f : 1.0f;
    const float factor = most == 0.0f ? 1.0f : limit / (most * raise);
    if (there && place == 0) a.scale[r] = most == 0.0f ? 1.0f : most * rstd / limit;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int64_t c = ((int64_t)j * waves * 64 + place) * kNormVec;
        const int count = (int)clamp_(D - c, 0, kNormVec);
        if (count <= 0 || !there) continue;
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int k = 0; k < kNormVec; k++) {
            const float q = v[j][k] * raise * factor;
            uint32_t byte;
            if (a.out_dtype == SCANSCAM_I8) {
                byte = (uint32_t)(int)__builtin_rintf(__builtin_fminf(__builtin_fmaxf(q, -127.0f), 127.0f)) & 0xffu;
            } else {
                const float f = q != q ? q : __builtin_fminf(__builtin_fmaxf(q, -448.0f), 448.0f);
                byte = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f, f, 0, false) & 0xffu;
            }
            if (k < 4) lo |= byte << (8 * k);
            else hi |= byte << (8 * k - 32);
        }
        uint8_t *to = static_cast<uint8_t *>(a.y) + r * D + c;
        if (count == kNormVec) {
            typedef uint32_t two_t __attribute__((ext_vector_type(2), aligned(1)));
            *reinterpret_cast<two_t *>(to) = two_t{lo, hi};
        } else {
#pragma unroll
            for (int k = 0; k < kNormVec; k++)
                if (k < count) to[k] = (uint8_t)((k < 4 ? lo >> (8 * k) : hi >> (8 * k - 32)) & 0xffu);
        }
    }
}

// Every group of `waves` waves takes rows g, g + groups, ...; the sums of gy * v over its rows stay in registers, are added up over
// the workgroup's groups in order, and go out as one part a workgroup.
template <int NV>
__global__ __launch_bounds__(1024) void norm_bwd_kernel(NormArgs args, int waves)
{
    const scanscam_norm &a = args.a;
    __shared__ float sums[16];
    extern __shared__ float part[];  // [channels] where a workgroup holds several rows at a time
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int here = blockDim.x / 64 / waves, mine = wave / waves;
    const int place = (wave % waves) * 64 + lane;
    const int64_t D = a.channels, groups = (int64_t)gridDim.x * here;
    const int sum_dtype = a.residual != nullptr ? a.residual_dtype : a.dtype;
    float gw[NV][kNormVec] = {};
    // (every group of a workgroup goes through the loop as often as the others: it has barriers where a row has several waves)
    for (int64_t base = (int64_t)blockIdx.x * here; base < a.rows; base += groups) {
        const bool there = base + mine < a.rows;
        const int64_t r = there ? base + mine : a.rows - 1;
        const float rstd = a.rstd[r];
        float u[NV][kNormVec], v[NV][kNormVec];
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t c = ((int64_t)j * waves * 64 + place) * kNormVec;
            const int count = (int)clamp_(D - c, 0, kNormVec);
            float w[kNormVec];
#pragma unroll
            for (int k = 0; k < kNormVec; k++) u[j][k] = v[j][k] = w[k] = 0.0f;
            if (count > 0) {
                load_any(a.gy, a.dtype, r * D + c, count, u[j]);
                load_any(a.residual != nullptr ? a.sum : a.x, sum_dtype, r * (a.residual != nullptr ? D : a.x_stride) + c, count, v[j]);
                load_any(a.weight.p, a.weight.dtype, c, count, w);
            }
#pragma unroll
            for (int k = 0; k < kNormVec; k++) {
                v[j][k] *= rstd;
                if (there) gw[j][k] = __builtin_fmaf(u[j][k], v[j][k], gw[j][k]);
                u[j][k] *= w[k];
                dot = __builtin_fmaf(u[j][k], v[j][k], dot);
            }
        }
        const float mean = across_waves(wave_sum(dot), waves, sums, [](float p, float q) { return p + q; }) / (float)D;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t c = ((int64_t)j * waves * 64 + place) * kNormVec;
            const int count = (int)clamp_(D - c, 0, kNormVec);
            if (count <= 0 || !there) continue;
            float g[kNormVec];
#pragma unroll
            for (int k = 0; k < kNormVec; k++) g[k] = 0.0f;
            if (a.gsum != nullptr) load_any(a.gsum, a.residual_dtype, r * D + c, count, g);
#pragma unroll
            for (int k = 0; k < kNormVec; k++) g[k] = __builtin_fmaf(rstd, u[j][k] - v[j][k] * mean, g[k]);
            store_any(a.gx, a.dtype, r * D + c, count, g);
            if (a.gresidual != nullptr) store_any(a.gresidual, a.residual_dtype, r * D + c, count, g);
        }
    }
    if (here == 1) {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t c = ((int64_t)j * waves * 64 + place) * kNormVec;
            if (c < D) store_some(args.part + (int64_t)blockIdx.x * D + c, (int)clamp_(D - c, 0, kNormVec), gw[j]);
        }
        return;
    }
    for (int g = 0; g < here; g++) {
        if (g == mine) {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int64_t c = ((int64_t)j * waves * 64 + place) * kNormVec;
#pragma unroll
                for (int k = 0; k < kNormVec; k++)
                    if (c + k < D) part[c + k] = g == 0 ? gw[j][k] : part[c + k] + gw[j][k];
            }
        }
        __syncthreads();
    }
    for (int64_t c = threadIdx.x; c < D; c += blockDim.x) args.part[(int64_t)blockIdx.x * D + c] = part[c];
}

__global__ __launch_bounds__(1024) void column_sum_kernel(ColumnSum a)
{
    __shared__ float sums[16][64];
    const int col = threadIdx.x & 63, slice = threadIdx.x >> 6;
    const int64_t m = (int64_t)blockIdx.x * 64 + col;
    float s = 0.0f;
    if (m < a.columns) {
#pragma unroll 8
        for (int64_t p = slice; p < a.parts; p += 16) s += a.in[p * a.pitch + m];
    }
    sums[slice][col] = s;
    __syncthreads();
    if (slice != 0 || m >= a.columns) return;
    for (int i = 1; i < 16; i++) s += sums[i][col];
    a.out[m] = s;
}

}  // namespace scanscam

namespace {

using namespace scanscam;

struct NormPlan {
    int waves, nv, groups;  // waves a row, vectors a lane, rows of a workgroup at a time
};

// A wave a row while its lanes need at most 4 vectors (2048 channels), more waves then; 32768 channels take 16 waves of 4.
NormPlan norm_plan(int64_t channels)
{
    const int64_t vectors = ceil_div(channels, 64 * kNormVec);
    int waves = 1;
    while (waves < 16 && vectors > 4 * waves) waves *= 2;
    int nv = 1;
    while (nv * waves < vectors) nv *= 2;
    return {waves, nv, waves >= 4 ? 1 : 4 / waves};
}

constexpr int64_t kNormMostChannels = 32768;

int64_t norm_bwd_workgroups(const scanscam_norm &a, const NormPlan &p)
{
    const int64_t all = ceil_div(a.rows, p.groups);
    return all < 512 ? all : 512;
}

int check_norm(const scanscam_norm *a)
{
    if (a == nullptr || a->rows < 0 || a->channels < 0 || a->x_stride < 0 || a->residual_stride < 0) return SCANSCAM_EINVAL;
    if (a->rows >= kMostTokens || a->channels > kNormMostChannels) return SCANSCAM_EINVAL;
    const int size = activation_size(a->dtype);
    if (size == 0 || (a->residual != nullptr && activation_size(a->residual_dtype) == 0)) return SCANSCAM_EDTYPE;
    if (a->rows == 0 || a->channels == 0) return SCANSCAM_OK;
    SCANSCAM_CHECK(check_param(a->weight, true));
    if (a->x == nullptr) return SCANSCAM_EINVAL;
    if (misaligned(a->x, (size_t)size)) return SCANSCAM_EALIGN;
    if (a->residual != nullptr && misaligned(a->residual, (size_t)activation_size(a->residual_dtype))) return SCANSCAM_EALIGN;
    if ((a->residual != nullptr) != (a->sum != nullptr)) return SCANSCAM_EINVAL;
    if (a->sum != nullptr && misaligned(a->sum, (size_t)activation_size(a->residual_dtype))) return SCANSCAM_EALIGN;
    return SCANSCAM_OK;
}

template <typename K1, typename K2, typename K4>
hipError_t launch_norm(K1 k1, K2 k2, K4 k4, const NormPlan &plan, unsigned grid, size_t lds, hipStream_t stream, NormArgs args)
{
    auto kernel = plan.nv == 1 ? k1 : plan.nv == 2 ? k2 : k4;
    int waves = plan.waves;
    void *params[] = {&args, &waves};
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3(grid), dim3(64 * plan.waves * plan.groups), params, lds, stream);
}

}  // namespace

extern "C" {

int scanscam_norm_fwd(const scanscam_norm *a, void *stream)
{
    SCANSCAM_CHECK(check_norm(a));
    const bool eight = a->out_dtype == SCANSCAM_I8 || a->out_dtype == SCANSCAM_F8;
    if (!eight && a->out_dtype != a->dtype) return SCANSCAM_EDTYPE;
    if (a->rows == 0 || a->channels == 0) return SCANSCAM_OK;
    if (a->y == nullptr || (eight && a->scale == nullptr)) return SCANSCAM_EINVAL;
    if (!eight && misaligned(a->y, (size_t)activation_size(a->dtype))) return SCANSCAM_EALIGN;
    const NormPlan plan = norm_plan(a->channels);
    const hipError_t err = launch_norm(norm_fwd_kernel<1>, norm_fwd_kernel<2>, norm_fwd_kernel<4>, plan,
                                       (unsigned)ceil_div(a->rows, plan.groups), 0, static_cast<hipStream_t>(stream), NormArgs{*a, nullptr});
    return err == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
}

size_t scanscam_norm_workspace_bytes(const scanscam_norm *a)
{
    if (a == nullptr || a->rows <= 0 || a->channels <= 0 || a->channels > kNormMostChannels) return 0;
    return (size_t)(norm_bwd_workgroups(*a, norm_plan(a->channels)) * a->channels) * sizeof(float);
}

int scanscam_norm_bwd(const scanscam_norm *a, void *stream)
{
    SCANSCAM_CHECK(check_norm(a));
    if (a->channels == 0) return SCANSCAM_OK;
    if (a->gweight == nullptr) return SCANSCAM_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a->rows == 0) return column_sum(nullptr, a->gweight, 0, 0, a->channels, s) == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
    if (a->gy == nullptr || a->gx == nullptr || a->rstd == nullptr || (a->gsum != nullptr && a->residual == nullptr) ||
        (a->gresidual != nullptr && a->residual == nullptr))
        return SCANSCAM_EINVAL;
    const size_t size = (size_t)activation_size(a->dtype);
    if (misaligned(a->gy, size) || misaligned(a->gx, size)) return SCANSCAM_EALIGN;
    if (a->workspace == nullptr || a->workspace_bytes < scanscam_norm_workspace_bytes(a)) return SCANSCAM_EWORKSPACE;
    if (misaligned(a->workspace, 16)) return SCANSCAM_EALIGN;
    const NormPlan plan = norm_plan(a->channels);
    const int64_t grid = norm_bwd_workgroups(*a, plan);
    float *part = static_cast<float *>(a->workspace);
    hipError_t err = launch_norm(norm_bwd_kernel<1>, norm_bwd_kernel<2>, norm_bwd_kernel<4>, plan, (unsigned)grid,
                                 plan.groups > 1 ? (size_t)a->channels * sizeof(float) : 0, s, NormArgs{*a, part});
    if (err == hipSuccess) err = column_sum(part, a->gweight, grid, a->channels, a->channels, s);
    return err == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
}

}  // extern "C"
