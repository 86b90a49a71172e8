// C ABI of the root-mean-square norm (declared in include/scanscam_ops.h): argument checks, launch shapes, launches; and the column sums
// that other operators use as well.
#include "rms_norm_kernels.hpp"

namespace scanscam {

__global__ __launch_bounds__(1024) void column_sum_kernel(ColumnSum a)
{
    __shared__ float sums[16][64];
    const int col = threadIdx.x & 63, slice = threadIdx.x >> 6;
    const int64_t column = (int64_t)blockIdx.x * 64 + col, all = a.columns[0] + a.columns[1] + a.columns[2];
    const int64_t group = a.first + blockIdx.y, begin = group * a.each, parts = a.each > 0 && a.each < a.parts - begin ? a.each : a.parts - begin;
    float *in = a.in + begin * a.pitch;
    float s = 0.0f;
    if (column < all) {
#pragma unroll 8
        for (int64_t p = slice; p < parts; p += 16) s += in[p * a.pitch + column];
    }
    sums[slice][col] = s;
    __syncthreads();
    if (slice != 0 || column >= all) return;
    for (int i = 1; i < 16; i++) s += sums[i][col];
    if (a.each > 0) {  // (a group's columns are one workgroup's alone, and all of it has been read)
        in[column] = s;
        return;
    }
    const int which = column < a.columns[0] ? 0 : column < a.columns[0] + a.columns[1] ? 1 : 2;
    const int64_t m = column - (which > 0 ? a.columns[0] : 0) - (which > 1 ? a.columns[1] : 0);
    float *out = which == 0 ? a.out[0] : which == 1 ? a.out[1] : a.out[2];
    if (out != nullptr) out[m] = s;
}

// The scales of rows without channels.
struct Ones {
    float *to;
    int64_t count;
};
__global__ __launch_bounds__(256) void ones_kernel(Ones a)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < a.count) a.to[i] = 1.0f;
}

}  // namespace scanscam

namespace {

using namespace scanscam;

// A wave a row while its lanes need at most 6 vectors of 16-bit types or 8 beside float32 (some 3000 and 2000 channels), more waves
// then; 32768 channels take 16. Where there are few rows, a row's waves are as many as have a vector for each lane. Rows
// that begin inside a vector have one more.
NormPlan norm_plan(const scanscam_norm &a)
{
    const bool wide = a.dtype == SCANSCAM_F32 || (a.residual != nullptr && a.residual_dtype == SCANSCAM_F32);
    const int vec = wide ? 4 : 8, most = wide ? 8 : 6;
    int64_t vectors = ceil_div(a.channels / vec + (a.channels % vec != 0 ? 2 : 0), 64);
    vectors = vectors < 16 * (32768 / vec / 64 / 16) ? vectors : 16 * (32768 / vec / 64 / 16);
    int waves = 1;
    while (waves < 16 && (vectors > most * waves || (vectors > waves && a.rows * waves < 1024))) waves *= 2;
    int nv = 1;
    while (nv * waves < vectors) nv = nv == 4 ? most : 2 * nv;
    return {waves, nv, waves >= 4 ? 1 : 4 / waves, (int64_t)waves * nv * 64 * vec >= a.channels + vec};
}

constexpr int64_t kNormMostChannels = 32768;

constexpr int64_t kNormMostParts = 1024;
int64_t norm_bwd_workgroups(const scanscam_norm &a, const NormPlan &p)
{
    const int64_t all = ceil_div(a.rows, p.groups);
    return all < kNormMostParts ? all : kNormMostParts;
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

// A forward call's arguments for `count` of its rows.
scanscam_norm rows_from(const scanscam_norm &a, int64_t row, int64_t count)
{
    const auto moved = [](auto *p, int64_t bytes) { return p == nullptr ? p : (decltype(p))((const char *)p + bytes); };
    const int size = activation_size(a.dtype), residual = activation_size(a.residual_dtype), out = activation_size(a.out_dtype);
    scanscam_norm now = a;
    now.rows = count;
    now.x = moved(a.x, row * a.x_stride * size);
    now.residual = moved(a.residual, row * a.residual_stride * residual);
    now.y = moved(a.y, row * a.channels * (out > 0 ? out : 1));
    now.sum = moved(a.sum, row * a.channels * residual);
    now.rstd = moved(a.rstd, row * (int64_t)sizeof(float));
    now.scale = moved(a.scale, row * (int64_t)sizeof(float));
    return now;
}

hipError_t run_norm(bool back, const NormPlan &plan, unsigned grid, size_t lds, hipStream_t stream, const NormArgs &args)
{
    switch (args.a.dtype) {
    case SCANSCAM_F32: return launch_norm<float>(back, plan, grid, lds, stream, args);
    case SCANSCAM_BF16: return launch_norm<__bf16>(back, plan, grid, lds, stream, args);
    default: return launch_norm<_Float16>(back, plan, grid, lds, stream, args);
    }
}

}  // namespace

extern "C" {

int scanscam_norm_fwd(const scanscam_norm *a, void *stream)
{
    SCANSCAM_CHECK(check_norm(a));
    const bool eight = a->out_dtype == SCANSCAM_I8 || a->out_dtype == SCANSCAM_F8;
    if (!eight && a->out_dtype != a->dtype) return SCANSCAM_EDTYPE;
    if (a->rows == 0 || (a->channels == 0 && !eight)) return SCANSCAM_OK;
    if ((a->y == nullptr && a->channels > 0) || (eight && a->scale == nullptr)) return SCANSCAM_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a->channels == 0) {
        const hipError_t err = launch_op(ones_kernel, dim3((unsigned)ceil_div(a->rows, 256)), dim3(256), 0, s, Ones{a->scale, a->rows});
        return err == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
    }
    if (!eight && misaligned(a->y, (size_t)activation_size(a->dtype))) return SCANSCAM_EALIGN;
    const NormPlan plan = norm_plan(*a);
    // A launch has fewer than 2^32 threads: more rows than that are several launches, a multiple of 8 rows each, so that a launch's
    // first row begins on a vector's border where the first one of all does.
    const int64_t threads = 64 * plan.waves * plan.groups, most = ((int64_t(1) << 32) / threads - 1) * plan.groups / 8 * 8;
    for (int64_t row = 0; row < a->rows; row += most) {
        const scanscam_norm now = rows_from(*a, row, a->rows - row < most ? a->rows - row : most);
        const hipError_t err = run_norm(false, plan, (unsigned)ceil_div(now.rows, plan.groups), 0, s, NormArgs{now, plan.waves, plan.shifted, nullptr});
        if (err != hipSuccess) return SCANSCAM_ELAUNCH;
    }
    return SCANSCAM_OK;
}

size_t scanscam_norm_workspace_bytes(const scanscam_norm *a)
{
    if (a == nullptr || a->rows <= 0 || a->channels <= 0 || a->channels > kNormMostChannels) return 0;
    // (enough for every number of rows a workgroup, which depends on the residual: it may be asked for before the pointers are there)
    return (size_t)((a->rows < kNormMostParts ? a->rows : kNormMostParts) * a->channels) * sizeof(float);
}

int scanscam_norm_bwd(const scanscam_norm *a, void *stream)
{
    SCANSCAM_CHECK(check_norm(a));
    if (a->channels == 0) return SCANSCAM_OK;
    if (a->gweight == nullptr) return SCANSCAM_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a->rows == 0) return column_sum({nullptr, 0, 0, {a->gweight}, {a->channels}}, s) == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
    if (a->gy == nullptr || a->gx == nullptr || a->rstd == nullptr || (a->gsum != nullptr && a->residual == nullptr) ||
        (a->gresidual != nullptr && a->residual == nullptr))
        return SCANSCAM_EINVAL;
    const size_t size = (size_t)activation_size(a->dtype);
    if (misaligned(a->gy, size) || misaligned(a->gx, size)) return SCANSCAM_EALIGN;
    if (a->workspace == nullptr || a->workspace_bytes < scanscam_norm_workspace_bytes(a)) return SCANSCAM_EWORKSPACE;
    if (misaligned(a->workspace, 16)) return SCANSCAM_EALIGN;
    const NormPlan plan = norm_plan(*a);
    const int64_t grid = norm_bwd_workgroups(*a, plan);
    float *part = static_cast<float *>(a->workspace);
    hipError_t err = run_norm(true, plan, (unsigned)grid, plan.groups > 1 ? (size_t)a->channels * sizeof(float) : 0, s, NormArgs{*a, plan.waves, false, part});
    if (err == hipSuccess) err = column_sum({part, grid, a->channels, {a->gweight}, {a->channels}}, s);
    return err == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
}

}  // extern "C"
