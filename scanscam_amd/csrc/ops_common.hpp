// What the kernels of the state space layer's operators share: parameters of any type, sequences in a stream of tokens, the
// activations' functions, column sums.
#pragma once

#include "scanscam_ops.h"

#include "scan_kernels.hpp"

#include <atomic>

namespace scanscam {

typedef float float4v __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;

__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A parameter's element, whatever its type; `fill` where there is no parameter.
__device__ __forceinline__ float param(const scanscam_param &p, int64_t i, float fill = 0.0f)
{
    if (p.p == nullptr) return fill;
    if (p.dtype == SCANSCAM_F32) return static_cast<const float *>(p.p)[i];
    if (p.dtype == SCANSCAM_BF16) return (float)static_cast<const __bf16 *>(p.p)[i];
    return (float)static_cast<const _Float16 *>(p.p)[i];
}

__device__ __forceinline__ int64_t index_at(const void *p, int wide, int64_t i)
{
    return wide ? static_cast<const int64_t *>(p)[i] : (int64_t)static_cast<const int32_t *>(p)[i];
}

// exp by the hardware's 2^x (one unit in the last place), 1/x likewise; both flush no result that fp32 sums would keep.
__device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
__device__ __forceinline__ float sigmoid_(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_(-x)); }

// log(1 + e^x) = max(x, 0) + log(1 + t), t = e^-|x| in (0, 1]. log(1 + t) = 2 artanh(w), w = t / (2 + t) <= 1/3: small t (step
// sizes of 0.001 are where a model starts) keep all their digits, which the logarithm of the rounded 1 + t loses. With v = 2 w,
// artanh(w) / w = 1 + v^2/12 + v^4/80 + ... as the polynomial of degree 4 in v^2 whose largest relative error over the range
// is least (found by repeated weighted least squares), below 2^-27. A NaN stays one through t.
__device__ __forceinline__ float softplus_(float x)
{
    const float t = exp_(-__builtin_fabsf(x));
    const float v = t * __builtin_amdgcn_rcpf(__builtin_fmaf(t, 0.5f, 1.0f)), q = v * v;
    float s = 0.000547109114f;
    s = __builtin_fmaf(s, q, 0.0021876411f);
    s = __builtin_fmaf(s, q, 0.0125067271f);
    s = __builtin_fmaf(s, q, 0.0833330229f);
    s = __builtin_fmaf(s, q, 1.0f);
    return __builtin_fmaf(v, s, __builtin_fmaxf(x, 0.0f));
}

// VEC neighbouring elements, of which the first `count` are there; they need no more than their own alignment.
template <typename ST, int VEC>
__device__ __forceinline__ void load_part(const ST *p, int count, float (&f)[VEC])
{
    if (count >= VEC) {
        constexpr int PIECE = VEC * sizeof(ST) > 16 ? 16 / sizeof(ST) : VEC;
        using raw_t = typename RawT<sizeof(ST) * PIECE>::type;
        typedef raw_t raw_unaligned_t __attribute__((aligned(sizeof(ST))));
#pragma unroll
        for (int j = 0; j < VEC; j += PIECE) {
            const raw_t raw = *reinterpret_cast<const raw_unaligned_t *>(p + j);
            const Elems<ST, PIECE> e = __builtin_bit_cast(Elems<ST, PIECE>, raw);
#pragma unroll
            for (int k = 0; k < PIECE; k++) f[j + k] = (float)e.e[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < VEC; k++) f[k] = k < count ? (float)p[k] : 0.0f;
    }
}
template <typename ST, int VEC>
__device__ __forceinline__ void store_some(ST *p, int count, const float (&f)[VEC])
{
    if (count >= VEC) {
        constexpr int PIECE = VEC * sizeof(ST) > 16 ? 16 / sizeof(ST) : VEC;
        using raw_t = typename RawT<sizeof(ST) * PIECE>::type;
        typedef raw_t raw_unaligned_t __attribute__((aligned(sizeof(ST))));
#pragma unroll
        for (int j = 0; j < VEC; j += PIECE) {
            Elems<ST, PIECE> e;
#pragma unroll
            for (int k = 0; k < PIECE; k++) e.e[k] = (ST)f[j + k];
            *reinterpret_cast<raw_unaligned_t *>(p + j) = __builtin_bit_cast(raw_t, e);
        }
    } else {
#pragma unroll
        for (int k = 0; k < VEC; k++)
            if (k < count) p[k] = (ST)f[k];
    }
}

// Whole vectors of neighbouring elements, as they are stored: what is asked for is waited for where it is taken apart.
template <typename ST, int VEC> struct Stored {
    Elems<ST, VEC> e;
    __device__ __forceinline__ void load(const ST *p)
    {
        constexpr int PIECE = VEC * sizeof(ST) > 16 ? 16 / sizeof(ST) : VEC;
        using raw_t = typename RawT<sizeof(ST) * PIECE>::type;
        typedef raw_t raw_unaligned_t __attribute__((aligned(sizeof(ST))));
        struct Raw { raw_t r[VEC / PIECE]; } raw;
#pragma unroll
        for (int i = 0; i < VEC / PIECE; i++) raw.r[i] = *reinterpret_cast<const raw_unaligned_t *>(p + i * PIECE);
        e = __builtin_bit_cast(decltype(e), raw);
    }
    __device__ __forceinline__ float operator[](int i) const { return (float)e.e[i]; }
};

// COUNT neighbouring elements of a parameter, of which the first `there` are there (all: in vectors).
template <int COUNT> __device__ __forceinline__ void params(const scanscam_param &p, int64_t at, int there, float (&f)[COUNT], float fill = 0.0f)
{
    if (p.p == nullptr) {
#pragma unroll
        for (int i = 0; i < COUNT; i++) f[i] = fill;
    } else if (there < COUNT || COUNT % 4 != 0) {
#pragma unroll
        for (int i = 0; i < COUNT; i++) f[i] = i < there ? param(p, at + i) : 0.0f;
    } else if (p.dtype == SCANSCAM_F32) {
#pragma unroll
        for (int i = 0; i < COUNT; i += 4) {
            Stored<float, 4> s;
            s.load(static_cast<const float *>(p.p) + at + i);
#pragma unroll
            for (int k = 0; k < 4; k++) f[i + k] = s[k];
        }
    } else if (p.dtype == SCANSCAM_BF16) {
#pragma unroll
        for (int i = 0; i < COUNT; i += 4) {
            Stored<__bf16, 4> s;
            s.load(static_cast<const __bf16 *>(p.p) + at + i);
#pragma unroll
            for (int k = 0; k < 4; k++) f[i + k] = s[k];
        }
    } else {
#pragma unroll
        for (int i = 0; i < COUNT; i += 4) {
            Stored<_Float16, 4> s;
            s.load(static_cast<const _Float16 *>(p.p) + at + i);
#pragma unroll
            for (int k = 0; k < 4; k++) f[i + k] = s[k];
        }
    }
}

// The sequence that token t of a packed stream belongs to: the last one that starts at or before t.
__device__ __forceinline__ int64_t sequence_of(const void *offsets, int wide, int64_t sequences, int64_t t)
{
    int64_t lo = 0, hi = sequences - 1;  // the answer lies in [lo, hi]
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        if (index_at(offsets, wide, mid) <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ int64_t clamp_(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// Sums over p < parts of in[p * pitch + m], in an order that the sizes alone decide: 16 threads a column, each over every 16th
// part, joined in order. More than kMostSummed parts are first summed in groups of kSummed, each into the place of its first one, so that
// no thread adds up more than 64. (A part is itself a sum: of up to 128 tokens of a convolution; of a stretch of time of the selective scan, a value
// a tile; of every 4096th row or more of a norm.) The columns are those of up to three outputs, one behind the other; an output may be NULL.
struct ColumnSum {
    float *in;
    int64_t parts, pitch;
    float *out[3];
    int64_t columns[3];
    int64_t each, first;  // parts of a group, and the first group; each = 0: all parts, to the outputs
};
constexpr int64_t kMostSummed = 1024, kSummed = 256;

__global__ __launch_bounds__(1024) void column_sum_kernel(ColumnSum a);

template <typename Kernel, typename Args>
inline hipError_t launch_op(Kernel kernel, dim3 grid, dim3 block, size_t lds, hipStream_t stream, const Args &args)
{
    Args copy = args;
    void *params[] = {&copy};
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, params, lds, stream);
}

// A launch that may need more LDS than a kernel gets unasked. The limit belongs to the process: it is set once on each device, to the most
// that any call needs (one that a call sets for itself could be lowered by another thread's before the launch).
template <auto Kernel, typename Args> inline hipError_t launch_wide(dim3 grid, int threads, int words, int most_words, hipStream_t stream, const Args &args)
{
    static std::atomic<uint64_t> ready{0};  // a bit a device
    int device = 0;
    hipError_t err = hipGetDevice(&device);
    if (err != hipSuccess) return err;
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if ((ready.load(std::memory_order_acquire) & bit) == 0) {
        err = hipFuncSetAttribute(reinterpret_cast<const void *>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, most_words * (int)sizeof(float));
        if (err != hipSuccess) return err;
        ready.fetch_or(bit, std::memory_order_release);
    }
    return launch_op(Kernel, grid, dim3((unsigned)threads), (size_t)words * sizeof(float), stream, args);
}

inline hipError_t column_sum(ColumnSum a, hipStream_t stream)
{
    const unsigned grid = (unsigned)ceil_div(a.columns[0] + a.columns[1] + a.columns[2], 64);
    for (; a.parts > kMostSummed; a.parts = ceil_div(a.parts, kSummed), a.pitch *= kSummed) {
        const int64_t groups = ceil_div(a.parts, kSummed), most = 32768;  // (a launch has at most 65535 workgroups in its second dimension)
        a.each = kSummed;
        for (a.first = 0; a.first < groups; a.first += most) {
            const int64_t now = groups - a.first < most ? groups - a.first : most;
            const hipError_t err = launch_op(column_sum_kernel, dim3(grid, (unsigned)now), dim3(1024), 0, stream, a);
            if (err != hipSuccess) return err;
        }
    }
    a.each = a.first = 0;
    return launch_op(column_sum_kernel, dim3(grid), dim3(1024), 0, stream, a);
}

// A single token's step in launches of fewer than 2^32 threads along each dimension and of a second dimension that a grid can have.
template <typename Step> struct StepPart {
    Step a;
    int64_t row0;     // the first row of this launch
    uint32_t block0;  // and its first block of channels
};
// `whole` does what one launch can, `part` each of several.
template <typename Kernel, typename Step>
inline hipError_t launch_step(Kernel whole, Kernel part, int64_t rows, int64_t blocks, dim3 block, hipStream_t stream, const Step &a)
{
    const int64_t most_rows = ((int64_t(1) << 32) / block.x - 1) * block.y, most_blocks = 32768;
    if (rows <= most_rows && blocks <= most_blocks)
        return launch_op(whole, dim3((unsigned)ceil_div(rows, block.y), (unsigned)blocks), block, 0, stream, StepPart<Step>{a, 0, 0});
    hipError_t err = hipSuccess;
    for (int64_t row = 0; row < rows; row += most_rows) {
        for (int64_t first = 0; first < blocks && err == hipSuccess; first += most_blocks) {
            const dim3 grid((unsigned)ceil_div(rows - row < most_rows ? rows - row : most_rows, block.y), (unsigned)(blocks - first < most_blocks ? blocks - first : most_blocks));
            err = launch_op(part, grid, block, 0, stream, StepPart<Step>{a, row, (uint32_t)first});
        }
    }
    return err;
}

// --- checks of arguments ---------------------------------------------------------------------------------------------------
inline int activation_size(int dtype)
{
    return dtype == SCANSCAM_F32 ? 4 : dtype == SCANSCAM_BF16 || dtype == SCANSCAM_F16 ? 2 : 0;
}
inline bool misaligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }
inline int check_tokens(const scanscam_tokens &t, int size)
{
    if (t.p == nullptr || t.batch < 0 || t.token < 0 || t.group < 0) return SCANSCAM_EINVAL;
    return misaligned(t.p, (size_t)size) ? SCANSCAM_EALIGN : SCANSCAM_OK;
}
inline int check_param(const scanscam_param &p, bool required)
{
    if (p.p == nullptr) return required ? SCANSCAM_EINVAL : SCANSCAM_OK;
    const int size = activation_size(p.dtype);
    if (size == 0) return SCANSCAM_EDTYPE;
    return misaligned(p.p, (size_t)size) ? SCANSCAM_EALIGN : SCANSCAM_OK;
}

constexpr int64_t kMostTokens = SCANSCAM_MOST_TOKENS, kMostChannels = SCANSCAM_MOST_CHANNELS;

#define SCANSCAM_CHECK(expr)                      \
    do {                                          \
        const int rc_ = (expr);                   \
        if (rc_ != SCANSCAM_OK) return rc_;       \
    } while (0)

}  // namespace scanscam
