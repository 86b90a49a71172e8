// C ABI of the selective scan (declared in include/scanscam_ops.h): argument checks, launch shapes, launches.
#include "selective_kernels.hpp"

#include <atomic>

namespace {

using namespace scanscam;

constexpr int kTokensALane = 8;  // K
constexpr int kTile = Geometry<kTokensALane>::kTile;
constexpr int kMostStates = 256;
constexpr int64_t kMostParts = 1024;

int check_sizes(int64_t channels, int64_t groups, int64_t N, int dtype)
{
    if (channels < 0 || channels > kMostChannels || groups < 1 || channels % groups != 0 || N < 1 || N > kMostStates) return SCANSCAM_EINVAL;
    return activation_size(dtype) == 0 ? SCANSCAM_EDTYPE : SCANSCAM_OK;
}

// The kernels reach the tokens of a tile from its first one with 32-bit offsets.
int check_near(const scanscam_tokens &t, int size)
{
    SCANSCAM_CHECK(check_tokens(t, size));
    return t.token < SCANSCAM_MOST_TOKEN_STRIDE ? SCANSCAM_OK : SCANSCAM_EINVAL;
}

int check_selective(const scanscam_selective *a)
{
    if (a == nullptr) return SCANSCAM_EINVAL;
    SCANSCAM_CHECK(check_sizes(a->channels, a->groups, a->N, a->dtype));
    if (a->batch < 0 || a->T < 0 || a->T >= kMostTokens || a->sequences < 0 || a->sequences >= kMostTokens || a->parts < 0 || a->parts > kMostParts) return SCANSCAM_EINVAL;
    if (a->offsets != nullptr ? a->batch != 1 || a->sequences < 1 : a->sequences != a->batch) return SCANSCAM_EINVAL;
    if (a->batch > 0 && a->T > (kMostTokens - 1) / a->batch) return SCANSCAM_EINVAL;
    if (a->channels == 0 || a->sequences == 0) return SCANSCAM_OK;
    SCANSCAM_CHECK(check_param(a->A, true));
    SCANSCAM_CHECK(check_param(a->D, false));
    SCANSCAM_CHECK(check_param(a->dt_bias, false));
    if (misaligned(a->offsets, a->offsets64 ? 8 : 4) || misaligned(a->state_in, 4) || misaligned(a->state_out, 4) || misaligned(a->saved, 16))
        return SCANSCAM_EALIGN;
    if (a->batch * a->T == 0) return SCANSCAM_OK;
    const int size = activation_size(a->dtype);
    for (const scanscam_tokens *t : {&a->x, &a->dt, &a->B, &a->C}) SCANSCAM_CHECK(check_near(*t, size));
    return a->z.p != nullptr ? check_near(a->z, size) : SCANSCAM_OK;
}

// A launch that may need more LDS than a kernel gets unasked. The limit belongs to the process: it is set once on each device, to the most
// that any call needs (one that a call sets for itself could be lowered by another thread's before the launch).
template <auto Kernel, typename Args> hipError_t launch_wide(dim3 grid, int threads, int words, int most_words, hipStream_t stream, const Args &args)
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

// A launch has fewer than 2^32 threads: more parts than that are several launches.
template <auto Kernel> hipError_t launch_units(SelectiveArgs args, int64_t units, int threads, int words, int most_words, hipStream_t stream)
{
    const int64_t blocks = args.a.groups * args.blocks, most = ((int64_t(1) << 32) / threads - 1) / blocks;
    hipError_t err = hipSuccess;
    for (int64_t first = 0; first < units && err == hipSuccess; first += most) {
        args.unit0 = (uint32_t)first;
        err = launch_wide<Kernel>(dim3((unsigned)(blocks * (units - first < most ? units - first : most))), threads, words, most_words, stream, args);
    }
    return err;
}

struct Plan {
    int split;     // forwards: waves that share the states of a channel out among them
    int64_t span;  // tokens of a part that the time of a sequence is cut into; packed ones that are not longer stay whole
};

int64_t forward_blocks(const scanscam_selective &a, int split) { return ceil_div(a.channels / a.groups, kFwdWaves / split * kRows); }
// Two sets of 16 channels a workgroup where that leaves two workgroups for every CU.
int backward_sets(const scanscam_selective &a)
{
    const int64_t wide = kBwdMostSets * kBwdChannels;
    return a.N <= kStateBlock && a.sequences * a.groups * ceil_div(a.channels / a.groups, wide) >= 512 ? kBwdMostSets : 1;
}
int64_t backward_blocks(const scanscam_selective &a) { return ceil_div(a.channels / a.groups, kBwdChannels * backward_sets(a)); }

// Parts of one length for about two workgroups a CU, whole tiles each. (Known at N = 16; from N = 40 on a CU holds one.)
int64_t span_for(const scanscam_selective &a, int64_t blocks, int64_t shortest)
{
    const int64_t tiles = (a.offsets != nullptr ? 1 : a.sequences) * ceil_div(a.T, kTile) * a.groups * blocks, each = ceil_div(tiles, 512);
    return (each > shortest ? each : shortest) * kTile;
}

// Parts that were asked for (a measurement's, or a test's).
int64_t span_of(const scanscam_selective &a)
{
    const int64_t each = ceil_div(ceil_div(a.T, kTile), a.parts);
    return (each > 0 ? each : 1) * kTile;
}

// Two workgroups fit a CU (one from N = 40 on; all figures here are of N = 16), and one keeps it nearly as busy, so that from 192 workgroups on nothing is cut. Below, sharing the states
// of a channel out costs less than parts of time, whose first pass repeats most of the arithmetic, as long as it is two waves
// (bf16, N = 16, us: [4, 2048, 1024] 120 whole, 83 by two waves, 92 in 4 parts; [6, 2048, 1024] 117, 113, 134); four
// or eight waves have too little to do for the tokens' own work and the barriers, so that with fewer channels parts win where there are
// tiles for them ([2, 2048, 1024] 114 whole, 61 by four waves, 56 in 8 parts; [1, 2048, 1024] 113, 59, 38 in 16), and not in
// short sequences ([1, 512, 2048] 34 whole, 24 by four waves, 28 in 4 parts). Packed sequences differ in length, and the longest may take
// longer than all work shared out evenly: two waves then halve the time that one workgroup is busy with it (13 sequences, 8021
// tokens, 2048 channels, six sets of lengths, one wave / two waves / cut into parts of four tiles: 113/133/189, 136/126/173, 292/207/188,
// 123/125/170, 151/128/179, 104/124/184 us).
Plan forward_plan(const scanscam_selective &a)
{
    if (a.parts > 0) return {1, span_of(a)};
    const int64_t whole = a.sequences * a.groups * forward_blocks(a, 1);
    if (whole >= 192) return {a.offsets != nullptr && whole < 1024 && a.N > 1 ? 2 : 1, kWhole};
    Plan p{1, kWhole};
    if (whole >= 96) {
        p.split = a.N > 1 ? 2 : 1;
    } else if (ceil_div(a.T, kTile) >= 8) {
        p.span = span_for(a, forward_blocks(a, 1), 1);
    } else {
        while (p.split < kFwdWaves && p.split < a.N && a.sequences * a.groups * forward_blocks(a, p.split) < 256) p.split *= 2;
    }
    return p;
}
Plan backward_plan(const scanscam_selective &a)
{
    if (a.parts > 0) return {1, span_of(a)};
    const int64_t blocks = backward_blocks(a), whole = a.sequences * a.groups * blocks;
    return {1, whole < 256 ? span_for(a, blocks, 1) : a.offsets != nullptr ? span_for(a, blocks, 4) : kWhole};
}

// Whether any sequence can be longer than a part.
bool cut(const scanscam_selective &a, int64_t span) { return a.T > span; }

uint32_t each_of(const scanscam_selective &a, int64_t span) { return (uint32_t)(a.T > span ? ceil_div(a.T, span) : 1); }
size_t ends_words(const scanscam_selective &a, int64_t span) { return cut(a, span) ? (size_t)(all_units(a, span) * (a.N + 1) * a.channels) : 0; }
size_t bc_words(const scanscam_selective &a) { return (size_t)(a.groups * backward_blocks(a) * a.batch * a.T * 2 * a.N); }

template <typename ST> hipError_t run_fwd(const scanscam_selective &a, hipStream_t stream)
{
    constexpr int K = kTokensALane;
    const Plan plan = forward_plan(a);
    const SelectiveArgs args{a, plan.split, 0, (uint32_t)forward_blocks(a, plan.split), each_of(a, plan.span), plan.span, static_cast<float *>(a.workspace), nullptr, nullptr};
    const int64_t units = all_units(a, plan.span);
    const int words = ForwardLds<K>::words(kFwdWaves / plan.split * kRows, (int)a.N);
    constexpr int most = ForwardLds<K>::words(kFwdWaves * kRows, kMostStates);
    if (cut(a, plan.span)) {
        const hipError_t err = launch_units<selective_fwd_kernel<ST, K, true>>(args, units, kFwdWaves * 64, words, most, stream);
        if (err != hipSuccess) return err;
    }
    return launch_units<selective_fwd_kernel<ST, K, false>>(args, units, kFwdWaves * 64, words, most, stream);
}

// gB and gC from the sums of the blocks; of no blocks (no channels) they are zero.
template <typename ST> hipError_t run_bc(const scanscam_selective &a, const float *bc, int64_t blocks, hipStream_t stream)
{
    // (a launch's values are numbered with 32 bits, its groups are its grid's second dimension)
    const int64_t tokens = a.batch * a.T, wide = 2 * a.N, most = (int64_t(1) << 31) / wide, most_groups = 32768;
    const bool four = a.N % 4 == 0;
    hipError_t err = hipSuccess;
    for (int64_t token = 0; token < tokens; token += most) {
        const int64_t now = tokens - token < most ? tokens - token : most;
        for (int64_t group = 0; group < a.groups && err == hipSuccess; group += most_groups) {
            const dim3 grid((unsigned)ceil_div(now * wide, four ? 1024 : 256), (unsigned)(a.groups - group < most_groups ? a.groups - group : most_groups));
            err = launch_op(four ? selective_bc_kernel<ST, 4> : selective_bc_kernel<ST, 1>, grid, dim3(256), 0, stream,
                            GroupSum{a, bc, blocks, (uint32_t)token, (uint32_t)now, (uint32_t)group});
        }
    }
    return err;
}

template <typename ST> hipError_t run_bwd(const scanscam_selective &a, hipStream_t stream)
{
    constexpr int K = kTokensALane;
    const Plan plan = backward_plan(a);
    const int sets = backward_sets(a);
    const int64_t blocks = backward_blocks(a), units = all_units(a, plan.span);
    float *ends = static_cast<float *>(a.workspace), *bc = ends + ends_words(a, plan.span), *sums = bc + bc_words(a);
    const SelectiveArgs args{a, sets, 0, (uint32_t)blocks, each_of(a, plan.span), plan.span, ends, bc, sums};
    const int words = BackwardLds<K>::words((int)a.N, sets);
    constexpr int one = BackwardLds<K>::words(kMostStates, 1), two = BackwardLds<K>::words(kStateBlock, kBwdMostSets), most = one > two ? one : two;
    hipError_t err = hipSuccess;
    if (cut(a, plan.span)) err = launch_units<selective_bwd_kernel<ST, K, true>>(args, units, kBwdWaves * 64, words, most, stream);
    if (err == hipSuccess) err = launch_units<selective_bwd_kernel<ST, K, false>>(args, units, kBwdWaves * 64, words, most, stream);
    if (err == hipSuccess) err = run_bc<ST>(a, bc, blocks, stream);
    const int64_t pitch = (a.N + 2) * a.channels;
    if (err == hipSuccess) err = column_sum({sums, units, pitch, {a.gA, a.gD, a.gdt_bias}, {a.N * a.channels, a.channels, a.channels}}, stream);
    return err;
}

template <typename ST> hipError_t run_step(const scanscam_selective_step &a, hipStream_t stream)
{
    int lanes = 1;
    while (lanes < 32 && lanes * 4 < a.N) lanes *= 2;
    const int64_t blocks = ceil_div(a.channels, 256 / lanes);
    switch (lanes) {
    case 1: return launch_step(selective_step_kernel<ST, 1, false>, selective_step_kernel<ST, 1, true>, a.rows, blocks, dim3(256), stream, a);
    case 2: return launch_step(selective_step_kernel<ST, 2, false>, selective_step_kernel<ST, 2, true>, a.rows, blocks, dim3(256), stream, a);
    case 4: return launch_step(selective_step_kernel<ST, 4, false>, selective_step_kernel<ST, 4, true>, a.rows, blocks, dim3(256), stream, a);
    case 8: return launch_step(selective_step_kernel<ST, 8, false>, selective_step_kernel<ST, 8, true>, a.rows, blocks, dim3(256), stream, a);
    case 16: return launch_step(selective_step_kernel<ST, 16, false>, selective_step_kernel<ST, 16, true>, a.rows, blocks, dim3(256), stream, a);
    default: return launch_step(selective_step_kernel<ST, 32, false>, selective_step_kernel<ST, 32, true>, a.rows, blocks, dim3(256), stream, a);
    }
}

int check_workspace(const scanscam_selective &a, int direction)
{
    const size_t bytes = scanscam_selective_workspace_bytes(&a, direction);
    if (bytes > 0 && (a.workspace == nullptr || a.workspace_bytes < bytes)) return SCANSCAM_EWORKSPACE;
    return misaligned(a.workspace, 16) ? SCANSCAM_EALIGN : SCANSCAM_OK;
}

int status(hipError_t err) { return err == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH; }

}  // namespace

extern "C" {

size_t scanscam_selective_saved_bytes(const scanscam_selective *a)
{
    if (a == nullptr || check_sizes(a->channels, a->groups, a->N, a->dtype) != SCANSCAM_OK || a->batch <= 0 || a->T <= 0 || a->sequences <= 0) return 0;
    return (size_t)(all_tiles(*a, kTile) * a->N * a->channels) * sizeof(float);
}

size_t scanscam_selective_workspace_bytes(const scanscam_selective *a, int direction)
{
    if (a == nullptr || check_sizes(a->channels, a->groups, a->N, a->dtype) != SCANSCAM_OK || a->batch <= 0 || a->T < 0 || a->sequences <= 0) return 0;
    if (direction == SCANSCAM_FORWARD) return ends_words(*a, forward_plan(*a).span) * sizeof(float);
    const int64_t span = backward_plan(*a).span;
    return (ends_words(*a, span) + bc_words(*a) + (size_t)(all_units(*a, span) * (a->N + 2) * a->channels)) * sizeof(float);
}

int scanscam_selective_fwd(const scanscam_selective *a, void *stream)
{
    SCANSCAM_CHECK(check_selective(a));
    if (a->channels == 0 || a->sequences == 0) return SCANSCAM_OK;
    if (a->batch * a->T > 0) SCANSCAM_CHECK(check_near(a->y, activation_size(a->dtype)));
    SCANSCAM_CHECK(check_workspace(*a, SCANSCAM_FORWARD));
    hipStream_t s = static_cast<hipStream_t>(stream);
    return status(a->dtype == SCANSCAM_F32    ? run_fwd<float>(*a, s)
                  : a->dtype == SCANSCAM_BF16 ? run_fwd<__bf16>(*a, s)
                                              : run_fwd<_Float16>(*a, s));
}

int scanscam_selective_bwd(const scanscam_selective *a, void *stream)
{
    SCANSCAM_CHECK(check_selective(a));
    if (a->channels == 0) {
        if (a->batch * a->T == 0) return SCANSCAM_OK;
        for (const scanscam_tokens *t : {&a->gB, &a->gC}) SCANSCAM_CHECK(check_near(*t, activation_size(a->dtype)));
        hipStream_t s = static_cast<hipStream_t>(stream);
        return status(a->dtype == SCANSCAM_F32    ? run_bc<float>(*a, nullptr, 0, s)
                      : a->dtype == SCANSCAM_BF16 ? run_bc<__bf16>(*a, nullptr, 0, s)
                                                  : run_bc<_Float16>(*a, nullptr, 0, s));
    }
    if (a->gA == nullptr) return SCANSCAM_EINVAL;
    if (a->sequences > 0) {
        if (a->batch * a->T > 0) {
            const int size = activation_size(a->dtype);
            for (const scanscam_tokens *t : {&a->gy, &a->gx, &a->gdt, &a->gB, &a->gC}) SCANSCAM_CHECK(check_near(*t, size));
            if (a->z.p != nullptr) SCANSCAM_CHECK(check_near(a->gz, size));
            if (a->saved == nullptr) return SCANSCAM_EINVAL;
        }
        if (misaligned(a->gstate_out, 4) || misaligned(a->gstate_in, 4)) return SCANSCAM_EALIGN;
        SCANSCAM_CHECK(check_workspace(*a, SCANSCAM_BACKWARD));
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a->sequences == 0) {
        return status(column_sum({nullptr, 0, 0, {a->gA, a->gD, a->gdt_bias}, {a->N * a->channels, a->channels, a->channels}}, s));
    }
    return status(a->dtype == SCANSCAM_F32    ? run_bwd<float>(*a, s)
                  : a->dtype == SCANSCAM_BF16 ? run_bwd<__bf16>(*a, s)
                                              : run_bwd<_Float16>(*a, s));
}

int scanscam_selective_step_fwd(const scanscam_selective_step *a, void *stream)
{
    if (a == nullptr) return SCANSCAM_EINVAL;
    SCANSCAM_CHECK(check_sizes(a->channels, a->groups, a->N, a->dtype));
    if (a->rows < 0 || a->rows >= kMostTokens || a->slots < 0) return SCANSCAM_EINVAL;
    if (a->rows == 0 || a->channels == 0) return SCANSCAM_OK;
    const int size = activation_size(a->dtype);
    for (const scanscam_tokens *t : {&a->x, &a->dt, &a->B, &a->C, &a->y}) SCANSCAM_CHECK(check_tokens(*t, size));
    if (a->z.p != nullptr) SCANSCAM_CHECK(check_tokens(a->z, size));
    SCANSCAM_CHECK(check_param(a->A, true));
    SCANSCAM_CHECK(check_param(a->D, false));
    SCANSCAM_CHECK(check_param(a->dt_bias, false));
    if (a->state == nullptr) return SCANSCAM_EINVAL;
    if (misaligned(a->state, 4) || misaligned(a->slot, a->slot64 ? 8 : 4)) return SCANSCAM_EALIGN;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return status(a->dtype == SCANSCAM_F32    ? run_step<float>(*a, s)
                  : a->dtype == SCANSCAM_BF16 ? run_step<__bf16>(*a, s)
                                              : run_step<_Float16>(*a, s));
}

}  // extern "C"
