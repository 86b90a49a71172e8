// Norm of every group of a row's channels, with an activation and a gate, and the gradients.
//
//   h = (x - mean) * rstd,  u = h * weight + bias,  y = act(u) * silu(z)
//   backwards, with g = gy * silu(z) * act'(u):  gz = gy * act(u) * silu'(z),  gweight = sum over rows of g * h,  gbias = of g,
//   e = g * weight:  gx = rstd * (e - mean(e) - h * mean(e * h))
//
// Memory bounds it: each tensor once. A group's channels of a row stay in the registers of a team of lanes (up to 64, then up to 8
// waves), so that mean and variance are taken one after the other from the values themselves, and the backward pass takes them anew
// instead of reading them. A team keeps its group and goes through rows, with the next row's values on their way: parameters are read
// once, and their gradients are sums in registers until the end. 32768 rows of 2048 in 16 groups, bf16, gated, with gradients: 217 us, 4.9 TB/s; 16384 rows
// of 2050 in 10, fp16: 44 us, 4.5 TB/s. Backwards that is for some eight groups and more (see the host's count of teams).
#pragma once

#include "ops_common.hpp"
#include "scanscam_attention.h"

namespace scanscam {

struct GroupNormArgs {
    scanscam_group_norm a;
    int64_t parts;  // teams of a group: each takes every parts-th row
    int32_t size;   // channels of a group
    int32_t waves;  // of a team, where it is more than one
    float *part;    // backward: [parts][weight's columns, bias's columns]
};

template <typename ST> constexpr int group_vec() { return 16 / (int)sizeof(ST); }
// Vectors of a lane where several waves are a team: 8 waves hold 8192 channels, and their backward pass fits the registers of two waves a SIMD.
template <typename ST> constexpr int group_most() { return sizeof(ST) == 4 ? 4 : 2; }

// Sum over L neighbouring lanes, to all of them.
template <int L> __device__ __forceinline__ float team_sum(float v)
{
    if constexpr (L >= 2) v += dpp_move<0xb1, 0xf>(0.0f, v);   // lanes 1 0 3 2
    if constexpr (L >= 4) v += dpp_move<0x4e, 0xf>(0.0f, v);   // lanes 2 3 0 1
    if constexpr (L >= 8) v += dpp_move<0x141, 0xf>(0.0f, v);  // the other four of eight
    if constexpr (L >= 16) v += dpp_move<0x140, 0xf>(0.0f, v); // the other eight of sixteen
    if constexpr (L >= 32) v += __shfl_xor(v, 16);
    if constexpr (L >= 64) v += __shfl_xor(v, 32);
    return v;
}
// ... and over the waves of a team, in order. The slots are used in turn, so that one barrier is enough.
template <int L, bool WAVES> __device__ __forceinline__ float over_team(float v, int waves, float (*slots)[8], int &turn)
{
    v = team_sum<L>(v);
    if constexpr (WAVES) {
        float *now = slots[turn];
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) now[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
        for (int w = 0; w < waves; w++) v += now[w];
    }
    return v;
}

__device__ __forceinline__ float silu_slope(float z, float s) { return s * __builtin_fmaf(z, 1.0f - s, 1.0f); }

// EXACT: a group is a whole number of vectors. Else its last vector ends where the group does and covers some of the channels of the one before a second
// time, which its sums leave out and both write alike: loads and stores of single channels took half of the time (groups of 205: 63 us of
// [16384, 2050]). A group smaller than a vector is one lane's, channel by channel.
template <typename ST, int L, int NV, bool WAVES, bool EXACT> struct Team {
    static constexpr int VEC = group_vec<ST>();
    int64_t group, part;
    int at[NV], count[NV], skip[NV];  // channels of the group: the first, how many of a vector's are there, and how many of them are another's
    bool there;
    __device__ __forceinline__ explicit Team(const GroupNormArgs &args)
    {
        const int64_t team = WAVES ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
        const int lane = WAVES ? threadIdx.x : threadIdx.x % L, lanes = WAVES ? 64 * args.waves : L;
        there = team < args.a.groups * args.parts;
        group = team % args.a.groups;
        part = team / args.a.groups;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int first = (j * lanes + lane) * VEC, left = args.size - first;
            at[j] = EXACT || left >= VEC || left <= 0 || args.size < VEC ? first : args.size - VEC;
            skip[j] = first - at[j];
            count[j] = left + skip[j];
        }
    }
    __device__ __forceinline__ bool own(int j, int k) const { return EXACT ? count[j] > 0 : k >= skip[j] && k < count[j]; }
    __device__ __forceinline__ void load(const ST *p, Elems<ST, VEC> (&e)[NV]) const
    {
        using raw_t = typename RawT<sizeof(ST) * VEC>::type;
        typedef raw_t unaligned __attribute__((aligned(sizeof(ST))));
#pragma unroll
        for (int j = 0; j < NV; j++) {
            e[j] = __builtin_bit_cast(Elems<ST, VEC>, raw_t{0, 0, 0, 0});
            if (EXACT ? count[j] > 0 : count[j] >= VEC) {
                const raw_t raw = *reinterpret_cast<const unaligned *>(p + at[j]);
                e[j] = __builtin_bit_cast(Elems<ST, VEC>, raw);
            } else if constexpr (!EXACT && L == 1) {
#pragma unroll
                for (int k = 0; k < VEC; k++)
                    if (k < count[j]) e[j].e[k] = p[at[j] + k];
            }
        }
    }
    template <typename T> __device__ __forceinline__ void store(T *p, int j, const float (&f)[VEC]) const
    {
        if (EXACT ? count[j] > 0 : count[j] >= VEC) store_some<T, VEC>(p + at[j], VEC, f);
        else if constexpr (!EXACT && L == 1) store_some<T, VEC>(p + at[j], count[j], f);
    }
    __device__ __forceinline__ void parameter(const scanscam_param &p, int64_t first, float (&f)[NV][VEC], float fill) const
    {
#pragma unroll
        for (int j = 0; j < NV; j++) params<VEC>(p, first + at[j], count[j], f[j], fill);
    }
    // A row's normalised values, in place, and 1 / sqrt(variance + eps).
    __device__ __forceinline__ float normalise(const Elems<ST, VEC> (&e)[NV], float (&h)[NV][VEC], const GroupNormArgs &args, float (*slots)[8], int &turn) const
    {
        const float share = 1.0f / (float)args.size;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                h[j][k] = (float)e[j].e[k];
                sum += EXACT || own(j, k) ? h[j][k] : 0.0f;  // (zeros where there is no channel)
            }
        const float mean = over_team<L, WAVES>(sum, args.waves, slots, turn) * share;
        sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                h[j][k] -= mean;
                const float mine = own(j, k) ? h[j][k] : 0.0f;
                sum = __builtin_fmaf(mine, mine, sum);
            }
        const float rstd = __builtin_amdgcn_rsqf(over_team<L, WAVES>(sum, args.waves, slots, turn) * share + args.a.eps);
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int k = 0; k < VEC; k++) h[j][k] *= rstd;
        return rstd;
    }
};

template <typename ST, int L, int NV, bool WAVES, bool EXACT> __global__ __launch_bounds__(WAVES ? 512 : 256) void group_norm_kernel(GroupNormArgs args)
{
    using T = Team<ST, L, NV, WAVES, EXACT>;
    constexpr int VEC = T::VEC;
    __shared__ float slots[2][8];
    const scanscam_group_norm &a = args.a;
    const T team(args);
    if (!team.there) return;
    int turn = 0;
    const int64_t first = team.group * args.size;
    float w[NV][VEC], b[NV][VEC];
    team.parameter(a.weight, first, w, 1.0f);
    team.parameter(a.bias, first, b, 0.0f);
    const ST *x = static_cast<const ST *>(a.x) + first, *z = static_cast<const ST *>(a.z) + (a.z != nullptr ? first : 0);
    ST *y = static_cast<ST *>(a.y) + first;
    Elems<ST, VEC> ex[NV], ez[NV];
    const auto ask = [&](int64_t r) {
        team.load(x + r * a.x_stride, ex);
        if (a.z != nullptr) team.load(z + r * a.z_stride, ez);
    };
    ask(team.part);
    for (int64_t r = team.part; r < a.rows; r += args.parts) {
        float h[NV][VEC], gate[NV][VEC];
        if (a.z != nullptr) {
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int k = 0; k < VEC; k++) gate[j][k] = (float)ez[j].e[k];
        }
        Elems<ST, VEC> now[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) now[j] = ex[j];
        if (r + args.parts < a.rows) ask(r + args.parts);
        team.normalise(now, h, args, slots, turn);
#pragma unroll
        for (int j = 0; j < NV; j++) {
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                float u = __builtin_fmaf(h[j][k], w[j][k], b[j][k]);
                if (a.activation == SCANSCAM_ACT_SILU) u *= sigmoid_(u);
                if (a.z != nullptr) u *= gate[j][k] * sigmoid_(gate[j][k]);
                h[j][k] = u;
            }
            team.store(y + r * a.channels, j, h[j]);
        }
    }
}

template <typename ST, int L, int NV, bool WAVES, bool EXACT> __global__ __launch_bounds__(WAVES ? 512 : 256) void group_norm_back_kernel(GroupNormArgs args)
{
    using T = Team<ST, L, NV, WAVES, EXACT>;
    constexpr int VEC = T::VEC;
    __shared__ float slots[2][8];
    const scanscam_group_norm &a = args.a;
    const T team(args);
    if (!team.there) return;
    int turn = 0;
    const int64_t first = team.group * args.size;
    float w[NV][VEC], b[NV][VEC], gw[NV][VEC], gb[NV][VEC];
    team.parameter(a.weight, first, w, 1.0f);
    team.parameter(a.bias, first, b, 0.0f);
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int k = 0; k < VEC; k++) gw[j][k] = gb[j][k] = 0.0f;
    const ST *x = static_cast<const ST *>(a.x) + first, *z = static_cast<const ST *>(a.z) + (a.z != nullptr ? first : 0), *gy = static_cast<const ST *>(a.gy) + first;
    ST *gx = static_cast<ST *>(a.gx) + first, *gz = static_cast<ST *>(a.gz) + (a.gz != nullptr ? first : 0);
    const float share = 1.0f / (float)args.size;
    Elems<ST, VEC> ex[NV], ez[NV], eg[NV];
    const auto ask = [&](int64_t r) {
        team.load(x + r * a.x_stride, ex);
        team.load(gy + r * a.channels, eg);
        if (a.z != nullptr) team.load(z + r * a.z_stride, ez);
    };
    ask(team.part);
    for (int64_t r = team.part; r < a.rows; r += args.parts) {
        float h[NV][VEC], g[NV][VEC], s[NV][VEC];
        Elems<ST, VEC> now[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            now[j] = ex[j];
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                g[j][k] = (float)eg[j].e[k];
                if (a.z != nullptr) s[j][k] = (float)ez[j].e[k];
            }
        }
        if (r + args.parts < a.rows) ask(r + args.parts);
        const float rstd = team.normalise(now, h, args, slots, turn);
        float sum = 0.0f, along = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                const float u = __builtin_fmaf(h[j][k], w[j][k], b[j][k]), su = a.activation == SCANSCAM_ACT_SILU ? sigmoid_(u) : 1.0f;
                float e = g[j][k];
                if (a.z != nullptr) {
                    const float zv = s[j][k], sz = sigmoid_(zv);
                    s[j][k] = e * (u * su) * silu_slope(zv, sz);  // from here on the gate's gradient
                    e *= zv * sz;
                }
                if (a.activation == SCANSCAM_ACT_SILU) e *= silu_slope(u, su);
                gw[j][k] = __builtin_fmaf(e, h[j][k], gw[j][k]);
                gb[j][k] += e;
                g[j][k] = e *= w[j][k];
                const float mine = team.own(j, k) ? e : 0.0f;
                sum += mine;
                along = __builtin_fmaf(mine, h[j][k], along);
            }
            if (a.gz != nullptr) team.store(gz + r * a.channels, j, s[j]);
        }
        sum = over_team<L, WAVES>(sum, args.waves, slots, turn) * share;
        along = over_team<L, WAVES>(along, args.waves, slots, turn) * share;
#pragma unroll
        for (int j = 0; j < NV; j++) {
#pragma unroll
            for (int k = 0; k < VEC; k++) g[j][k] = rstd * (g[j][k] - sum - h[j][k] * along);
            team.store(gx + r * a.channels, j, g[j]);
        }
    }
    const int64_t columns = a.gweight != nullptr ? a.channels : 0, pitch = columns + (a.gbias != nullptr ? a.channels : 0);
    if (pitch == 0) return;
    float *part = args.part + team.part * pitch + first;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if (a.gweight != nullptr) team.store(part, j, gw[j]);
        if (a.gbias != nullptr) team.store(part + columns, j, gb[j]);
    }
}

struct GroupNormPlan {
    int lanes, nv, waves;  // of a team: lanes of a wave, vectors a lane, waves
};

// One per storage type, in a file of its own.
template <typename ST> hipError_t launch_group_norm(bool back, const GroupNormPlan &plan, hipStream_t stream, const GroupNormArgs &args);

template <typename ST, int L, int NV, bool WAVES, bool EXACT> hipError_t launch_team(bool back, hipStream_t stream, const GroupNormArgs &args)
{
    const int64_t teams = args.a.groups * args.parts, grid = WAVES ? teams : ceil_div(teams, 256 / L);
    return launch_op(back ? group_norm_back_kernel<ST, L, NV, WAVES, EXACT> : group_norm_kernel<ST, L, NV, WAVES, EXACT>, dim3((unsigned)grid), dim3(WAVES ? 64 * args.waves : 256), 0,
                     stream, args);
}
template <typename ST, bool EXACT> hipError_t launch_group_norm_of(bool back, const GroupNormPlan &plan, hipStream_t stream, const GroupNormArgs &args)
{
    if (plan.waves > 1) return launch_team<ST, 64, group_most<ST>(), true, EXACT>(back, stream, args);
    if (plan.nv > 1) return launch_team<ST, 64, 2, false, EXACT>(back, stream, args);
    switch (plan.lanes) {
    case 1: return launch_team<ST, 1, 1, false, EXACT>(back, stream, args);
    case 2: return launch_team<ST, 2, 1, false, EXACT>(back, stream, args);
    case 4: return launch_team<ST, 4, 1, false, EXACT>(back, stream, args);
    case 8: return launch_team<ST, 8, 1, false, EXACT>(back, stream, args);
    case 16: return launch_team<ST, 16, 1, false, EXACT>(back, stream, args);
    case 32: return launch_team<ST, 32, 1, false, EXACT>(back, stream, args);
    default: return launch_team<ST, 64, 1, false, EXACT>(back, stream, args);
    }
}
template <typename ST> hipError_t launch_group_norm_with(bool back, const GroupNormPlan &plan, hipStream_t stream, const GroupNormArgs &args)
{
    return args.size % group_vec<ST>() == 0 ? launch_group_norm_of<ST, true>(back, plan, stream, args) : launch_group_norm_of<ST, false>(back, plan, stream, args);
}
#define SCANSCAM_DEFINE_GROUP_NORM_LAUNCH(ST)                                                                                                      \
    template <> hipError_t launch_group_norm<ST>(bool back, const GroupNormPlan &plan, hipStream_t stream, const GroupNormArgs &args)              \
    {                                                                                                                                              \
        return launch_group_norm_with<ST>(back, plan, stream, args);                                                                               \
    }

}  // namespace scanscam
