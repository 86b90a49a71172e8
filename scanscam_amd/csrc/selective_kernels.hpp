// The selective scan over whole sequences and its gradients.
//
//   d = softplus(dt + bias) (or dt + bias);  u = d x
//   h[t][n] = e[t][n] h[t-1][n] + u[t] B[t][n],  e = exp(d A[n]);   v[t] = sum_n C[t][n] h[t][n];   y = (v + D x) silu(z)
//
// and with g0 = gy silu(z), going back in time,
//
//   G[t][n] = g0[t] C[t][n] + e[t+1][n] G[t+1][n]
//   gC[t][n] = sum_c g0 h[t][n];  gB[t][n] = sum_c u G[t][n];  s1 = sum_n G B;  s2 = sum_n A (e G h[t-1])
//   gx = d s1 + D g0;  gd = x s1 + s2;  gA[n] = sum_t d e G h[t-1];  gD = sum_t g0 x;  gz = gy (v + D x) silu'(z)
//
// Layout of the work. A row of 16 lanes holds K neighbouring tokens a lane of one channel, so that a wave scans TILE = 16 K
// tokens of 4 channels at once: each lane folds its K tokens into one affine map, the 16 maps are scanned with DPP row shifts
// (4 steps that stay inside a row, so channels never mix), and each lane replays its tokens from its carry. A tile's last lane hands
// the state on through LDS. All N states of a channel are taken one after the other by the same lanes, which keeps d, u and
// the sum over n in registers, and B and C, the same for all channels, come from LDS. What a token costs once (softplus, the gate,
// rounding) is done by other lanes on the way between the channel-fastest tensors and the token-fastest rows in LDS.
//
// The vector unit bounds it: per token, channel and state one exponential (two issue slots) and five multiply-adds forwards,
// with N = 16 some 130 slots for 8 bytes of 16-bit tensors.
#pragma once

#include "ops_common.hpp"

namespace scanscam {

constexpr int kTimeLanes = 16;   // lanes of a row: tokens of one channel
constexpr int kRows = 4;         // channels of a wave
constexpr int kStateBlock = 16;  // states whose B and C are in LDS at a time

struct SelectiveArgs {
    scanscam_selective a;
    int split;        // waves that share the states of a channel out among them
    int64_t blocks;   // of channels, in a group
};

// What follows from K. Tokens lie in LDS as [K / 4][16 lanes][4], 4 floats of padding behind each 64, so that the 16-byte reads of
// neighbouring lanes are neighbours and the single writes of a wave spread over the banks.
template <int K> struct Geometry {
    static constexpr int kTile = kTimeLanes * K;
    static constexpr int kLine = 68;
    static constexpr int kPitch = K / 4 * kLine + (K / 4 % 4 == 1 ? 0 : K / 4 % 4 == 2 ? 12 : K / 4 % 4 == 3 ? 8 : 4);
    static __device__ __forceinline__ int place(int t) { return (t % K) / 4 * kLine + t / K * 4 + (t & 3); }
    static __device__ __forceinline__ void read(const float *row, int lane, float (&f)[K])
    {
#pragma unroll
        for (int j = 0; j < K / 4; j++) {
            const float4v q = *reinterpret_cast<const float4v *>(row + j * kLine + lane * 4);
#pragma unroll
            for (int i = 0; i < 4; i++) f[4 * j + i] = q[i];
        }
    }
    static __device__ __forceinline__ void write(float *row, int lane, const float (&f)[K])
    {
#pragma unroll
        for (int j = 0; j < K / 4; j++)
            *reinterpret_cast<float4v *>(row + j * kLine + lane * 4) = float4v{f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]};
    }
};

// A scan step over affine maps h -> a h + b inside rows of 16 lanes: lanes without a source are left as they are (their a is
// finite, see finite_).
template <int CTRL> __device__ __forceinline__ void row_step(float &a, float &b)
{
    const float a1 = dpp_move<CTRL, 0xf>(1.0f, a), b1 = dpp_move<CTRL, 0xf>(0.0f, b);
    b = __builtin_fmaf(a, b1, b);
    a = a * a1;
}
// Inclusive over ascending lanes (FORWARDS) or descending ones.
template <bool FORWARDS> __device__ __forceinline__ void row_scan(float &a, float &b)
{
    if constexpr (FORWARDS) {
        row_step<0x111>(a, b);
        row_step<0x112>(a, b);
        row_step<0x114>(a, b);
        row_step<0x118>(a, b);
    } else {
        row_step<0x101>(a, b);
        row_step<0x102>(a, b);
        row_step<0x104>(a, b);
        row_step<0x108>(a, b);
    }
}
__device__ __forceinline__ float row_prev(float v, float fill) { return dpp_move<0x111, 0xf>(fill, v); }
__device__ __forceinline__ float row_next(float v, float fill) { return dpp_move<0x101, 0xf>(fill, v); }
__device__ __forceinline__ float row_sum(float v)
{
    v += dpp_move<0x111, 0xf>(0.0f, v);
    v += dpp_move<0x112, 0xf>(0.0f, v);
    v += dpp_move<0x114, 0xf>(0.0f, v);
    v += dpp_move<0x118, 0xf>(0.0f, v);
    return v;  // in lane 15
}
// A lane's whole decay. It multiplies zeros where a lane has no source: an overflow (growing states only) must not make those NaN.
__device__ __forceinline__ float finite_(float a) { return __builtin_fminf(a, __FLT_MAX__); }

// The stretch of tokens that a workgroup goes through.
struct Stretch {
    int64_t seq, batch, start, end;
};
__device__ __forceinline__ Stretch stretch_of(const scanscam_selective &a, int64_t unit)
{
    if (a.offsets == nullptr) return {unit, unit, 0, a.T};
    const int64_t start = clamp_(index_at(a.offsets, a.offsets64, unit), 0, a.T);
    return {unit, 0, start, clamp_(index_at(a.offsets, a.offsets64, unit + 1), start, a.T)};
}
// Tiles of the stretches before this one, for `saved`: a sequence of L tokens has at most L / TILE + 1 of them.
template <int TILE> __device__ __forceinline__ int64_t first_tile(const scanscam_selective &a, const Stretch &s)
{
    if (a.offsets == nullptr) return s.seq * ((a.T + TILE - 1) / TILE);
    return s.start / TILE + s.seq;
}
__host__ __device__ inline int64_t all_tiles(const scanscam_selective &a, int64_t tile)
{
    return a.offsets == nullptr ? a.sequences * ceil_div(a.T, tile) : a.T / tile + a.sequences;
}

template <typename ST>
__device__ __forceinline__ const ST *token_at(const scanscam_tokens &x, int64_t batch, int64_t t, int64_t c)
{
    return static_cast<const ST *>(x.p) + batch * x.batch + t * x.token + c;
}

// ---------------------------------------------------------------------------------------------------------------------------
// Forwards. A workgroup of 8 waves takes 8 / split groups of 4 channels through a stretch, tile by tile.
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int kFwdWaves = 8;

template <int K> struct ForwardLds {
    using G = Geometry<K>;
    static constexpr int kRowsOut = kFwdWaves * kRows;  // channels x split: rows of sums over n
    // floats: d and u of the channels, sums, B and C; then A and the carries of all states
    static __host__ __device__ constexpr int words(int channels, int N)
    {
        return 2 * channels * G::kPitch + kRowsOut * G::kPitch + 2 * kStateBlock * G::kPitch + 2 * channels * N;
    }
};

template <typename ST, int K>
__global__ __launch_bounds__(kFwdWaves * 64) void selective_fwd_kernel(SelectiveArgs args)
{
    using G = Geometry<K>;
    constexpr int TILE = G::kTile, P = G::kPitch;
    constexpr int kThreads = kFwdWaves * 64, kItems = kFwdWaves * TILE / kThreads;  // groups of 4 channels x tokens, a thread
    const scanscam_selective &a = args.a;
    const int N = (int)a.N, split = args.split, sets = kFwdWaves / split, channels = sets * kRows;
    extern __shared__ float lds[];
    float *ld = lds, *lu = ld + channels * P, *ly = lu + channels * P, *lB = ly + kFwdWaves * kRows * P, *lC = lB + kStateBlock * P;
    float *lA = lC + kStateBlock * P, *lh = lA + channels * N;  // [N][channels] each

    const int64_t per_group = a.channels / a.groups;
    const int64_t group = blockIdx.x / args.blocks, c0 = (blockIdx.x - group * args.blocks) * channels;  // c0: inside the group
    const int here = (int)clamp_(per_group - c0, 0, channels);
    const int64_t first = group * per_group + c0;  // first channel
    const Stretch s = stretch_of(a, blockIdx.y);

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, row = lane >> 4, tl = lane & 15;
    const int set = wave / split, part = wave % split;
    const int ch = set * kRows + row;

    for (int i = threadIdx.x; i < channels * N; i += kThreads) {
        const int n = i / channels, c = i - n * channels;
        const bool there = c < here;
        const int64_t at = (first + c) * N + n;
        lA[i] = there ? param(a.A, at) * kLog2e : 0.0f;
        lh[i] = there && a.state_in != nullptr ? a.state_in[s.seq * a.channels * N + at] : 0.0f;
    }

    // This thread's items on the way in and out: 4 channels at one token each.
    const int set_in = threadIdx.x % sets, c_in = set_in * kRows, count = (int)clamp_(here - c_in, 0, 4);
    float bias[4], skip[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        bias[i] = i < count ? param(a.dt_bias, first + c_in + i) : 0.0f;
        skip[i] = i < count ? param(a.D, first + c_in + i) : 0.0f;
    }
    int64_t tile = first_tile<TILE>(a, s);
    for (int64_t t0 = s.start; t0 < s.end; t0 += TILE, tile++) {
        const int length = (int)(s.end - t0 < TILE ? s.end - t0 : TILE);
        float x[kItems][4], z[kItems][4];
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const int t = threadIdx.x / sets + j * (kThreads / sets);
            if (t >= TILE) continue;
            float d[4];
            const bool there = t < length && count > 0;
#pragma unroll
            for (int i = 0; i < 4; i++) x[j][i] = z[j][i] = d[i] = 0.0f;
            if (there) {
                load_part(token_at<ST>(a.x, s.batch, t0 + t, first + c_in), count, x[j]);
                load_part(token_at<ST>(a.dt, s.batch, t0 + t, first + c_in), count, d);
                if (a.z.p != nullptr) load_part(token_at<ST>(a.z, s.batch, t0 + t, first + c_in), count, z[j]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // (tokens past the end and channels that are not there: no decay, nothing added)
                d[i] = there && i < count ? (a.softplus ? softplus_(d[i] + bias[i]) : d[i] + bias[i]) : 0.0f;
                ld[(c_in + i) * P + G::place(t)] = d[i];
                lu[(c_in + i) * P + G::place(t)] = d[i] * x[j][i];
            }
        }
        float y[K] = {};
        for (int n0 = 0; n0 < N; n0 += kStateBlock) {
            const int states = N - n0 < kStateBlock ? N - n0 : kStateBlock;
            if (n0 > 0) __syncthreads();
            for (int i = threadIdx.x; i < TILE * kStateBlock; i += kThreads) {
                const int n = i % kStateBlock, t = i / kStateBlock;
                const bool there = t < length && n < states;
                lB[n * P + G::place(t)] = there ? (float)token_at<ST>(a.B, s.batch, t0 + t, group * a.B.group + n0 + n)[0] : 0.0f;
                lC[n * P + G::place(t)] = there ? (float)token_at<ST>(a.C, s.batch, t0 + t, group * a.C.group + n0 + n)[0] : 0.0f;
            }
            __syncthreads();
            if (n0 == 0 && a.saved != nullptr) {
                // The states that this tile starts from, [tile][N][channels]; the barriers around keep them from moving on.
                float *to = static_cast<float *>(a.saved) + tile * N * a.channels + first;
                for (int i = threadIdx.x; i < channels * N; i += kThreads) {
                    const int n = i / channels, c = i - n * channels;
                    if (c < here) to[(int64_t)n * a.channels + c] = lh[i];
                }
                __syncthreads();
            }
            float d[K], u[K], total = 0.0f;
            G::read(ld + ch * P, tl, d);
            G::read(lu + ch * P, tl, u);
#pragma unroll
            for (int k = 0; k < K; k++) total += d[k];
            for (int n = part; n < states; n += split) {
                float *carry = lh + (n0 + n) * channels + ch;
                const float A = lA[(n0 + n) * channels + ch], h0 = *carry;
                float e[K], b[K];
                G::read(lB + n * P, tl, b);
                float h = tl == 0 ? h0 : 0.0f;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    e[k] = __builtin_amdgcn_exp2f(d[k] * A);
                    b[k] *= u[k];
                    h = __builtin_fmaf(e[k], h, b[k]);
                }
                float decay = finite_(__builtin_amdgcn_exp2f(total * A));
                row_scan<true>(decay, h);
                if (tl == kTimeLanes - 1) *carry = h;
                h = row_prev(h, h0);
                float C[K];
                G::read(lC + n * P, tl, C);
#pragma unroll
                for (int k = 0; k < K; k++) {
                    h = __builtin_fmaf(e[k], h, b[k]);
                    y[k] = __builtin_fmaf(C[k], h, y[k]);
                }
            }
        }
        G::write(ly + (part * channels + ch) * P, tl, y);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const int t = threadIdx.x / sets + j * (kThreads / sets);
            if (t >= length || count <= 0) continue;
            float out[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float v = skip[i] * x[j][i];
                for (int q = 0; q < split; q++) v += ly[(q * channels + c_in + i) * P + G::place(t)];
                out[i] = a.z.p != nullptr ? v * (z[j][i] * sigmoid_(z[j][i])) : v;
            }
            store_some(const_cast<ST *>(token_at<ST>(a.y, s.batch, t0 + t, first + c_in)), count, out);
        }
    }
    if (a.state_out == nullptr) return;
    __syncthreads();
    for (int i = threadIdx.x; i < channels * N; i += kThreads) {
        const int c = i / N, n = i - c * N;
        if (c < here) a.state_out[(s.seq * a.channels + first + c) * N + n] = lh[n * channels + c];
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Backwards. A workgroup of 4 waves takes 16 channels back through a stretch. The sums over n (s1, s2, v) belong to a channel, the
// sums over channels (gB, gC) to a state: a wave keeps the latter for its 4 of 16 states in registers while it goes over the
// 4 groups of channels, and the former are added up in LDS, where in every step each group of channels is one wave's alone.
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int kBwdWaves = 4, kBwdChannels = kBwdWaves * kRows, kBwdStates = kStateBlock / kBwdWaves;

struct BackwardArgs {
    SelectiveArgs f;
    float *bc;     // [blocks of all groups][tokens][2][N]: sums of gB and gC over a workgroup's channels
    float *sums;   // [stretches][channels][N + 2]: sums over a stretch's tokens for A, D and dt_bias
};

template <int K> struct BackwardLds {
    using G = Geometry<K>;
    // d, u, g0 and s1, s2, v; B and C; A, the states' and the gradients' carries and the sums for A
    static __host__ __device__ constexpr int words(int N)
    {
        return 6 * kBwdChannels * G::kPitch + 2 * kStateBlock * G::kPitch + 4 * kBwdChannels * N;
    }
};

template <typename ST, int K>
__global__ __launch_bounds__(kBwdWaves * 64) void selective_bwd_kernel(BackwardArgs args)
{
    using G = Geometry<K>;
    constexpr int TILE = G::kTile, P = G::kPitch, channels = kBwdChannels;
    constexpr int kThreads = kBwdWaves * 64, kItems = kBwdWaves * TILE / kThreads;
    const scanscam_selective &a = args.f.a;
    const int N = (int)a.N;
    extern __shared__ float lds[];
    float *ld = lds, *lu = ld + channels * P, *lg = lu + channels * P;
    float *l1 = lg + channels * P, *l2 = l1 + channels * P, *lv = l2 + channels * P;
    float *lB = lv + channels * P, *lC = lB + kStateBlock * P;
    float *lA = lC + kStateBlock * P, *lh = lA + channels * N, *lG = lh + channels * N, *lS = lG + channels * N;  // [N][channels]

    const int64_t per_group = a.channels / a.groups;
    const int64_t group = blockIdx.x / args.f.blocks, c0 = (blockIdx.x - group * args.f.blocks) * channels;
    const int here = (int)clamp_(per_group - c0, 0, channels);
    const int64_t first = group * per_group + c0;
    const Stretch s = stretch_of(a, blockIdx.y);
    const bool gated = a.z.p != nullptr;

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, row = lane >> 4, tl = lane & 15;

    for (int i = threadIdx.x; i < channels * N; i += kThreads) {
        const int n = i / channels, c = i - n * channels;
        const bool there = c < here;
        const int64_t at = (first + c) * N + n;
        lA[i] = there ? param(a.A, at) * kLog2e : 0.0f;
        lG[i] = there && a.gstate_out != nullptr ? a.gstate_out[s.seq * a.channels * N + at] : 0.0f;
        lS[i] = 0.0f;
    }

    const int set_in = threadIdx.x % kBwdWaves, c_in = set_in * kRows, count = (int)clamp_(here - c_in, 0, 4);
    float bias[4], skip[4], sum_skip[4] = {}, sum_bias[4] = {};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        bias[i] = i < count ? param(a.dt_bias, first + c_in + i) : 0.0f;
        skip[i] = i < count ? param(a.D, first + c_in + i) : 0.0f;
    }
    const int64_t tiles = (s.end - s.start + TILE - 1) / TILE;
    for (int64_t tile = tiles - 1; tile >= 0; tile--) {
        const int64_t t0 = s.start + tile * TILE;
        const int length = (int)(s.end - t0 < TILE ? s.end - t0 : TILE);
        const float *from = static_cast<const float *>(a.saved) + (first_tile<TILE>(a, s) + tile) * N * a.channels + first;
        __syncthreads();
        for (int i = threadIdx.x; i < channels * N; i += kThreads) {
            const int n = i / channels, c = i - n * channels;
            lh[i] = c < here ? from[(int64_t)n * a.channels + c] : 0.0f;
        }
        float x[kItems][4], raw[kItems][4], d[kItems][4], z[kItems][4], gy[kItems][4];
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const int t = threadIdx.x / kBwdWaves + j * (kThreads / kBwdWaves);
            const bool there = t < length && count > 0;
#pragma unroll
            for (int i = 0; i < 4; i++) x[j][i] = raw[j][i] = z[j][i] = gy[j][i] = 0.0f;
            if (there) {
                load_part(token_at<ST>(a.x, s.batch, t0 + t, first + c_in), count, x[j]);
                load_part(token_at<ST>(a.dt, s.batch, t0 + t, first + c_in), count, raw[j]);
                load_part(token_at<ST>(a.gy, s.batch, t0 + t, first + c_in), count, gy[j]);
                if (gated) load_part(token_at<ST>(a.z, s.batch, t0 + t, first + c_in), count, z[j]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                raw[j][i] += bias[i];
                d[j][i] = there && i < count ? (a.softplus ? softplus_(raw[j][i]) : raw[j][i]) : 0.0f;
                const int at = (c_in + i) * P + G::place(t);
                ld[at] = d[j][i];
                lu[at] = d[j][i] * x[j][i];
                lg[at] = gated ? gy[j][i] * (z[j][i] * sigmoid_(z[j][i])) : gy[j][i];
                l1[at] = l2[at] = lv[at] = 0.0f;
            }
        }
        for (int n0 = 0; n0 < N; n0 += kStateBlock) {
            const int states = N - n0 < kStateBlock ? N - n0 : kStateBlock;
            if (n0 > 0) __syncthreads();
            for (int i = threadIdx.x; i < TILE * kStateBlock; i += kThreads) {
                const int n = i % kStateBlock, t = i / kStateBlock;
                const bool there = t < length && n < states;
                lB[n * P + G::place(t)] = there ? (float)token_at<ST>(a.B, s.batch, t0 + t, group * a.B.group + n0 + n)[0] : 0.0f;
                lC[n * P + G::place(t)] = there ? (float)token_at<ST>(a.C, s.batch, t0 + t, group * a.C.group + n0 + n)[0] : 0.0f;
            }
            float gB[kBwdStates][K] = {}, gC[kBwdStates][K] = {};
            for (int step = 0; step < kBwdWaves; step++) {
                __syncthreads();
                const int ch = ((wave + step) % kBwdWaves) * kRows + row;
                float d[K], u[K], g0[K], s1[K], s2[K], v[K], total = 0.0f;
                G::read(ld + ch * P, tl, d);
                G::read(lu + ch * P, tl, u);
                G::read(lg + ch * P, tl, g0);
                G::read(l1 + ch * P, tl, s1);
                G::read(l2 + ch * P, tl, s2);
                G::read(lv + ch * P, tl, v);
#pragma unroll
                for (int k = 0; k < K; k++) total += d[k];
#pragma unroll
                for (int q = 0; q < kBwdStates; q++) {
                    const int n = wave * kBwdStates + q;
                    if (n >= states) continue;
                    const int at = (n0 + n) * channels + ch;
                    const float A = lA[at], h0 = lh[at], G0 = lG[at];
                    float e[K], h[K], B[K], C[K];
                    G::read(lB + n * P, tl, B);
                    G::read(lC + n * P, tl, C);
                    float fold = tl == 0 ? h0 : 0.0f, back = tl == kTimeLanes - 1 ? G0 : 0.0f;
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        e[k] = __builtin_amdgcn_exp2f(d[k] * A);
                        h[k] = u[k] * B[k];
                        fold = __builtin_fmaf(e[k], fold, h[k]);
                    }
#pragma unroll
                    for (int k = K - 1; k >= 0; k--) back = e[k] * __builtin_fmaf(g0[k], C[k], back);
                    const float decay = finite_(__builtin_amdgcn_exp2f(total * A));
                    float a1 = decay, a2 = decay;
                    row_scan<true>(a1, fold);
                    row_scan<false>(a2, back);
                    if (tl == 0) lG[at] = back;
                    const float before = row_prev(fold, h0);
                    float g = row_next(back, G0);
                    float state = before;
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        state = __builtin_fmaf(e[k], state, h[k]);
                        h[k] = state;
                        v[k] = __builtin_fmaf(C[k], state, v[k]);
                        gC[q][k] = __builtin_fmaf(g0[k], state, gC[q][k]);
                    }
                    float sum = 0.0f;
#pragma unroll
                    for (int k = K - 1; k >= 0; k--) {
                        g = __builtin_fmaf(g0[k], C[k], g);  // G[t]
                        gB[q][k] = __builtin_fmaf(u[k], g, gB[q][k]);
                        s1[k] = __builtin_fmaf(B[k], g, s1[k]);
                        g *= e[k];
                        const float r = g * (k > 0 ? h[k - 1] : before);
                        s2[k] = __builtin_fmaf(A, r, s2[k]);
                        sum = __builtin_fmaf(d[k], r, sum);
                    }
                    sum = row_sum(sum);
                    if (tl == kTimeLanes - 1) lS[at] += sum;
                }
                G::write(l1 + ch * P, tl, s1);
                G::write(l2 + ch * P, tl, s2);
                G::write(lv + ch * P, tl, v);
            }
            // gB and gC over the 4 channels of the rows: lanes 0-15 end up with the first, ... of every four values.
#pragma unroll
            for (int q = 0; q < kBwdStates; q++) {
                const int n = wave * kBwdStates + q;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    float b = gB[q][k], c = gC[q][k];
                    b += __shfl_xor(b, 16);
                    b += __shfl_xor(b, 32);
                    c += __shfl_xor(c, 16);
                    c += __shfl_xor(c, 32);
                    const int t = tl * K + k;
                    if (row == 0 && n < states && t < length) {
                        float *to = args.bc + (((int64_t)blockIdx.x * a.batch + s.batch) * a.T + t0 + t) * 2 * N + n0 + n;
                        to[0] = b;
                        to[N] = c;
                    }
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const int t = threadIdx.x / kBwdWaves + j * (kThreads / kBwdWaves);
            if (t >= length || count <= 0) continue;
            float gx[4], gd[4], gz[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = (c_in + i) * P + G::place(t);
                const float s1 = l1[at], s2 = l2[at] * (1.0f / kLog2e), v = lv[at] + skip[i] * x[j][i], g0 = lg[at];
                gx[i] = __builtin_fmaf(d[j][i], s1, skip[i] * g0);
                gd[i] = __builtin_fmaf(x[j][i], s1, s2);
                if (a.softplus) gd[i] *= sigmoid_(raw[j][i]);
                sum_skip[i] = __builtin_fmaf(g0, x[j][i], sum_skip[i]);
                sum_bias[i] += gd[i];
                const float sg = sigmoid_(z[j][i]);
                gz[i] = gy[j][i] * v * (sg * __builtin_fmaf(z[j][i], 1.0f - sg, 1.0f));
            }
            store_some(const_cast<ST *>(token_at<ST>(a.gx, s.batch, t0 + t, first + c_in)), count, gx);
            store_some(const_cast<ST *>(token_at<ST>(a.gdt, s.batch, t0 + t, first + c_in)), count, gd);
            if (gated) store_some(const_cast<ST *>(token_at<ST>(a.gz, s.batch, t0 + t, first + c_in)), count, gz);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < channels * N; i += kThreads) {
        const int c = i / N, n = i - c * N;
        if (c >= here) continue;
        const int64_t at = (s.seq * a.channels + first + c) * N + n;
        if (a.gstate_in != nullptr) a.gstate_in[at] = lG[n * channels + c];
        args.sums[(s.seq * (N + 2)) * a.channels + (first + c) * N + n] = lS[n * channels + c];
    }
    // D's and the bias's: over the threads of a channel, through the tokens' rows (64 threads a set of 4 channels).
    __syncthreads();
    float *red = lds;  // [64][2][channels]
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int t = threadIdx.x / kBwdWaves;
        red[(t * 2 + 0) * channels + c_in + i] = sum_skip[i];
        red[(t * 2 + 1) * channels + c_in + i] = sum_bias[i];
    }
    __syncthreads();
    if (threadIdx.x < 2 * channels) {
        const int which = threadIdx.x / channels, c = threadIdx.x % channels;
        float sum = 0.0f;
        for (int t = 0; t < 64; t++) sum += red[(t * 2 + which) * channels + c];
        if (c < here) args.sums[(s.seq * (N + 2) + N + which) * a.channels + first + c] = sum;
    }
}

// gB and gC: the sums of the workgroups of a group of channels, in order.
struct GroupSum {
    scanscam_selective a;
    const float *bc;
    int64_t blocks;
};
template <typename ST>
__global__ __launch_bounds__(256) void selective_bc_kernel(GroupSum args)
{
    const scanscam_selective &a = args.a;
    const int64_t wide = 2 * a.N, tokens = a.batch * a.T;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, group = blockIdx.y;
    if (i >= tokens * wide) return;
    const int64_t token = i / wide;
    int64_t n = i - token * wide;
    const float *from = args.bc + group * args.blocks * tokens * wide + i;
    float sum = 0.0f;
    for (int64_t b = 0; b < args.blocks; b++) sum += from[b * tokens * wide];
    const scanscam_tokens &to = n < a.N ? a.gB : a.gC;
    if (n >= a.N) n -= a.N;
    const int64_t batch = token / a.T;
    const_cast<ST *>(token_at<ST>(to, batch, token - batch * a.T, group * to.group + n))[0] = (ST)sum;
}

// ---------------------------------------------------------------------------------------------------------------------------
// One token: LANES lanes a channel, each with 4 neighbouring states at a time.
// ---------------------------------------------------------------------------------------------------------------------------
template <typename ST, int LANES>
__global__ __launch_bounds__(256) void selective_step_kernel(scanscam_selective_step a)
{
    const int lane = threadIdx.x % LANES, N = (int)a.N;
    const int64_t c = (int64_t)blockIdx.y * (256 / LANES) + threadIdx.x / LANES, row = blockIdx.x;
    const int64_t slot = a.slot != nullptr ? index_at(a.slot, a.slot64, row) : row;
    const bool there = c < a.channels;
    if (slot < 0 || slot >= a.slots) {
        if (there && lane == 0) const_cast<ST *>(token_at<ST>(a.y, 0, row, c))[0] = (ST)0.0f;
        return;
    }
    float y = 0.0f, x = 0.0f;
    if (there) {
        const int64_t group = c / (a.channels / a.groups);
        x = (float)token_at<ST>(a.x, 0, row, c)[0];
        float d = (float)token_at<ST>(a.dt, 0, row, c)[0] + param(a.dt_bias, c);
        if (a.softplus) d = softplus_(d);
        const ST *B = token_at<ST>(a.B, 0, row, group * a.B.group), *C = token_at<ST>(a.C, 0, row, group * a.C.group);
        float *state = a.state + (slot * a.channels + c) * N;
        for (int n0 = lane * 4; n0 < N; n0 += LANES * 4) {
            const int count = N - n0 < 4 ? N - n0 : 4;
            float h[4], b[4], w[4];
            load_part(state + n0, count, h);
            load_part(B + n0, count, b);
            load_part(C + n0, count, w);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (i >= count) break;
                const float A = param(a.A, c * N + n0 + i);
                h[i] = __builtin_fmaf(exp_(d * A), h[i], d * x * b[i]);
                y = __builtin_fmaf(w[i], h[i], y);
            }
            store_some(state + n0, count, h);
        }
    }
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) y += __shfl_xor(y, m);
    if (there && lane == 0) {
        y = __builtin_fmaf(param(a.D, c), x, y);
        if (a.z.p != nullptr) {
            const float z = (float)token_at<ST>(a.z, 0, row, c)[0];
            y *= z * sigmoid_(z);
        }
        const_cast<ST *>(token_at<ST>(a.y, 0, row, c))[0] = (ST)y;
    }
}

}  // namespace scanscam
