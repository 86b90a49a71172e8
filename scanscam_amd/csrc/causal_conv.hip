// The short causal convolution of every channel with its own K taps, its gradients, and its form for single tokens.
//
//   p[t] = bias + sum_k w[k] x[t - (K-1) + k],   y = act(p)         (x before a sequence: state_in, or 0)
//   gp = gy act'(p);   gx[t] = sum_k w[k] gp[t + (K-1) - k];   gw[k] = sum_t gp[t] x[t - (K-1) + k];   gbias = sum_t gp
//
// Memory bounds it: x in, y out (backwards x and gy in, gx out). A lane owns a 16-byte vector of neighbouring channels and
// walks over a stretch of time with the last K - 1 inputs in registers, so that an element is loaded once but for the K - 1 at
// the border of two stretches, which the caches still hold. A lane whose vector would reach past the last channel takes
// the last whole one instead and does some of its neighbour's work again, the same (fewer channels than a vector's go
// element by element); tokens are asked for several at a time, as one token's latency is longer than its arithmetic. [8, 4096, 2048] in bf16
// with K = 4: 53 us forwards (268 MB, 5.1 TB/s). 8021 packed tokens, 66 MB: 26 us from memory, 20 from the caches, where a wave's stretch of 8 tokens is a search for
// its sequence and three trips to memory; with the first tokens asked for before the search it took 23, with two groups under way
// at once 24: both cost registers and so waves.
#include "ops_common.hpp"

namespace scanscam {

struct ConvArgs {
    scanscam_conv a;
    float *part;      // backward: [stretches][K + 1][channels] sums of gp x and of gp
    int64_t stretch;  // tokens of a lane
    int64_t stretches;
    int64_t unit0;    // the first unit of this launch: a stretch of a batch element, or a sequence's state
};

__device__ __forceinline__ float act_(float p, int kind) { return kind == SCANSCAM_ACT_SILU ? p * sigmoid_(p) : p; }
__device__ __forceinline__ float act_slope(float p, int kind)
{
    if (kind != SCANSCAM_ACT_SILU) return 1.0f;
    const float s = sigmoid_(p);
    return s * __builtin_fmaf(p, 1.0f - s, 1.0f);
}

// The sequence at token t of batch element b: its number, first token and the one after its last. Packed tokens that belong to
// no sequence (offsets that do not start at 0 or end at T) count as the next or the last one's.
struct Span { int64_t seq, start, end; };
__device__ __forceinline__ Span span_at(const scanscam_conv &a, int64_t b, int64_t t)
{
    if (a.offsets == nullptr) return {b, 0, a.T};
    const int64_t s = sequence_of(a.offsets, a.offsets64, a.sequences, t);
    const int64_t start = clamp_(index_at(a.offsets, a.offsets64, s), 0, t);
    int64_t end = index_at(a.offsets, a.offsets64, s + 1);
    if (end <= t || end > a.T || s == a.sequences - 1) end = a.T;
    return {s, start, end};
}

// One input row of a sequence, `at` tokens after its start (at < 0: its state), as this lane's vector.
template <typename ST, int VEC>
__device__ __forceinline__ void conv_input(const scanscam_conv &a, int64_t b, const Span &s, int64_t at, int K, int64_t c, int count,
                                           float (&f)[VEC])
{
    if (at >= 0) {
        load_part(static_cast<const ST *>(a.x.p) + b * a.x.batch + (s.start + at) * a.x.token + c, count, f);
    } else if (a.state_in != nullptr) {
        load_part(static_cast<const ST *>(a.state_in) + (s.seq * (K - 1) + (K - 1) + at) * a.channels + c, count, f);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) f[i] = 0.0f;
    }
}

// Tokens asked for at a time.
constexpr int kAhead = 4;

// kAhead rows of a tensor from token t on (those past its end: the last one again), asked for without a wait between them.
template <typename ST, int VEC>
__device__ __forceinline__ void ask(Stored<ST, VEC> (&rows)[kAhead], const ST *from, int64_t stride, int64_t t, int64_t T)
{
#pragma unroll
    for (int j = 0; j < kAhead; j++) rows[j].load(from + (t + j < T ? t + j : T - 1) * stride);
}

// This lane's vector of channels: the first one, and how many there are (VEC but where there are fewer channels than that).
template <int VEC> __device__ __forceinline__ int64_t lane_channels(int64_t channels, int64_t c, int &count)
{
    count = channels < VEC ? (int)channels : VEC;
    return c < channels - count ? c : channels - count;
}

// Taps and bias of a lane's channels.
template <int VEC, int K> struct Taps {
    float w[VEC * K], bias[VEC];
    __device__ __forceinline__ void load(const scanscam_param &weight, const scanscam_param &b, int64_t c, int count)
    {
        params(weight, c * K, count * K, w);
        params(b, c, count, bias);
    }
    __device__ __forceinline__ float operator()(int i, int k) const { return w[i * K + k]; }
};

template <typename ST, int K>
__global__ __launch_bounds__(256) void conv_fwd_kernel(ConvArgs args)
{
    constexpr int VEC = 16 / sizeof(ST);
    const scanscam_conv &a = args.a;
    const int64_t mine = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    if (mine >= a.channels) return;
    int count;
    const int64_t c = lane_channels<VEC>(a.channels, mine, count);
    const int64_t unit = args.unit0 + (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int64_t walks = a.batch * args.stretches;
    if (unit >= walks) {  // the states after the last tokens
        const int64_t s = unit - walks;
        if (s >= a.sequences || a.state_out == nullptr) return;
        Span q{s, 0, a.T};
        int64_t b = s;
        if (a.offsets != nullptr) {
            b = 0;
            q.start = clamp_(index_at(a.offsets, a.offsets64, s), 0, a.T);
            q.end = clamp_(index_at(a.offsets, a.offsets64, s + 1), q.start, a.T);
        }
        for (int k = 0; k < K - 1; k++) {
            float f[VEC];
            conv_input<ST, VEC>(a, b, q, q.end - q.start - (K - 1) + k, K, c, count, f);
            store_some(static_cast<ST *>(a.state_out) + (s * (K - 1) + k) * a.channels + c, count, f);
        }
        return;
    }
    const int64_t b = unit / args.stretches, t0 = (unit - b * args.stretches) * args.stretch;
    const int64_t t1 = t0 + args.stretch < a.T ? t0 + args.stretch : a.T;
    if (t0 >= t1) return;
    Taps<VEC, K> taps;
    taps.load(a.weight, a.bias, c, count);
    const ST *from = static_cast<const ST *>(a.x.p) + b * a.x.batch + c;
    ST *to = static_cast<ST *>(a.y.p) + b * a.y.batch + c;
    float x[K][VEC];  // x[k]: the input that tap k reads
    const auto token = [&](int64_t t) {  // x[K - 1] is there
        float y[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            y[i] = taps.bias[i];
#pragma unroll
            for (int k = 0; k < K; k++) y[i] = __builtin_fmaf(taps(i, k), x[k][i], y[i]);
            y[i] = act_(y[i], a.activation);
        }
        store_some(to + t * a.y.token, count, y);
#pragma unroll
        for (int k = 0; k + 1 < K; k++) {
#pragma unroll
            for (int i = 0; i < VEC; i++) x[k][i] = x[k + 1][i];
        }
    };
    for (int64_t t = t0; t < t1;) {
        const Span s = span_at(a, b, t);
        const int64_t last = s.end < t1 ? s.end : t1;
#pragma unroll
        for (int k = 0; k < K - 1; k++) conv_input<ST, VEC>(a, b, s, t - s.start - (K - 1) + k, K, c, count, x[k]);
        for (; count == VEC && t + kAhead <= last; t += kAhead) {
            Stored<ST, VEC> ahead[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; j++) ahead[j].load(from + (t + j) * a.x.token);
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
#pragma unroll
                for (int i = 0; i < VEC; i++) x[K - 1][i] = ahead[j][i];
                token(t + j);
            }
        }
        for (; t < last; t++) {
            load_part(from + t * a.x.token, count, x[K - 1]);
            token(t);
        }
    }
}

// A stretch's gx needs gp of the K - 1 tokens after it: they are computed again. The sums for gw and gbias cover the stretch itself.
// A lane has 4 channels whatever the type: 8 of 16 bits leave two waves a SIMD, 4 leave three, and cover twice as much time in the same
// number of waves, so that fewer tokens are at a stretch's border. Those are loaded kAhead at a time as well. (A training step of
// [8, 4096, 2048] in bf16, K = 4, borders' tokens one by one / together: 8 channels and 64 tokens 159 / 155 us, 4 channels and 128 tokens
// 160 / 144, of which 87 are this kernel's: 4.6 TB/s. The next group asked for before this one is worked on: 166, for its registers.)
constexpr int kBackChannels = 4;
template <typename ST, int K>
__global__ __launch_bounds__(256, 2) void conv_bwd_kernel(ConvArgs args)
{
    constexpr int VEC = kBackChannels;
    const scanscam_conv &a = args.a;
    const int64_t mine = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    if (mine >= a.channels) return;
    int count;
    const int64_t c = lane_channels<VEC>(a.channels, mine, count);
    const int64_t unit = args.unit0 + (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (unit >= a.batch * args.stretches) {
        // Sequences without a token: the state goes through as it is.
        const int64_t s = unit - a.batch * args.stretches;
        if (s >= a.sequences || a.gstate_in == nullptr) return;
        if (a.offsets != nullptr ? index_at(a.offsets, a.offsets64, s + 1) > index_at(a.offsets, a.offsets64, s) : a.T > 0) return;
        for (int k = 0; k < K - 1; k++) {
            float f[VEC] = {};
            const int64_t at = (s * (K - 1) + k) * a.channels + c;
            if (a.gstate_out != nullptr) load_part(static_cast<const ST *>(a.gstate_out) + at, count, f);
            store_some(static_cast<ST *>(a.gstate_in) + at, count, f);
        }
        return;
    }
    const int64_t b = unit / args.stretches, t0 = (unit - b * args.stretches) * args.stretch;
    const int64_t t1 = t0 + args.stretch < a.T ? t0 + args.stretch : a.T;
    Taps<VEC, K> taps;
    taps.load(a.weight, a.bias, c, count);
    float gw[VEC * K] = {}, gb[VEC] = {};
    const ST *from = static_cast<const ST *>(a.x.p) + b * a.x.batch + c, *from_gy = static_cast<const ST *>(a.gy.p) + b * a.gy.batch + c;
    for (int64_t t = t0; t < t1;) {
        const Span s = span_at(a, b, t);
        const int64_t first = t, last = s.end < t1 ? s.end : t1, length = s.end - s.start;
        float x[K][VEC], gp[K][VEC];  // of the tokens t - (K-1) + k
#pragma unroll
        for (int k = 0; k < K - 1; k++) {
            conv_input<ST, VEC>(a, b, s, t - s.start - (K - 1) + k, K, c, count, x[k]);
#pragma unroll
            for (int i = 0; i < VEC; i++) gp[k][i] = 0.0f;  // (not needed: their gx is another stretch's, or the state's)
        }
        // gp of token t, whose x is there, from its gy; `sums`: it is the stretch's own.
        const auto slope = [&](const float (&g)[VEC], bool sums) {
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                float p = taps.bias[i];
#pragma unroll
                for (int k = 0; k < K; k++) p = __builtin_fmaf(taps(i, k), x[k][i], p);
                gp[K - 1][i] = g[i] * act_slope(p, a.activation);
            }
            if (!sums) return;
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                gb[i] += gp[K - 1][i];
#pragma unroll
                for (int k = 0; k < K; k++) gw[i * K + k] = __builtin_fmaf(gp[K - 1][i], x[k][i], gw[i * K + k]);
            }
        };
        // The input K - 1 tokens back has met all its taps.
        const auto input_gradient = [&](float (&g)[VEC]) {
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                g[i] = 0.0f;
#pragma unroll
                for (int k = 0; k < K; k++) g[i] = __builtin_fmaf(taps(i, K - 1 - k), gp[k][i], g[i]);
            }
        };
        const auto move_on = [&]() {
#pragma unroll
            for (int k = 0; k + 1 < K; k++) {
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    x[k][i] = x[k + 1][i];
                    gp[k][i] = gp[k + 1][i];
                }
            }
        };
        // Any token: at the borders of stretches and sequences.
        const auto token = [&](const Stored<ST, VEC> &x_row, const Stored<ST, VEC> &gy_row) {
            if (t < s.end) {
                float g[VEC];
                if (count == VEC) {
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        x[K - 1][i] = x_row[i];
                        g[i] = gy_row[i];
                    }
                } else {
                    load_part(from + t * a.x.token, count, x[K - 1]);
                    load_part(from_gy + t * a.gy.token, count, g);
                }
                slope(g, t < last);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i++) gp[K - 1][i] = 0.0f;
            }
            const int64_t at = t - (K - 1) - s.start;  // counted from the sequence's start; the state's rows are below 0
            const bool own = t - (K - 1) >= first, state = at < 0 && first == s.start;
            if (own || (state && a.gstate_in != nullptr)) {
                float g[VEC];
                input_gradient(g);
                const int64_t kept = at - (length - (K - 1));  // its row of the state after the sequence, if it is one
                if (kept >= 0 && a.gstate_out != nullptr) {
                    float more[VEC];
                    load_part(static_cast<const ST *>(a.gstate_out) + (s.seq * (K - 1) + kept) * a.channels + c, count, more);
#pragma unroll
                    for (int i = 0; i < VEC; i++) g[i] += more[i];
                }
                if (own) store_some(static_cast<ST *>(a.gx.p) + b * a.gx.batch + (t - (K - 1)) * a.gx.token + c, count, g);
                else store_some(static_cast<ST *>(a.gstate_in) + (s.seq * (K - 1) + (K - 1) + at) * a.channels + c, count, g);
            }
            move_on();
        };
        // The first K - 1 tokens and the last: theirs are asked for kAhead at a time too.
        const auto border = [&](int64_t stop) {
#pragma unroll 1
            while (t < stop) {
                Stored<ST, VEC> ahead[kAhead], ahead_gy[kAhead];
                if (count == VEC) {
                    ask(ahead, from, a.x.token, t, a.T);
                    ask(ahead_gy, from_gy, a.gy.token, t, a.T);
                }
                int64_t n = stop - t < kAhead ? stop - t : kAhead;
#pragma unroll 1
                for (; n > 0; n--, t++) {
                    token(ahead[0], ahead_gy[0]);
#pragma unroll
                    for (int q = 0; q + 1 < kAhead; q++) {
                        ahead[q] = ahead[q + 1];
                        ahead_gy[q] = ahead_gy[q + 1];
                    }
                }
            }
        };
        border(first + K - 1 < last + K - 1 ? first + K - 1 : last + K - 1);
        // Tokens inside the stretch whose gx goes out to K - 1 tokens back, a token's row of its own, kept by no state.
        ST *to = static_cast<ST *>(a.gx.p) + b * a.gx.batch + c;
        for (; count == VEC && t + kAhead <= last; t += kAhead) {
            Stored<ST, VEC> ahead[kAhead], ahead_gy[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                ahead[j].load(from + (t + j) * a.x.token);
                ahead_gy[j].load(from_gy + (t + j) * a.gy.token);
            }
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                float g[VEC];
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    x[K - 1][i] = ahead[j][i];
                    g[i] = ahead_gy[j][i];
                }
                slope(g, true);
                input_gradient(g);
                store_some(to + (t + j - (K - 1)) * a.gx.token, count, g);
                move_on();
            }
        }
        border(last + K - 1);
        t = last;
    }
    float *part = args.part + unit * (K + 1) * a.channels;
#pragma unroll
    for (int i = 0; i < VEC; i++) {
        if (i >= count) break;
#pragma unroll
        for (int k = 0; k < K; k++) part[(c + i) * K + k] = gw[i * K + k];
        part[(int64_t)K * a.channels + c + i] = gb[i];
    }
}

// A lane's vector of one row: the window moves on by a token. 512 rows of 2048 channels in bf16, K = 4, 17 MB: 7 us where other
// states are stepped in between, 6 where the same ones are and stay in the caches; mostly a launch and one trip to memory.
// (PART: one of several launches, whose place only they look up.)
template <typename ST, int K, bool PART>
__global__ __launch_bounds__(256) void conv_step_kernel(StepPart<scanscam_conv_step> args)
{
    const scanscam_conv_step &a = args.a;
    constexpr int VEC = 16 / sizeof(ST);
    const int64_t c = ((int64_t)((PART ? args.block0 : 0) + blockIdx.y) * blockDim.x + threadIdx.x) * VEC;
    const int64_t row = (PART ? args.row0 : 0) + (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (c >= a.channels || row >= a.rows) return;
    const int count = (int)clamp_(a.channels - c, 0, VEC);  // (no lane does another's work again here: the state is read and written in place)
    const int64_t slot = a.slot != nullptr ? index_at(a.slot, a.slot64, row) : row;
    float y[VEC] = {};
    if (slot >= 0 && slot < a.slots) {
        ST *state = static_cast<ST *>(a.state) + slot * (K - 1) * a.channels + c;
        const ST *from = static_cast<const ST *>(a.x.p) + row * a.x.token + c;
        Taps<VEC, K> taps;
        float x[K][VEC];
        if (count == VEC) {
            Stored<ST, VEC> ahead[K];
#pragma unroll
            for (int k = 0; k < K - 1; k++) ahead[k].load(state + (int64_t)k * a.channels);
            ahead[K - 1].load(from);
            taps.load(a.weight, a.bias, c, count);
#pragma unroll
            for (int k = 0; k < K; k++) {
#pragma unroll
                for (int i = 0; i < VEC; i++) x[k][i] = ahead[k][i];
            }
        } else {
#pragma unroll
            for (int k = 0; k < K - 1; k++) load_part(state + (int64_t)k * a.channels, count, x[k]);
            load_part(from, count, x[K - 1]);
            taps.load(a.weight, a.bias, c, count);
        }
#pragma unroll
        for (int k = 0; k < K - 1; k++) store_some(state + (int64_t)k * a.channels, count, x[k + 1]);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            y[i] = taps.bias[i];
#pragma unroll
            for (int k = 0; k < K; k++) y[i] = __builtin_fmaf(taps(i, k), x[k][i], y[i]);
            y[i] = act_(y[i], a.activation);
        }
    }
    store_some(static_cast<ST *>(a.y.p) + row * a.y.token + c, count, y);
}

}  // namespace scanscam

namespace {

using namespace scanscam;

constexpr int64_t kMostConvTaps = 8;

int check_conv_sizes(int64_t channels, int64_t K, int dtype, int activation)
{
    if (channels < 0 || channels > kMostChannels || K < 1 || K > kMostConvTaps) return SCANSCAM_EINVAL;
    if (activation != SCANSCAM_ACT_NONE && activation != SCANSCAM_ACT_SILU) return SCANSCAM_EINVAL;
    return activation_size(dtype) == 0 ? SCANSCAM_EDTYPE : SCANSCAM_OK;
}

int check_conv(const scanscam_conv *a)
{
    if (a == nullptr) return SCANSCAM_EINVAL;
    SCANSCAM_CHECK(check_conv_sizes(a->channels, a->K, a->dtype, a->activation));
    if (a->batch < 0 || a->T < 0 || a->T >= kMostTokens || a->batch >= kMostTokens || a->sequences < 0 || a->sequences >= kMostTokens)
        return SCANSCAM_EINVAL;
    if (a->offsets != nullptr ? a->batch != 1 || a->sequences < 1 : a->sequences != a->batch) return SCANSCAM_EINVAL;
    if (a->batch > 0 && a->T > (kMostTokens - 1) / a->batch) return SCANSCAM_EINVAL;
    if (a->channels == 0) return SCANSCAM_OK;
    SCANSCAM_CHECK(check_param(a->weight, true));
    SCANSCAM_CHECK(check_param(a->bias, false));
    if (a->offsets != nullptr && misaligned(a->offsets, a->offsets64 ? 8 : 4)) return SCANSCAM_EALIGN;
    const size_t size = (size_t)activation_size(a->dtype);
    if (misaligned(a->state_in, size) || misaligned(a->state_out, size) || misaligned(a->gstate_in, size) || misaligned(a->gstate_out, size))
        return SCANSCAM_EALIGN;
    return SCANSCAM_OK;
}

struct ConvPlan {
    int64_t stretch, stretches, units;
    dim3 block;
    unsigned blocks;  // of channels
};

// Stretches of up to 64 tokens (backwards 128: their borders cost more), shorter where there are too few to give every SIMD two waves.
ConvPlan conv_plan(const scanscam_conv &a, bool back, bool states)
{
    const int64_t vec = back ? kBackChannels : 16 / activation_size(a.dtype), lanes = ceil_div(a.channels, vec);
    ConvPlan p;
    p.stretch = back ? 128 : 64;
    while (p.stretch > 8 && ceil_div(lanes * a.batch * ceil_div(a.T, p.stretch), 64) < 2048) p.stretch /= 2;
    p.stretches = ceil_div(a.T, p.stretch);
    int x = 1;
    while (x < 256 && x < lanes) x *= 2;
    const int y = 256 / x;
    p.units = a.batch * p.stretches + (states ? a.sequences : 0);
    p.block = dim3(x, y);
    p.blocks = (unsigned)ceil_div(lanes, x);
    return p;
}

// A launch has fewer than 2^32 threads along each of its dimensions: more units than that are several launches.
template <typename ST, int K> hipError_t run_conv(ConvArgs args, const ConvPlan &p, bool back, hipStream_t stream)
{
    const int64_t most = ((int64_t(1) << 32) / p.block.x - 1) * p.block.y;
    hipError_t err = hipSuccess;
    for (; args.unit0 < p.units && err == hipSuccess; args.unit0 += most) {
        const int64_t now = p.units - args.unit0 < most ? p.units - args.unit0 : most;
        const dim3 grid((unsigned)ceil_div(now, p.block.y), p.blocks);
        err = back ? launch_op(conv_bwd_kernel<ST, K>, grid, p.block, 0, stream, args) : launch_op(conv_fwd_kernel<ST, K>, grid, p.block, 0, stream, args);
    }
    return err;
}
template <typename ST> hipError_t run_conv(const ConvArgs &args, const ConvPlan &p, bool back, hipStream_t stream)
{
    switch (args.a.K) {
    case 1: return run_conv<ST, 1>(args, p, back, stream);
    case 2: return run_conv<ST, 2>(args, p, back, stream);
    case 3: return run_conv<ST, 3>(args, p, back, stream);
    case 4: return run_conv<ST, 4>(args, p, back, stream);
    case 5: return run_conv<ST, 5>(args, p, back, stream);
    case 6: return run_conv<ST, 6>(args, p, back, stream);
    case 7: return run_conv<ST, 7>(args, p, back, stream);
    default: return run_conv<ST, 8>(args, p, back, stream);
    }
}
hipError_t run_conv(const ConvArgs &args, const ConvPlan &p, bool back, hipStream_t stream)
{
    switch (args.a.dtype) {
    case SCANSCAM_F32: return run_conv<float>(args, p, back, stream);
    case SCANSCAM_BF16: return run_conv<__bf16>(args, p, back, stream);
    default: return run_conv<_Float16>(args, p, back, stream);
    }
}

template <typename ST> hipError_t run_step(const scanscam_conv_step &a, int64_t blocks, dim3 block, hipStream_t stream)
{
    switch (a.K) {
    case 1: return launch_step(conv_step_kernel<ST, 1, false>, conv_step_kernel<ST, 1, true>, a.rows, blocks, block, stream, a);
    case 2: return launch_step(conv_step_kernel<ST, 2, false>, conv_step_kernel<ST, 2, true>, a.rows, blocks, block, stream, a);
    case 3: return launch_step(conv_step_kernel<ST, 3, false>, conv_step_kernel<ST, 3, true>, a.rows, blocks, block, stream, a);
    case 4: return launch_step(conv_step_kernel<ST, 4, false>, conv_step_kernel<ST, 4, true>, a.rows, blocks, block, stream, a);
    case 5: return launch_step(conv_step_kernel<ST, 5, false>, conv_step_kernel<ST, 5, true>, a.rows, blocks, block, stream, a);
    case 6: return launch_step(conv_step_kernel<ST, 6, false>, conv_step_kernel<ST, 6, true>, a.rows, blocks, block, stream, a);
    case 7: return launch_step(conv_step_kernel<ST, 7, false>, conv_step_kernel<ST, 7, true>, a.rows, blocks, block, stream, a);
    default: return launch_step(conv_step_kernel<ST, 8, false>, conv_step_kernel<ST, 8, true>, a.rows, blocks, block, stream, a);
    }
}

}  // namespace

extern "C" {

int scanscam_conv_fwd(const scanscam_conv *a, void *stream)
{
    SCANSCAM_CHECK(check_conv(a));
    const bool states = a->state_out != nullptr && a->K > 1;
    if (a->channels == 0 || (a->batch * a->T == 0 && !states)) return SCANSCAM_OK;
    if (a->batch * a->T > 0) {
        const int size = activation_size(a->dtype);
        SCANSCAM_CHECK(check_tokens(a->x, size));
        SCANSCAM_CHECK(check_tokens(a->y, size));
    }
    const ConvPlan p = conv_plan(*a, false, states);
    const hipError_t err = run_conv({*a, nullptr, p.stretch, p.stretches, 0}, p, false, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
}

size_t scanscam_conv_workspace_bytes(const scanscam_conv *a)
{
    if (check_conv_sizes(a != nullptr ? a->channels : -1, a != nullptr ? a->K : 0, a != nullptr ? a->dtype : 0, 0) != SCANSCAM_OK ||
        a->batch <= 0 || a->T <= 0 || a->channels == 0)
        return 0;
    const ConvPlan p = conv_plan(*a, true, false);
    return (size_t)(a->batch * p.stretches * (a->K + 1) * a->channels) * sizeof(float);
}

int scanscam_conv_bwd(const scanscam_conv *a, void *stream)
{
    SCANSCAM_CHECK(check_conv(a));
    if (a->channels == 0) return SCANSCAM_OK;
    if (a->gweight == nullptr) return SCANSCAM_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool tokens = a->batch * a->T > 0, states = a->gstate_in != nullptr && a->K > 1;
    if (tokens) {
        const int size = activation_size(a->dtype);
        SCANSCAM_CHECK(check_tokens(a->x, size));
        SCANSCAM_CHECK(check_tokens(a->gy, size));
        SCANSCAM_CHECK(check_tokens(a->gx, size));
        if (a->workspace == nullptr || a->workspace_bytes < scanscam_conv_workspace_bytes(a)) return SCANSCAM_EWORKSPACE;
        if (misaligned(a->workspace, 16)) return SCANSCAM_EALIGN;
    }
    const ConvPlan p = conv_plan(*a, true, states);
    float *part = static_cast<float *>(a->workspace);
    hipError_t err = run_conv({*a, part, p.stretch, p.stretches, 0}, p, true, s);
    const int64_t parts = a->batch * p.stretches, wide = a->K * a->channels, pitch = wide + a->channels;
    if (err == hipSuccess) err = column_sum({part, parts, pitch, {a->gweight, a->gbias}, {wide, a->channels}}, s);
    return err == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
}

int scanscam_conv_step_fwd(const scanscam_conv_step *a, void *stream)
{
    if (a == nullptr) return SCANSCAM_EINVAL;
    SCANSCAM_CHECK(check_conv_sizes(a->channels, a->K, a->dtype, a->activation));
    if (a->rows < 0 || a->rows >= kMostTokens || a->slots < 0) return SCANSCAM_EINVAL;
    if (a->rows == 0 || a->channels == 0) return SCANSCAM_OK;
    const int size = activation_size(a->dtype);
    SCANSCAM_CHECK(check_tokens(a->x, size));
    SCANSCAM_CHECK(check_tokens(a->y, size));
    SCANSCAM_CHECK(check_param(a->weight, true));
    SCANSCAM_CHECK(check_param(a->bias, false));
    if (a->K > 1 && a->state == nullptr) return SCANSCAM_EINVAL;
    if (misaligned(a->state, (size_t)size) || misaligned(a->slot, a->slot64 ? 8 : 4)) return SCANSCAM_EALIGN;
    const int64_t lanes = ceil_div(a->channels, 16 / size);
    int x = 1;
    while (x < 256 && x < lanes) x *= 2;
    const dim3 block(x, 256 / x);
    const int64_t blocks = ceil_div(lanes, x);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t err = a->dtype == SCANSCAM_F32    ? run_step<float>(*a, blocks, block, s)
                           : a->dtype == SCANSCAM_BF16 ? run_step<__bf16>(*a, blocks, block, s)
                                                       : run_step<_Float16>(*a, blocks, block, s);
    return err == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
}

}  // extern "C"
