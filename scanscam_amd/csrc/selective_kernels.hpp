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
// The vector unit bounds it. Forwards a lane's 8 tokens take 74 issue slots a state (65 instructions; 9 exponentials take two), of which 56
// are the formula's: 148 a token and channel at N = 16, with 63 more for what a token costs once, for 8 bytes of 16-bit tensors.
// Backwards they take 171 a state, 342 a token and channel, with 162 more. At 2.4 GHz and 4 cycles a slot that is 360 and 860 us for
// [8, 4096, 2048] with N = 16; in bf16 with the gate it takes 371 us forwards (2.9e12 states a second, 1.6 TB/s) and 1075 backwards, where
// two waves a SIMD (256 registers, 80 KB of LDS a workgroup) leave a fifth of the slots empty. More waves of 4 tokens a lane were
// slower: they scan twice as often.
#pragma once

#include "ops_common.hpp"

namespace scanscam {

constexpr int kTimeLanes = 16;   // lanes of a row: tokens of one channel
constexpr int kRows = 4;         // channels of a wave
constexpr int kStateBlock = 16;  // states whose B and C are in LDS at a time

// What follows from K. Tokens lie in LDS as [K / 4][16 lanes][4], 4 floats of padding behind each 64, so that the 16-byte reads of
// neighbouring lanes are neighbours and the single writes of a wave spread over the banks: the pitch is 4 or 12 modulo 16, which
// sends the 4 groups of channels that a wave writes to different quarters of them.
template <int K> struct Geometry {
    static constexpr int kTile = kTimeLanes * K;
    static constexpr int kLine = 68;
    static constexpr int kPitch = K / 4 * kLine + (K / 4 % 2 == 1 ? 0 : 4);
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

// Inclusive scan over affine maps h -> a h + b inside rows of 16 lanes, over ascending lanes (FORWARDS) or descending ones, as
// DPP operands of the multiply-add itself: b += a' s b, a *= a' s a; a lane without a source writes nothing, so neither
// an identity nor a mask is needed and a channel never meets another one's values. Two instructions and a wait state a step; as builtins
// (moves with identities to fill) it was seven, a quarter of the forward kernel's instructions. A DPP source needs two
// wait states behind its write: the first nop covers whatever wrote a and b, the others the step before.
#define SCANSCAM_ROW_STEP(DIR, N)                                                       \
    "v_fmac_f32_dpp %1, %1, %0 row_" DIR ":" N " row_mask:0xf bank_mask:0xf\n\t"       \
    "v_mul_f32_dpp %0, %0, %0 row_" DIR ":" N " row_mask:0xf bank_mask:0xf\n\t"        \
    "s_nop 0\n\t"
template <bool FORWARDS> __device__ __forceinline__ void row_scan(float &a, float &b)
{
    if constexpr (FORWARDS) {
        asm volatile("s_nop 1\n\t" SCANSCAM_ROW_STEP("shr", "1") SCANSCAM_ROW_STEP("shr", "2") SCANSCAM_ROW_STEP("shr", "4")
                     "v_fmac_f32_dpp %1, %1, %0 row_shr:8 row_mask:0xf bank_mask:0xf\n\t" "s_nop 1"
                     : "+v"(a), "+v"(b));
    } else {
        asm volatile("s_nop 1\n\t" SCANSCAM_ROW_STEP("shl", "1") SCANSCAM_ROW_STEP("shl", "2") SCANSCAM_ROW_STEP("shl", "4")
                     "v_fmac_f32_dpp %1, %1, %0 row_shl:8 row_mask:0xf bank_mask:0xf\n\t" "s_nop 1"
                     : "+v"(a), "+v"(b));
    }
}
// Both at once: each fills the other's wait states.
#define SCANSCAM_ROW_STEPS(N)                                                      \
    "v_fmac_f32_dpp %1, %1, %0 row_shr:" N " row_mask:0xf bank_mask:0xf\n\t"       \
    "v_fmac_f32_dpp %3, %3, %2 row_shl:" N " row_mask:0xf bank_mask:0xf\n\t"
#define SCANSCAM_ROW_DECAYS(N)                                                     \
    "v_mul_f32_dpp %0, %0, %0 row_shr:" N " row_mask:0xf bank_mask:0xf\n\t"        \
    "v_mul_f32_dpp %2, %2, %2 row_shl:" N " row_mask:0xf bank_mask:0xf\n\t"
__device__ __forceinline__ void row_scans(float &a, float &up, float &b, float &down)
{
    asm volatile("s_nop 1\n\t" SCANSCAM_ROW_STEPS("1") SCANSCAM_ROW_DECAYS("1") SCANSCAM_ROW_STEPS("2") SCANSCAM_ROW_DECAYS("2")
                 SCANSCAM_ROW_STEPS("4") SCANSCAM_ROW_DECAYS("4") SCANSCAM_ROW_STEPS("8") "s_nop 1"
                 : "+v"(a), "+v"(up), "+v"(b), "+v"(down));
}
#undef SCANSCAM_ROW_DECAYS
#undef SCANSCAM_ROW_STEPS
#undef SCANSCAM_ROW_STEP
__device__ __forceinline__ float row_prev(float v, float fill) { return dpp_move<0x111, 0xf>(fill, v); }
__device__ __forceinline__ float row_next(float v, float fill) { return dpp_move<0x101, 0xf>(fill, v); }
// The sums of four values over a row's lanes, in lane 15: four chains that fill each other's wait states.
__device__ __forceinline__ void row_sums(float (&v)[4])
{
#define SCANSCAM_ROW_ADDS(N)                                                       \
    "v_add_f32_dpp %0, %0, %0 row_shr:" N " row_mask:0xf bank_mask:0xf\n\t"        \
    "v_add_f32_dpp %1, %1, %1 row_shr:" N " row_mask:0xf bank_mask:0xf\n\t"        \
    "v_add_f32_dpp %2, %2, %2 row_shr:" N " row_mask:0xf bank_mask:0xf\n\t"        \
    "v_add_f32_dpp %3, %3, %3 row_shr:" N " row_mask:0xf bank_mask:0xf\n\t"
    asm volatile("s_nop 1\n\t" SCANSCAM_ROW_ADDS("1") SCANSCAM_ROW_ADDS("2") SCANSCAM_ROW_ADDS("4") SCANSCAM_ROW_ADDS("8")
                 : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
#undef SCANSCAM_ROW_ADDS
}
// The sums over the four rows of four values, the sum of value r in row r. A swap of halves puts two values' lanes behind each
// other, so that an addition serves both: six instructions, where four sums of their own take sixteen.
__device__ __forceinline__ float halves_sum(float a, float b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}
__device__ __forceinline__ float rows_sum(float v0, float v1, float v2, float v3)
{
    const float a = halves_sum(v0, v2), b = halves_sum(v1, v3);
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// The stretch of tokens that a workgroup goes through: a part of a sequence, `span` tokens (whole tiles) from its start on, one of
// `parts`. Parts are numbered through all sequences. Those of packed ones are counted from their starts, without a look at the
// sequences before: one of L tokens has at most L / span + 1 parts, so that sequence s begins with number start / span + s.
// Numbers that no part has (`part` is then past the last one) get a stretch without tokens.
struct Stretch {
    int64_t seq, batch, part, parts, unit, start, end, tile;  // unit: its number; tile: that of its first tile, for `saved`, counted likewise
    __device__ __forceinline__ bool last() const { return part == parts - 1; }
};
constexpr int64_t kWhole = int64_t(1) << 40;  // a span that cuts nothing

// The longest of up to 64 packed sequences, the next one, ...: what runs longest has to begin first (a workgroup has a sequence's
// whole time to go through). A lane has a sequence; every wave counts for each of them those that come before it.
__device__ __forceinline__ int64_t by_length(const scanscam_selective &a, int64_t unit)
{
    const int lane = threadIdx.x & 63, sequences = (int)a.sequences;
    const int at = lane < sequences ? lane : sequences - 1;
    const int length = (int)(clamp_(index_at(a.offsets, a.offsets64, at + 1), 0, a.T) - clamp_(index_at(a.offsets, a.offsets64, at), 0, a.T));
    int before = 0;
    for (int j = 0; j < sequences; j++) {
        const int other = __builtin_amdgcn_readlane(length, j);
        before += other > length || (other == length && j < lane);
    }
    return __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < sequences && before == (int)unit));
}

// `each`: the parts of a sequence where all have one length. (Numbers of parts and tiles have 32 bits, a division of 64 takes the
// hundred instructions that a short call cannot hide; only packed sequences that are cut need it.)
template <int TILE> __device__ __forceinline__ Stretch stretch_of(const scanscam_selective &a, uint32_t unit, int64_t span, uint32_t each)
{
    Stretch s;
    if (a.offsets == nullptr) {
        const uint32_t seq = each > 1 ? unit / each : unit;
        s.seq = s.batch = seq;
        s.unit = unit;
        s.part = unit - seq * each;
        s.parts = each;
        s.start = 0;
        s.end = a.T;
        s.tile = (int64_t)seq * ((a.T + TILE - 1) / TILE);
    } else if (span == kWhole) {
        s.seq = s.unit = a.sequences <= 64 ? by_length(a, unit) : unit;
        s.batch = s.part = 0;
        s.parts = 1;
        s.start = clamp_(index_at(a.offsets, a.offsets64, s.seq), 0, a.T);
        s.end = clamp_(index_at(a.offsets, a.offsets64, s.seq + 1), s.start, a.T);
        s.tile = s.start / TILE + s.seq;
    } else {
        int64_t lo = 0, hi = a.sequences - 1;  // the last sequence that begins with this number or a lower one
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) >> 1;
            if (clamp_(index_at(a.offsets, a.offsets64, mid), 0, a.T) / span + mid <= unit) lo = mid;
            else hi = mid - 1;
        }
        s.seq = lo;
        s.batch = 0;
        s.unit = unit;
        s.start = clamp_(index_at(a.offsets, a.offsets64, lo), 0, a.T);
        s.end = clamp_(index_at(a.offsets, a.offsets64, lo + 1), s.start, a.T);
        s.part = unit - s.start / span - lo;
        s.part = s.part < 0 ? 0 : s.part;
        s.parts = s.end - s.start > span ? (s.end - s.start + span - 1) / span : 1;
        s.tile = s.start / TILE + lo;
    }
    if (span != kWhole) {
        const int64_t length = s.end - s.start, from = s.part * span < length ? s.part * span : length;
        s.tile += from / TILE;
        s.start += from;
        s.end = s.start + span < s.end ? s.start + span : s.end;
    }
    return s;
}
// The numbers that there are.
__host__ __device__ inline int64_t all_units(const scanscam_selective &a, int64_t span)
{
    return a.offsets == nullptr ? a.sequences * (a.T > span ? ceil_div(a.T, span) : 1) : a.T / span + a.sequences;
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

// An element a 32-bit number of them behind a place that is the same for all lanes: an address of a scalar base and a vector offset.
template <typename ST> __device__ __forceinline__ const ST *behind(const ST *base, uint32_t elements)
{
    return reinterpret_cast<const ST *>(reinterpret_cast<const char *>(base) + (uint64_t)(uint32_t)(elements * (uint32_t)sizeof(ST)));
}
template <typename ST> __device__ __forceinline__ ST *behind(ST *base, uint32_t elements)
{
    return reinterpret_cast<ST *>(reinterpret_cast<char *>(base) + (uint64_t)(uint32_t)(elements * (uint32_t)sizeof(ST)));
}

// Four neighbouring elements as they are stored. Where not all quads of a workgroup are whole, they are read one by one, those
// past the end as the last one.
template <typename ST> struct Quad {
    ST e[4];
    using raw_t = typename RawT<sizeof(ST) * 4>::type;
    typedef raw_t raw_unaligned_t __attribute__((aligned(sizeof(ST))));
    __device__ __forceinline__ void load(const ST *base, uint32_t at, int count, bool whole)
    {
        if (whole) {
            const raw_t raw = *reinterpret_cast<const raw_unaligned_t *>(behind(base, at));
            *this = __builtin_bit_cast(Quad, raw);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) e[i] = *behind(base, at + (uint32_t)(i < count ? i : count - 1));
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return (float)e[i]; }
    // Waits here for what load() asked for.
    __device__ __forceinline__ void arrive()
    {
        raw_t raw = __builtin_bit_cast(raw_t, *this);
        asm volatile("" : "+v"(raw));
        *this = __builtin_bit_cast(Quad, raw);
    }
};
template <typename ST> __device__ __forceinline__ void store_quad(ST *base, uint32_t at, int count, bool whole, const float (&f)[4])
{
    Quad<ST> q;
#pragma unroll
    for (int i = 0; i < 4; i++) q.e[i] = (ST)f[i];
    if (whole) {
        *reinterpret_cast<typename Quad<ST>::raw_unaligned_t *>(behind(base, at)) = __builtin_bit_cast(typename Quad<ST>::raw_t, q);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < count) *behind(base, at + (uint32_t)i) = q.e[i];
    }
}

// The same value, of which the compiler does not know that it is: what is derived from it is computed again for every tile, where
// it would otherwise be kept in registers (or spilled) through the scan of one.
__device__ __forceinline__ int again(int v)
{
    asm volatile("" : "+v"(v));
    return v;
}

// What a thread brings in of B and C for a block of states: quads of neighbouring states of a token each.
template <typename ST, int TILE, int THREADS> struct StateInputs {
    static constexpr int kQuads = kStateBlock / 4, kCount = TILE * kQuads / THREADS;
    static_assert(TILE * kQuads % THREADS == 0, "every thread has as many quads");
    Quad<ST> B[kCount], C[kCount];
    __device__ __forceinline__ void load(const scanscam_selective &a, int64_t batch, int64_t group, int64_t t0, int length, int n0)
    {
        const ST *fromB = token_at<ST>(a.B, batch, t0, group * a.B.group), *fromC = token_at<ST>(a.C, batch, t0, group * a.C.group);
        const int thread = again((int)threadIdx.x), N = (int)a.N, n = n0 + thread % kQuads * 4;
        const int at = n < N ? n : 0;  // (past the last state: any that is there)
        const bool whole = N % 4 == 0;
#pragma unroll
        for (int j = 0; j < kCount; j++) {
            const int t = (thread + j * THREADS) / kQuads, row = t < length ? t : length - 1;
            B[j].load(fromB, (uint32_t)row * (uint32_t)a.B.token + (uint32_t)at, N - at, whole);
            C[j].load(fromC, (uint32_t)row * (uint32_t)a.C.token + (uint32_t)at, N - at, whole);
        }
    }
    __device__ __forceinline__ void arrive()
    {
#pragma unroll
        for (int j = 0; j < kCount; j++) {
            B[j].arrive();
            C[j].arrive();
        }
    }
    template <typename G> __device__ __forceinline__ void store(float *lB, float *lC, int length, int states) const
    {
        const int thread = again((int)threadIdx.x), n = thread % kQuads * 4;
        const bool full = length == TILE && states == kStateBlock;
#pragma unroll
        for (int j = 0; j < kCount; j++) {
            const int t = (thread + j * THREADS) / kQuads, at = n * G::kPitch + G::place(t);
            float b[4], c[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                b[k] = B[j][k];
                c[k] = C[j][k];
            }
            if (!full) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const bool there = t < length && n + k < states;
                    b[k] = there ? b[k] : 0.0f;
                    c[k] = there ? c[k] : 0.0f;
                }
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                lB[at + k * G::kPitch] = b[k];
                lC[at + k * G::kPitch] = c[k];
            }
        }
    }
};

// Step sizes of a thread's items from what is stored: four channels at a token each. (The branches are the same for all lanes and
// stand outside of the loops, which then run without them.)
template <typename ST, int ITEMS>
__device__ __forceinline__ void step_sizes(const Quad<ST> (&dt)[ITEMS], const float (&bias)[4], bool softplus, float (&d)[ITEMS][4])
{
#pragma unroll
    for (int j = 0; j < ITEMS; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) d[j][i] = dt[j][i] + bias[i];
    if (softplus) {
#pragma unroll
        for (int j = 0; j < ITEMS; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) d[j][i] = softplus_(d[j][i]);
    }
}

struct SelectiveArgs {
    scanscam_selective a;
    int share;        // forwards: waves that share the states of a channel out among them; backwards: sets of 16 channels that a workgroup takes
    uint32_t unit0;   // the first part of this launch's
    uint32_t blocks;  // of channels, in a group
    uint32_t each;    // parts of a sequence where all are of one length
    int64_t span;     // tokens of a part of a sequence
    float *ends;      // [parts of all sequences][N + 1][channels]: the states that a part alone ends with (backwards: starts with), its sum of d
    float *bc;        // backwards: [blocks of all groups][tokens][2][N], sums of gB and gC over a workgroup's channels
    float *sums;      // backwards: [parts of all sequences][N + 2][channels], sums over a part's tokens for A, D and dt_bias
};

// Workgroups are dealt out to the 8 dies in turn, each with an L2 cache of its own, while neighbouring blocks of channels share the
// 128-byte lines of every token (a block of 16 channels of 16 bits is a quarter of one) and all of B and C: dealt out one by
// one, a line is fetched by up to four dies, and written by them in pieces. So a die takes 8 neighbours in turn. (Layer [8, 4096, 2048]
// in bf16, forwards / forwards and backwards, and packed prompts forwards, us: one by one 388 / 1558, 133; 4 in turn 381 / 1533, 126; 8
// 371 / 1522, 127; 16 377 / 1532, 127; 32 381 / 1530, 133; an eighth of all work each 388 / 1535, 170.)
struct Work {
    uint32_t block, unit;  // block of channels among all groups'; part of a sequence
};
__device__ __forceinline__ Work work_of(uint32_t blocks, uint32_t unit0)
{
    constexpr uint32_t kDies = 8, near = 8, round = near * kDies;
    uint32_t i = blockIdx.x;
    if (i < gridDim.x / round * round) i = i / round * round + i % kDies * near + i % round / kDies;
    const uint32_t unit = i / blocks;
    return {i - unit * blocks, unit0 + unit};
}

// The state before a part (the gradient behind it): that of the sequence's end, taken through the parts between. A part alone
// is the map h -> exp(A * sum of d) h + its own end.
__device__ __forceinline__ float carried(const SelectiveArgs &args, const Stretch &s, int n, int64_t channel, float A, float h, bool forwards)
{
    const scanscam_selective &a = args.a;
    const int64_t pitch = (a.N + 1) * a.channels;
    const float *ends = args.ends + (s.unit - s.part) * pitch + channel;
    if (s.part >= s.parts) return h;
    // (eight parts asked for at a time: one by one, their latencies were 11 of the 75 us of a call in 59 parts)
    const int64_t count = forwards ? s.part : s.parts - 1 - s.part, from = forwards ? 0 : s.parts - 1, step = forwards ? pitch : -pitch;
    const float *at = ends + from * pitch;
    int64_t q = 0;
    for (; q + 8 <= count; q += 8) {
        float sum[8], end[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            sum[j] = at[j * step + a.N * a.channels];
            end[j] = at[j * step + n * a.channels];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) h = __builtin_fmaf(__builtin_amdgcn_exp2f(A * sum[j]), h, end[j]);
        at += 8 * step;
    }
    for (; q < count; q++, at += step) h = __builtin_fmaf(__builtin_amdgcn_exp2f(A * at[a.N * a.channels]), h, at[n * a.channels]);
    return h;
}

// Waves that share a SIMD belong to two workgroups. One that loads, stores, exchanges or scans over lanes, which is short and full of waits,
// goes before one that is at its states' arithmetic: taken in turn, the two would come to wait at the same time. (Layer [8, 4096, 2048]
// in bf16: forwards 392 us without, 378 with; forwards and backwards 1657 and 1546.)
__device__ __forceinline__ void wave_first(bool first)
{
    if (first) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
}

struct Carry { float A, h; };  // A log2(e), and the state

// ---------------------------------------------------------------------------------------------------------------------------
// Forwards. A workgroup of 8 waves takes 8 / split groups of 4 channels through a stretch, tile by tile; the next tile's tensors
// are loaded while this one is scanned. With ENDS only the states at the stretch's end are found, from zeros: [1, 30001, 256] in fp32,
// in 59 parts, 47 us and then 66 (backwards 74 and 183, in 30).
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int kFwdWaves = 8;

template <int K> struct ForwardLds {
    using G = Geometry<K>;
    static constexpr int kSums = kFwdWaves * kRows;  // channels x split: rows of sums over n
    // floats: d and u of the channels, sums, B and C; D; A and the carries of all states; where lanes write that have nothing to say. (Of 32
    // channels 76 KB at N = 16, two workgroups a CU up to N = 39, one from 40 on: [8, 4096, 2048] in bf16 takes 621 us at N = 32, 973 at 40.)
    static __host__ __device__ constexpr int words(int channels, int N)
    {
        return 2 * channels * G::kPitch + kSums * G::kPitch + 2 * kStateBlock * G::kPitch + channels + 2 * channels * N + 2;
    }
};

template <typename ST, int K, bool ENDS>
__global__ __launch_bounds__(kFwdWaves * 64, 4) void selective_fwd_kernel(SelectiveArgs args)
{
    using G = Geometry<K>;
    constexpr int TILE = G::kTile, P = G::kPitch;
    constexpr int kThreads = kFwdWaves * 64, kItems = kFwdWaves * TILE / kThreads;  // groups of 4 channels x tokens, a thread
    const scanscam_selective &a = args.a;
    const int N = (int)a.N, split = args.share, sets = kFwdWaves / split, channels = sets * kRows;
    extern __shared__ float lds[];
    float *ld = lds, *lu = ld + channels * P, *ly = lu + channels * P, *lB = ly + kFwdWaves * kRows * P, *lC = lB + kStateBlock * P;
    float *lskip = lC + kStateBlock * P;
    Carry *lh = reinterpret_cast<Carry *>(lskip + channels), *nowhere = lh + channels * N;  // [N][channels]

    const int64_t per_group = a.groups > 1 ? (uint32_t)a.channels / (uint32_t)a.groups : a.channels;
    const Work w = work_of((uint32_t)a.groups * args.blocks, args.unit0);
    const uint32_t group = a.groups > 1 ? w.block / args.blocks : 0, c0 = (w.block - group * args.blocks) * channels;  // c0: inside the group
    const int here = (int)clamp_(per_group - c0, 0, channels);
    const int64_t first = group * per_group + c0;  // first channel
    const Stretch s = stretch_of<TILE>(a, w.unit, args.span, args.each);
    if (ENDS && s.part >= s.parts - 1) return;  // (nothing follows it)
    const bool gated = !ENDS && a.z.p != nullptr;

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, row = lane >> 4, tl = lane & 15;
    const int part = wave % split, ch = wave / split * kRows + row;

    // This thread's items on the way in and out: 4 channels at one token each. Tokens past the end and channels that are not there
    // are read from places that are, and have no decay and add nothing.
    const int set_in = threadIdx.x % sets, c_in = set_in * kRows, count = (int)clamp_(here - c_in, 0, 4);
    const int t_in = threadIdx.x / sets, t_step = kThreads / sets;
    const uint32_t c_from = count > 0 ? c_in : 0;
    const int c_count = count > 0 ? count : here;
    const bool whole = here % 4 == 0;
    float bias[4], sum_d[4] = {};
    Quad<ST> x[kItems], dt[kItems], z[kItems];
    StateInputs<ST, TILE, kThreads> bc;
    const auto fetch = [&](int64_t t0) {
        const int length = (int)(s.end - t0 < TILE ? s.end - t0 : TILE), t_mine = again(t_in);
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const uint32_t t = t_mine + j * t_step < length ? t_mine + j * t_step : length - 1;
            x[j].load(token_at<ST>(a.x, s.batch, t0, first), t * (uint32_t)a.x.token + c_from, c_count, whole);
            dt[j].load(token_at<ST>(a.dt, s.batch, t0, first), t * (uint32_t)a.dt.token + c_from, c_count, whole);
        }
        bc.load(a, s.batch, group, t0, length, 0);
    };
    const auto fetch_gate = [&](int64_t t0, int length) {
        const int t_mine = again(t_in);
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const uint32_t t = t_mine + j * t_step < length ? t_mine + j * t_step : length - 1;
            z[j].load(token_at<ST>(a.z, s.batch, t0, first), t * (uint32_t)a.z.token + c_from, c_count, whole);
        }
    };
    wave_first(true);
    if (s.start < s.end) fetch(s.start);  // (first of all: what follows waits for loads of its own)
    params(a.dt_bias, first + c_in, count, bias);
    if ((int)threadIdx.x < channels) lskip[threadIdx.x] = (int)threadIdx.x < here ? param(a.D, first + threadIdx.x) : 0.0f;
    for (int i = threadIdx.x; i < channels * N; i += kThreads) {
        const int n = i / channels, c = i - n * channels;
        Carry q{0.0f, 0.0f};
        if (c < here) {
            const int64_t at = (first + c) * N + n;
            q.A = param(a.A, at) * kLog2e;
            if (!ENDS) {
                if (a.state_in != nullptr) q.h = a.state_in[s.seq * a.channels * N + at];
                q.h = carried(args, s, n, first + c, q.A, q.h, true);
            }
        }
        lh[i] = q;
    }
    int64_t tile = s.tile;
    for (int64_t t0 = s.start; t0 < s.end; t0 += TILE, tile++) {
        const int length = (int)(s.end - t0 < TILE ? s.end - t0 : TILE);
        Quad<ST> x_now[kItems];
        const int t_mine = again(t_in);
        const bool full = length == TILE && here == channels;
        float d_in[kItems][4], u_in[kItems][4];
        step_sizes(dt, bias, a.softplus, d_in);
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            x_now[j] = x[j];
#pragma unroll
            for (int i = 0; i < 4; i++) u_in[j][i] = d_in[j][i] * x[j][i];
        }
        if (!full) {
#pragma unroll
            for (int j = 0; j < kItems; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool there = t_mine + j * t_step < length && i < count;
                    d_in[j][i] = there ? d_in[j][i] : 0.0f;
                    u_in[j][i] = there ? u_in[j][i] : 0.0f;
                }
        }
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const int t = t_mine + j * t_step, at = c_in * P + G::place(t);
            if (t >= TILE) continue;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (ENDS) sum_d[i] += d_in[j][i];
                ld[at + i * P] = d_in[j][i];
                lu[at + i * P] = u_in[j][i];
            }
        }
        float y[K] = {};
        for (int n0 = 0; n0 < N; n0 += kStateBlock) {
            const int states = N - n0 < kStateBlock ? N - n0 : kStateBlock;
            if (n0 > 0) __syncthreads();
            bc.template store<G>(lB, lC, length, states);
            __syncthreads();
            if (!ENDS && n0 == 0 && a.saved != nullptr) {
                // The states that this tile starts from, [tile][N][channels]; the barriers around keep them from moving on.
                float *to = static_cast<float *>(a.saved) + tile * N * a.channels + first;
                for (int i = threadIdx.x; i < channels * N; i += kThreads) {
                    const int n = i / channels, c = i - n * channels;
                    if (c < here) to[(int64_t)n * a.channels + c] = lh[i].h;
                }
                __syncthreads();
            }
            if (gated && n0 == 0) fetch_gate(t0, length);
            if (n0 + kStateBlock < N) bc.load(a, s.batch, group, t0, length, n0 + kStateBlock);
            else if (t0 + TILE < s.end) fetch(t0 + TILE);
            float d[K], u[K], total = 0.0f;
            G::read(ld + ch * P, tl, d);
            G::read(lu + ch * P, tl, u);
#pragma unroll
            for (int k = 0; k < K; k++) total += d[k];
            wave_first(false);
            const Carry *carry = lh + (n0 + part) * channels + ch;
            Carry *out = tl == kTimeLanes - 1 ? lh + (n0 + part) * channels + ch : nowhere;
            const int in_step = split * channels, out_step = tl == kTimeLanes - 1 ? in_step : 0;
            const float *from = lB + part * P;
            for (int n = part; n < states; n += split, carry += in_step, out += out_step, from += split * P) {
                const Carry c = *carry;
                float e[K], b[K];
                G::read(from, tl, b);
                float h = tl == 0 ? c.h : 0.0f;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    e[k] = __builtin_amdgcn_exp2f(d[k] * c.A);
                    b[k] *= u[k];
                    h = __builtin_fmaf(e[k], h, b[k]);
                }
                float decay = __builtin_amdgcn_exp2f(total * c.A);
                row_scan<true>(decay, h);
                out->h = h;
                if (ENDS) continue;
                h = row_prev(h, c.h);
                float C[K];
                G::read(from + kStateBlock * P, tl, C);
#pragma unroll
                for (int k = 0; k < K; k++) {
                    h = __builtin_fmaf(e[k], h, b[k]);
                    y[k] = __builtin_fmaf(C[k], h, y[k]);
                }
            }
        }
        wave_first(true);
        if (!ENDS) G::write(ly + (part * channels + ch) * P, tl, y);
        __syncthreads();
        if (ENDS) continue;
        // What was asked for ahead is waited for before anything is stored: a wait behind the stores would be one for them too.
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            x[j].arrive();
            dt[j].arrive();
            z[j].arrive();
        }
        bc.arrive();
        const int t_out = again(t_in);
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const int t = t_out + j * t_step;
            if (t >= length || count <= 0) continue;
            float out[4];
            const float *sums = ly + c_in * P + G::place(t);
            const float4v skip = *reinterpret_cast<const float4v *>(lskip + c_in);
#pragma unroll
            for (int i = 0; i < 4; i++) out[i] = __builtin_fmaf(skip[i], x_now[j][i], sums[i * P]);
#pragma unroll 1
            for (int q = 1; q < split; q++) {
                sums += channels * P;
#pragma unroll
                for (int i = 0; i < 4; i++) out[i] += sums[i * P];
            }
            if (gated) {
#pragma unroll
                for (int i = 0; i < 4; i++) out[i] *= z[j][i] * sigmoid_(z[j][i]);
            }
            store_quad(const_cast<ST *>(token_at<ST>(a.y, s.batch, t0, first)), (uint32_t)t * (uint32_t)a.y.token + c_from, count, whole, out);
        }
    }
    __syncthreads();
    if (ENDS) {
        float *to = args.ends + s.unit * (N + 1) * a.channels + first;
        for (int i = threadIdx.x; i < channels * N; i += kThreads) {
            const int n = i / channels, c = i - n * channels;
            if (c < here) to[(int64_t)n * a.channels + c] = lh[i].h;
        }
        // The sum of d, over the threads of a channel in order.
        float *red = lds;  // [threads a set][channels]
#pragma unroll
        for (int i = 0; i < 4; i++) red[t_in * channels + c_in + i] = sum_d[i];
        __syncthreads();
        if ((int)threadIdx.x < here) {
            float sum = 0.0f;
            for (int t = 0; t < t_step; t++) sum += red[t * channels + threadIdx.x];
            to[(int64_t)N * a.channels + threadIdx.x] = sum;
        }
    } else if (a.state_out != nullptr && s.last()) {
        for (int i = threadIdx.x; i < channels * N; i += kThreads) {
            const int c = i / N, n = i - c * N;
            if (c < here) a.state_out[(s.seq * a.channels + first + c) * N + n] = lh[n * channels + c].h;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Backwards. A workgroup of 4 waves takes 16 channels back through a stretch. The sums over n (s1, s2, v) belong to a channel, the
// sums over channels (gB, gC) to a state: a wave keeps the latter for its 4 of 16 states in registers while it goes over the
// 4 groups of channels, and the former are added up in LDS, where in every step each group of channels is one wave's alone. Of
// many channels with up to 16 states it takes two times 16, one after the other in every tile, before gB and gC go out: half
// the sums for selective_bc_kernel to join. With ENDS only the gradient at the stretch's start is found, from zeros.
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int kBwdWaves = 4, kBwdChannels = kBwdWaves * kRows, kBwdStates = kStateBlock / kBwdWaves;

constexpr int kBwdMostSets = 2;  // of 16 channels

template <int K> struct BackwardLds {
    using G = Geometry<K>;
    // d, u, g0 and s1, s2, v; B and C; A, the gradients' carries and the sums for A; a block's states; bias, D and the sums for them. (Two
    // workgroups a CU up to N = 40.)
    static __host__ __device__ constexpr int words(int N, int sets)
    {
        return 6 * kBwdChannels * G::kPitch + 2 * kStateBlock * G::kPitch + 3 * sets * kBwdChannels * padded(N) + kBwdChannels * kStateBlock +
               (2 + 2 * kBwdWaves) * sets * kBwdChannels + nowhere(sets);
    }
    // A wave goes through its states without a branch: those past the last one have no decay, no B and no C.
    static __host__ __device__ constexpr int padded(int N) { return (N + kBwdStates - 1) / kBwdStates * kBwdStates; }
    static __host__ __device__ constexpr int nowhere(int sets) { return 3 * sets * kBwdChannels * kBwdStates; }  // where lanes write that have nothing to say
};

template <typename ST, int K, bool ENDS>
__global__ __launch_bounds__(kBwdWaves * 64, 2) void selective_bwd_kernel(SelectiveArgs args)
{
    using G = Geometry<K>;
    constexpr int TILE = G::kTile, P = G::kPitch, channels = kBwdChannels;
    constexpr int kThreads = kBwdWaves * 64, kItems = kBwdWaves * TILE / kThreads;
    const scanscam_selective &a = args.a;
    const int N = (int)a.N, wide = args.share * channels, slots = wide * BackwardLds<K>::padded(N);  // wide: all channels of the workgroup
    extern __shared__ float lds[];
    float *ld = lds, *lu = ld + channels * P, *lg = lu + channels * P;
    float *l1 = lg + channels * P, *l2 = l1 + channels * P, *lv = l2 + channels * P;
    float *lB = lv + channels * P, *lC = lB + kStateBlock * P;
    Carry *lG = reinterpret_cast<Carry *>(lC + kStateBlock * P);                   // [N][wide]
    float *lS = reinterpret_cast<float *>(lG + slots), *lh = lS + slots;           // [N][wide], [16][channels]
    float *lbias = lh + channels * kStateBlock, *lskip = lbias + wide, *lsum = lskip + wide;  // lsum: [waves][2][wide]
    float *nowhere = lsum + 2 * kBwdWaves * wide;

    const int64_t per_group = a.groups > 1 ? (uint32_t)a.channels / (uint32_t)a.groups : a.channels;
    const Work w = work_of((uint32_t)a.groups * args.blocks, args.unit0);
    const uint32_t group = a.groups > 1 ? w.block / args.blocks : 0, c0 = (w.block - group * args.blocks) * wide;
    const int here = (int)clamp_(per_group - c0, 0, wide), sets = (here + channels - 1) / channels;
    const int64_t first = group * per_group + c0;
    const Stretch s = stretch_of<TILE>(a, w.unit, args.span, args.each);
    if (ENDS && (s.part == 0 || s.part >= s.parts)) return;
    const bool gated = a.z.p != nullptr;

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, row = lane >> 4, tl = lane & 15;

    const int c_in = threadIdx.x % kBwdWaves * kRows;
    const int t_in = threadIdx.x / kBwdWaves, t_step = kThreads / kBwdWaves;
    const bool whole = here % 4 == 0;
    // Channels from c_in on that set `set` has, and where they are read: those that are not there from places that are.
    const auto count_of = [&](int set) { return (int)clamp_(here - set * channels - c_in, 0, 4); };
    const int64_t tiles = (s.end - s.start + TILE - 1) / TILE;
    Quad<ST> x[kItems], dt[kItems], gy[kItems], z[kItems];
    StateInputs<ST, TILE, kThreads> bc;
    const auto fetch = [&](int64_t t0, int set) {
        const int length = (int)(s.end - t0 < TILE ? s.end - t0 : TILE), t_mine = again(t_in), have = count_of(set);
        const int count = have > 0 ? have : here - set * channels;
        const int64_t from = first + set * channels;
        const uint32_t c = have > 0 ? c_in : 0;
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const uint32_t t = t_mine + j * t_step < length ? t_mine + j * t_step : length - 1;
            x[j].load(token_at<ST>(a.x, s.batch, t0, from), t * (uint32_t)a.x.token + c, count, whole);
            dt[j].load(token_at<ST>(a.dt, s.batch, t0, from), t * (uint32_t)a.dt.token + c, count, whole);
            gy[j].load(token_at<ST>(a.gy, s.batch, t0, from), t * (uint32_t)a.gy.token + c, count, whole);
            if (gated) z[j].load(token_at<ST>(a.z, s.batch, t0, from), t * (uint32_t)a.z.token + c, count, whole);
        }
    };
    const auto fetch_bc = [&](int64_t t0, int n0) { bc.load(a, s.batch, group, t0, (int)(s.end - t0 < TILE ? s.end - t0 : TILE), n0); };
    // The states that a tile starts from, one a thread in a block of 16.
    static_assert(channels * kStateBlock == kThreads, "one a thread");
    float h_saved = 0.0f;
    const auto fetch_states = [&](int64_t tile, int set, int n0) {
        if (ENDS) return;
        const int thread = again((int)threadIdx.x), n = n0 + thread / channels, c = set * channels + thread % channels;
        const float *from = static_cast<const float *>(a.saved) + (s.tile + tile) * N * a.channels + first;
        h_saved = c < here && n < N ? *(from + (int64_t)n * a.channels + c) : 0.0f;
    };
    wave_first(true);
    if (tiles > 0) {
        fetch(s.start + (tiles - 1) * TILE, 0);
        fetch_bc(s.start + (tiles - 1) * TILE, 0);
        fetch_states(tiles - 1, 0, 0);
    }
    for (int i = threadIdx.x; i < slots; i += kThreads) {
        const int n = i / wide, c = i - n * wide;
        Carry q{0.0f, 0.0f};
        if (c < here && n < N) {
            const int64_t at = (first + c) * N + n;
            q.A = param(a.A, at) * kLog2e;
            if (!ENDS) {
                if (a.gstate_out != nullptr) q.h = a.gstate_out[s.seq * a.channels * N + at];
                q.h = carried(args, s, n, first + c, q.A, q.h, false);
            }
        }
        lG[i] = q;
        lS[i] = 0.0f;
    }

    for (int i = threadIdx.x; i < wide; i += kThreads) {
        lbias[i] = i < here ? param(a.dt_bias, first + i) : 0.0f;
        lskip[i] = i < here ? param(a.D, first + i) : 0.0f;
    }
    for (int i = threadIdx.x; i < 2 * kBwdWaves * wide; i += kThreads) lsum[i] = 0.0f;
    // What was asked for ahead is waited for before anything is stored, as in the forward kernel.
    const auto arrive = [&]() {
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            x[j].arrive();
            dt[j].arrive();
            gy[j].arrive();
            z[j].arrive();
        }
        bc.arrive();
        asm volatile("" : "+v"(h_saved));
    };
    // Whether every wave has states in the first block: then what it finds in its first step is the first there is of s1, s2 and v.
    const bool busy = N > (kBwdWaves - 1) * kBwdStates;
    for (int64_t tile = tiles - 1; tile >= 0; tile--) {
        const int64_t t0 = s.start + tile * TILE;
        const int length = (int)(s.end - t0 < TILE ? s.end - t0 : TILE);
        float gB[kBwdStates][K], gC[kBwdStates][K];
        for (int set = 0; set < sets; set++) {
        const int count = count_of(set);
        __syncthreads();
        Quad<ST> x_now[kItems], dt_now[kItems], gy_now[kItems], z_now[kItems];
        const int t_mine = again(t_in);
        const bool full = length == TILE && here - set * channels >= channels;
        const float4v bias4 = *reinterpret_cast<const float4v *>(lbias + set * channels + c_in);
        const float bias[4] = {bias4[0], bias4[1], bias4[2], bias4[3]};
        float sums_in[2][4] = {};
        float d_in[kItems][4], u_in[kItems][4], g_in[kItems][4];
        step_sizes(dt, bias, a.softplus, d_in);
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            x_now[j] = x[j];
            dt_now[j] = dt[j];
            gy_now[j] = gy[j];
            z_now[j] = z[j];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                u_in[j][i] = d_in[j][i] * x[j][i];
                g_in[j][i] = gy[j][i];
            }
        }
        if (gated) {
#pragma unroll
            for (int j = 0; j < kItems; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) g_in[j][i] *= z[j][i] * sigmoid_(z[j][i]);
        }
        if (!full) {
#pragma unroll
            for (int j = 0; j < kItems; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool there = t_mine + j * t_step < length && i < count;
                    d_in[j][i] = there ? d_in[j][i] : 0.0f;
                    u_in[j][i] = there ? u_in[j][i] : 0.0f;
                    g_in[j][i] = there ? g_in[j][i] : 0.0f;
                }
        }
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const int at = c_in * P + G::place(t_mine + j * t_step);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                ld[at + i * P] = d_in[j][i];
                lu[at + i * P] = u_in[j][i];
                lg[at + i * P] = g_in[j][i];
                if (!ENDS && !busy) l1[at + i * P] = l2[at + i * P] = lv[at + i * P] = 0.0f;
                if (ENDS) sums_in[1][i] += d_in[j][i];
            }
        }
        for (int n0 = 0; n0 < N; n0 += kStateBlock) {
            const int states = N - n0 < kStateBlock ? N - n0 : kStateBlock;
            if (n0 > 0) __syncthreads();
            if (set == 0) bc.template store<G>(lB, lC, length, states);
            if (!ENDS) lh[threadIdx.x] = h_saved;
            if (set == 0) {
#pragma unroll
                for (int q = 0; q < kBwdStates; q++)
#pragma unroll
                    for (int k = 0; k < K; k++) gB[q][k] = gC[q][k] = 0.0f;
            }
            for (int step = 0; step < kBwdWaves; step++) {
                __syncthreads();
                if (step == 0) {
                    if (n0 + kStateBlock < N) {
                        fetch_bc(t0, n0 + kStateBlock);
                        fetch_states(tile, set, n0 + kStateBlock);
                    } else if (set + 1 < sets) {
                        fetch(t0, set + 1);
                        fetch_states(tile, set + 1, 0);
                    } else if (tile > 0) {
                        fetch(t0 - TILE, 0);
                        fetch_bc(t0 - TILE, 0);
                        fetch_states(tile - 1, 0, 0);
                    }
                }
                if (wave * kBwdStates >= states) continue;
                const int ch = ((wave + step) % kBwdWaves) * kRows + row, from = (n0 + wave * kBwdStates) * wide + set * channels + ch;
                // (an address for every lane instead of a branch around the one that writes: the four states below stay one block)
                Carry *out = tl == 0 ? lG + from : reinterpret_cast<Carry *>(nowhere);
                float *sums = tl == kTimeLanes - 1 ? lS + from : nowhere + 2 * wide * kBwdStates;
                float d[K], u[K], g0[K], s1[K], s2[K], v[K], total = 0.0f;
                G::read(ld + ch * P, tl, d);
                G::read(lg + ch * P, tl, g0);
                if (!ENDS) {
                    G::read(lu + ch * P, tl, u);
                    if (busy && step == 0 && n0 == 0) {
#pragma unroll
                        for (int k = 0; k < K; k++) s1[k] = s2[k] = v[k] = 0.0f;
                    } else {
                        G::read(l1 + ch * P, tl, s1);
                        G::read(l2 + ch * P, tl, s2);
                        G::read(lv + ch * P, tl, v);
                    }
                }
#pragma unroll
                for (int k = 0; k < K; k++) total += d[k];
                float sum_A[kBwdStates];
                wave_first(false);
                static_assert(kBwdStates == 4, "row_sums takes a wave's states");
#pragma unroll
                for (int q = 0; q < kBwdStates; q++) {
                    const int n = wave * kBwdStates + q;
                    const Carry c = lG[from + q * wide];
                    float e[K], C[K];
                    G::read(lC + n * P, tl, C);
                    float back = tl == kTimeLanes - 1 ? c.h : 0.0f, a2 = __builtin_amdgcn_exp2f(total * c.A);
#pragma unroll
                    for (int k = 0; k < K; k++) e[k] = __builtin_amdgcn_exp2f(d[k] * c.A);
                    if constexpr (ENDS) {
#pragma unroll
                        for (int k = K - 1; k >= 0; k--) back = e[k] * __builtin_fmaf(g0[k], C[k], back);
                        row_scan<false>(a2, back);
                        out[q * wide].h = back;
                        continue;
                    }
                    // Forwards in time and backwards side by side: each is one chain of dependent operations.
                    float h[K], B[K];
                    G::read(lB + n * P, tl, B);
                    const float h0 = lh[(wave * kBwdStates + q) * channels + ch];
                    float fold = tl == 0 ? h0 : 0.0f, a1 = a2;
#pragma unroll
                    for (int k = 0; k < K; k++) h[k] = u[k] * B[k];
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        fold = __builtin_fmaf(e[k], fold, h[k]);
                        back = e[K - 1 - k] * __builtin_fmaf(g0[K - 1 - k], C[K - 1 - k], back);
                    }
                    wave_first(true);
                    row_scans(a1, fold, a2, back);
                    wave_first(false);
                    out[q * wide].h = back;
                    const float before = row_prev(fold, h0);
                    float g = row_next(back, c.h), state = before;
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        const int r = K - 1 - k;
                        state = __builtin_fmaf(e[k], state, h[k]);
                        g = __builtin_fmaf(g0[r], C[r], g);  // G[t]
                        h[k] = state;
                        v[k] = __builtin_fmaf(C[k], state, v[k]);
                        gC[q][k] = __builtin_fmaf(g0[k], state, gC[q][k]);
                        gB[q][r] = __builtin_fmaf(u[r], g, gB[q][r]);
                        s1[r] = __builtin_fmaf(B[r], g, s1[r]);
                        g *= e[r];
                        B[r] = g;  // e G: what G hands to the token before
                    }
                    float sum = 0.0f;
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        const float r = B[k] * (k > 0 ? h[k - 1] : before);
                        s2[k] = __builtin_fmaf(c.A, r, s2[k]);
                        sum = __builtin_fmaf(d[k], r, sum);
                    }
                    sum_A[q] = sum;
                    __builtin_amdgcn_sched_barrier(0x104);  // the next state's reads may go ahead, its arithmetic would need more registers
                }
                if (ENDS) continue;
                row_sums(sum_A);
#pragma unroll
                for (int q = 0; q < kBwdStates; q++) sums[q * wide] += sum_A[q];
                G::write(l1 + ch * P, tl, s1);
                G::write(l2 + ch * P, tl, s2);
                G::write(lv + ch * P, tl, v);
            }
            if (ENDS) continue;
            wave_first(true);
            if (set + 1 < sets) {
                __syncthreads();
                arrive();
                continue;
            }
            // gB and gC over the 4 channels of the rows, into the places of B and C (a state's are one wave's alone), and out.
#pragma unroll
            for (int q = 0; q < kBwdStates; q++) {
                const int at = (wave * kBwdStates + q) * P + tl * 4 + row;
#pragma unroll
                for (int m = 0; m < K / 4; m++) {
                    lB[at + m * G::kLine] = rows_sum(gB[q][4 * m], gB[q][4 * m + 1], gB[q][4 * m + 2], gB[q][4 * m + 3]);
                    lC[at + m * G::kLine] = rows_sum(gC[q][4 * m], gC[q][4 * m + 1], gC[q][4 * m + 2], gC[q][4 * m + 3]);
                }
            }
            __syncthreads();
            arrive();
            float *to = args.bc + (((int64_t)w.block * a.batch + s.batch) * a.T + t0) * 2 * N + n0;
            const int thread = again((int)threadIdx.x);
#pragma unroll
            for (int j = 0; j < TILE * 2 * kStateBlock / 4 / kThreads; j++) {
                const int i = thread + j * kThreads, n = i % 4 * 4, which = i / 4 % 2, t = i / 8;
                const float *from = (which ? lC : lB) + n * P + G::place(t);
                const float f[4] = {from[0], from[P], from[2 * P], from[3 * P]};
                if (t < length && n < states) store_quad(to, (uint32_t)((2 * t + which) * N + n), states - n, states - n >= 4, f);
            }
        }
        if (!ENDS) {
        const float4v skip = *reinterpret_cast<const float4v *>(lskip + set * channels + c_in);
        const int64_t from = first + set * channels;
        const int t_out = again(t_in);
#pragma unroll
        for (int j = 0; j < kItems; j++) {
            const int t = t_out + j * t_step;
            if (t >= length || count <= 0) continue;
            float gx[4], gd[4], gz[4];
            const int at = c_in * P + G::place(t);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float xi = x_now[j][i], s1 = l1[at + i * P], s2 = l2[at + i * P] * (1.0f / kLog2e), g0 = lg[at + i * P];
                gx[i] = __builtin_fmaf(ld[at + i * P], s1, skip[i] * g0);
                gd[i] = __builtin_fmaf(xi, s1, s2);
                sums_in[0][i] = __builtin_fmaf(g0, xi, sums_in[0][i]);
            }
            if (a.softplus) {
#pragma unroll
                for (int i = 0; i < 4; i++) gd[i] *= sigmoid_(dt_now[j][i] + bias[i]);
            }
            if (gated) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float zi = z_now[j][i], sg = sigmoid_(zi), v = __builtin_fmaf(skip[i], x_now[j][i], lv[at + i * P]);
                    gz[i] = gy_now[j][i] * v * (sg * __builtin_fmaf(zi, 1.0f - sg, 1.0f));
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) sums_in[1][i] += gd[i];
            store_quad(const_cast<ST *>(token_at<ST>(a.gx, s.batch, t0, from)), (uint32_t)t * (uint32_t)a.gx.token + c_in, count, whole, gx);
            store_quad(const_cast<ST *>(token_at<ST>(a.gdt, s.batch, t0, from)), (uint32_t)t * (uint32_t)a.gdt.token + c_in, count, whole, gd);
            if (gated) store_quad(const_cast<ST *>(token_at<ST>(a.gz, s.batch, t0, from)), (uint32_t)t * (uint32_t)a.gz.token + c_in, count, whole, gz);
        }
        }
        // The sums for D and the bias (ENDS: of d) over the wave's tokens: over the 4 lanes of a row that have the same channels, then over
        // the rows, which leaves channel r of every 4 in row r's last lanes.
#pragma unroll
        for (int which = ENDS ? 1 : 0; which < 2; which++) {
            float (&v)[4] = sums_in[which];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[i] += dpp_move<0x114, 0xf>(0.0f, v[i]);
                v[i] += dpp_move<0x118, 0xf>(0.0f, v[i]);
            }
            const float sum = rows_sum(v[0], v[1], v[2], v[3]);
            if (tl >= 12) lsum[(wave * 2 + which) * wide + set * channels + (tl - 12) * 4 + row] += sum;
        }
        }
    }
    __syncthreads();
    float *to = ENDS ? args.ends + s.unit * (N + 1) * a.channels + first
                     : args.sums + s.unit * (N + 2) * a.channels + first * N;
    for (int i = threadIdx.x; i < wide * N; i += kThreads) {
        if (ENDS) {
            const int n = i / wide, c = i - n * wide;
            if (c < here) to[(int64_t)n * a.channels + c] = lG[i].h;
        } else {
            const int c = i / N, n = i - c * N;
            if (c >= here) continue;
            if (a.gstate_in != nullptr && s.part == 0) a.gstate_in[(s.seq * a.channels + first + c) * N + n] = lG[n * wide + c].h;
            to[i] = lS[n * wide + c];
        }
    }
    for (int i = threadIdx.x; i < 2 * wide; i += kThreads) {
        const int which = i / wide, c = i - which * wide;
        if (c >= here) continue;
        float sum = 0.0f;
        for (int q = 0; q < kBwdWaves; q++) sum += lsum[(q * 2 + which) * wide + c];
        if (!ENDS) args.sums[(s.unit * (N + 2) + N + which) * a.channels + first + c] = sum;
        else if (which == 1) to[(int64_t)N * a.channels + c] = sum;
    }
}

// gB and gC: the sums of the workgroups of a group of channels, in order. Memory bounds it: what the workgroups wrote, read once. Eight
// loads of 16 bytes are under way at a time: [8, 4096, 2048], N = 16, 64 workgroups a token, 268 MB: 58 us, 4.6 TB/s (4 bytes a lane,
// as many loads as the compiler took together: 75).
struct GroupSum {
    scanscam_selective a;
    const float *bc;
    int64_t blocks;
    uint32_t token0, tokens, group0;  // of this launch
};
// VEC: neighbouring states of a lane, 4 where their number allows it.
template <typename ST, int VEC>
__global__ __launch_bounds__(256) void selective_bc_kernel(GroupSum args)
{
    constexpr int kTogether = 8;
    const scanscam_selective &a = args.a;
    const uint32_t wide = 2 * (uint32_t)a.N, i = (blockIdx.x * 256 + threadIdx.x) * VEC;
    const int64_t group = args.group0 + blockIdx.y;
    if (i >= args.tokens * wide) return;
    typedef float vec_t __attribute__((ext_vector_type(VEC), aligned(4)));
    const int64_t pitch = a.batch * a.T * wide;
    const float *from = args.bc + group * args.blocks * pitch + (int64_t)args.token0 * wide + i;
    vec_t sum = 0.0f;
    int64_t b = 0;
    for (; b + kTogether <= args.blocks; b += kTogether, from += kTogether * pitch) {
        vec_t v[kTogether];
#pragma unroll
        for (int j = 0; j < kTogether; j++) v[j] = *reinterpret_cast<const vec_t *>(from + j * pitch);
#pragma unroll
        for (int j = 0; j < kTogether; j++) sum += v[j];
    }
    for (; b < args.blocks; b++, from += pitch) sum += *reinterpret_cast<const vec_t *>(from);
    const uint32_t place = i / wide, token = args.token0 + place, batch = token / (uint32_t)a.T;
    uint32_t n = i - place * wide;
    const scanscam_tokens &to = n < a.N ? a.gB : a.gC;
    if (n >= a.N) n -= (uint32_t)a.N;
    float f[VEC];
#pragma unroll
    for (int k = 0; k < VEC; k++) f[k] = sum[k];
    store_some(const_cast<ST *>(token_at<ST>(to, batch, token - batch * (uint32_t)a.T, group * to.group + n)), VEC, f);
}

// ---------------------------------------------------------------------------------------------------------------------------
// One token: LANES lanes a channel, each with 4 neighbouring states at a time, so that a wave reads and writes the states, which are nearly
// all there is, in one piece; everything is asked for before any of it is used. 512 rows of 2048 channels, N = 16, bf16, 143 MB: 44 us, 3.2 TB/s,
// where other states are stepped in between; 29 us where the same 67 MB of states are stepped again, which stay in the card's cache of 256 MB.
// One row: 3 us, which are a launch and one trip to memory.
// ---------------------------------------------------------------------------------------------------------------------------
// (PART: one of several launches, whose place only they look up: 29.3 us where all did, 28.8 so.)
template <typename ST, int LANES, bool PART>
__global__ __launch_bounds__(256) void selective_step_kernel(StepPart<scanscam_selective_step> args)
{
    const scanscam_selective_step &a = args.a;
    const int lane = threadIdx.x % LANES, N = (int)a.N;
    const int64_t c = (int64_t)((PART ? args.block0 : 0) + blockIdx.y) * (256 / LANES) + threadIdx.x / LANES, row = (PART ? args.row0 : 0) + blockIdx.x;
    const int64_t slot = a.slot != nullptr ? index_at(a.slot, a.slot64, row) : row;
    const bool there = c < a.channels;
    if (slot < 0 || slot >= a.slots) {
        if (there && lane == 0) const_cast<ST *>(token_at<ST>(a.y, 0, row, c))[0] = (ST)0.0f;
        return;
    }
    float y = 0.0f, x = 0.0f, z = 0.0f, skip = 0.0f;
    if (there) {
        // (everything is asked for before any of it is used)
        const ST x_in = token_at<ST>(a.x, 0, row, c)[0], dt_in = token_at<ST>(a.dt, 0, row, c)[0];
        const ST z_in = a.z.p != nullptr ? token_at<ST>(a.z, 0, row, c)[0] : (ST)0.0f;
        const int64_t group = (uint32_t)c / (uint32_t)(a.channels / a.groups);
        const ST *B = token_at<ST>(a.B, 0, row, group * a.B.group), *C = token_at<ST>(a.C, 0, row, group * a.C.group);
        float *state = a.state + (slot * a.channels + c) * N;
        const float bias = param(a.dt_bias, c);
        skip = param(a.D, c);
        float d = 0.0f;
        for (int n0 = lane * 4; n0 < N; n0 += LANES * 4) {
            const int count = N - n0 < 4 ? N - n0 : 4;
            float h[4], b[4], w[4], A[4];
            if (count == 4) {
                Stored<float, 4> h_in;
                Stored<ST, 4> b_in, w_in;
                h_in.load(state + n0);
                b_in.load(B + n0);
                w_in.load(C + n0);
                params(a.A, c * N + n0, 4, A);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    h[i] = h_in[i];
                    b[i] = b_in[i];
                    w[i] = w_in[i];
                }
            } else {
                load_part(state + n0, count, h);
                load_part(B + n0, count, b);
                load_part(C + n0, count, w);
                params(a.A, c * N + n0, count, A);
            }
            if (n0 < LANES * 4) {
                x = (float)x_in;
                d = (float)dt_in + bias;
                if (a.softplus) d = softplus_(d);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                h[i] = __builtin_fmaf(exp_(d * A[i]), h[i], d * x * b[i]);  // (past the last state: zeros)
                y = __builtin_fmaf(w[i], h[i], y);
            }
            store_some(state + n0, count, h);
        }
        x = (float)x_in;
        z = (float)z_in;
    }
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) y += __shfl_xor(y, m);
    if (there && lane == 0) {
        y = __builtin_fmaf(skip, x, y);
        if (a.z.p != nullptr) y *= z * sigmoid_(z);
        const_cast<ST *>(token_at<ST>(a.y, 0, row, c))[0] = (ST)y;
    }
}

}  // namespace scanscam
