// Linear attention with a decay for each head, whole sequences: device code.
//
//   S[t] = e^g[t] S[t-1] + k[t] v[t]^T          (K x V values a head, in fp32)
//   o[t] = scale S[t]^T q[t]
//   backwards, H[t] the gradient of S[t]:  H[t] = scale q[t] do[t]^T + e^g[t+1] H[t+1]
//   dq[t] = scale S[t] do[t],  dk[t] = H[t] v[t],  dv[t] = H[t]^T k[t],  dg[t] = <H[t], e^g[t] S[t-1]>
//
// Chunks of C tokens turn it into matrix products. With G the sums of g from the chunk's first token on and S the state before it,
//   o[t] = scale (e^G[t] S^T q[t] + sum over s <= t of e^(G[t]-G[s]) (q[t] k[s]) v[s]),
//   S'   = e^G[end] S + sum over s of e^(G[end]-G[s]) k[s] v[s]^T.
// dq is the same with (do, v, k) in place of (q, k, v), dk and dv the same backwards in time with (v, do, q) and (k, q, do).
//
// The gradient of a decay is summed up from what passes it: inside of a chunk the pairs
// s < t, M[t,s] = e^(G[t]-G[s]) (q[t] k[s]) (do[t] v[s]); across its borders R[t] = q[t] (what dq[t] takes from S) and
// W[s] = k[s] (what dk[s] takes from H). With X[c] = e^G[end] <H, S>, which passes the whole chunk,
//   dg[t] = X[c] + sum over u >= t of R[u] + sum over s < t of W[s] + sum over s < t <= u of M[u,s],
//   X[c] + sum of W = X[c+1] + sum of the next chunk's R  (both are the product of state and gradient at the border),
// so that X follows from a border on without either state, in 64 bits. R, W and M are fp32's: what their roundings leave in X, some 2^-24 of the products on the way
// from the border, stays also where X is much smaller than these; it is zero where the chunk's decays let nothing through. To keep the way short, at every eighth border the
// pass over queries stores its state, and the pass over keys takes the product anew. The sums of M are differences of sums over rows and columns, which leave 2^-53 of them.
// W and R are fp32's: states go into products in several terms.
//
// Layout. A workgroup takes a head of a sequence (or of a part of it) through its chunks. A wave holds all rows of its own columns of the
// state in the matrix unit's accumulators; these are, as they lie, operands of the next product: with lane = 16 g + n a 16 x 16 tile
// holds rows 4 g + r of column n, and an operand of 32 rows (16 bits) may have its rows in any order that both operands share: rows
// 4 g + (0..3) and 16 + 4 g + (0..3). So the state is rounded to an operand without leaving the registers, and so are the scores, by way of
// LDS (they are shared by the waves) in the operand's own order. Tiles of the tensors lie in LDS as they are in memory; products over
// time read them by transposing loads.
//
// What bounds it: neither memory nor the matrix unit, but the chain of a chunk (loads to LDS, scores, a barrier, sums, the state's update, a barrier) in few waves,
// for a state's columns and a chunk's operands leave registers for two waves a SIMD. [8, 4096, 16 x 128] in bf16, in four parts: ends of parts 60 us, outputs
// 154 (of 537 MB, 3.5 TB/s; 566 by the counters), ends backwards 73, gradients of queries 258, of keys and values 410, decays 12.
// In counters the matrix unit is busy for 26 % of the time forwards and for 18 to 20 % of the gradients' kernels, the vector unit (terms, decays, addresses) for 41 and 33 to 36 %.
#pragma once

#include "ops_common.hpp"
#include "scanscam_attention.h"

#include <type_traits>

namespace scanscam {

typedef short short4v __attribute__((ext_vector_type(4)));
typedef uint32_t raw16 __attribute__((ext_vector_type(4)));

struct AttendArgs {
    scanscam_attend a;
    int64_t first;            // the first unit of this launch; a unit is a part of a head of a sequence
    int64_t tokens;           // batch * T
    int64_t per, cuts;        // tokens of a part, whole chunks (0: all of the sequence); borders between parts that there is room for
    int32_t parts, each;      // parts of a sequence of T tokens, heads that share queries and keys
    // [heads][border between parts][K][V]: what the part before it (gradients: behind it) adds to the state, then the state there; and [heads][border between parts],
    // that part's decay. The borders of a sequence follow each other, those of all sequences too.
    float *ends, *back_ends;
    struct Power {
        float rest;     // rest 2^whole, a part's decay: of logs above zero float32 may not hold it
        int32_t whole;
    } *powers;
    float *reads, *writes;    // [heads][tokens]: R[t] and W[t]
    double *inside;           // [heads][tokens]: the sum of M[t,s] over s less that of M[s,t]
    double *last;             // [sequences][heads]: <gradient of the last state, last state>
    float *borders;           // [border][heads]: the state at a border, tile by tile as the lanes hold it
    double *cross;            // [border][heads]: its product with the gradient there
    int64_t most_borders;     // of a batch element
    float *part_q, *part_k;   // [tokens][heads][K]: gradients of shared queries and keys by head; NULL where none are shared
    float *decays;            // [tokens][heads]: gradients of decays
};

// What differs with the activations' type: an operand is 16 bytes a lane, KS rows of 16 columns.
template <typename ST> struct Operand {
    typedef ST frag __attribute__((ext_vector_type(8)));
    static constexpr int KS = 32, CHUNK = 64;  // rows of an operand; tokens of a chunk
};
// (float32's operands are four steps of the matrix unit's instruction, its tiles twice the size: half the tokens)
template <> struct Operand<float> {
    typedef float4v frag;
    static constexpr int KS = 16, CHUNK = 32;
};
template <typename ST> using frag_t = typename Operand<ST>::frag;

__device__ __forceinline__ float4v mma(const frag_t<__bf16> &a, const frag_t<__bf16> &b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float4v mma(const frag_t<_Float16> &a, const frag_t<_Float16> &b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float4v mma(const float4v &a, const float4v &b, float4v c)
{
#pragma unroll
    for (int r = 0; r < 4; r++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
    return c;
}

// Terms of the activations' type that a float32 factor is taken apart into where float32 results come from it (states that are handed over, gradients
// of states and of decays): all 24 bits, 22 in fp16. Where only 16-bit results come from it, two: 2^-17 of it is lost, and results are as far from 64 bits as ones that
// are rounded once (with the state in one term they were 1.2 to 1.3 times as far, and outputs 141 us of [8, 4096, 16 x 128] in bf16 for 161).
template <typename ST> constexpr int kTerms = 3;
template <> inline constexpr int kTerms<_Float16> = 2;
template <> inline constexpr int kTerms<float> = 1;
template <typename ST> constexpr int kTermsRounded = sizeof(ST) == 2 ? 2 : 1;

// fp16 has five bits of exponent: what is taken apart is first brought to a largest value of 2^14 in the wave, by a power of two, so that the second
// term's smallest step is 2^-38 of it and nothing overflows.
__device__ __forceinline__ float most_of(float v)
{
    const auto top = [](float a, float b) { return a > b ? a : b; };
    v = top(v, dpp_move<0x111, 0xf>(0.0f, v));
    v = top(v, dpp_move<0x112, 0xf>(0.0f, v));
    v = top(v, dpp_move<0x114, 0xf>(0.0f, v));
    v = top(v, dpp_move<0x118, 0xf>(0.0f, v));
    v = top(v, dpp_move<0x142, 0xa>(0.0f, v));
    v = top(v, dpp_move<0x143, 0xc>(0.0f, v));
    return read_lane(v, 63);
}
// `largest(finite)`: the wave's largest absolute value, or largest finite one: one that is not finite is no measure for the others. (The power's inverse is finite too.)
template <typename F> __device__ __forceinline__ float scale_to_fp16(F largest)
{
    float most = largest(false);
    if (__builtin_expect(!(most < __builtin_inff()), 0)) most = largest(true);
    if (!(most > 1e-30f)) return 1.0f;
    return __builtin_ldexpf(1.0f, 14 - (int)(__builtin_bit_cast(uint32_t, most) >> 23) + 127);
}

template <typename ST, int TERMS, int N> __device__ __forceinline__ void split(const float (&x)[N], frag_t<ST> (&out)[TERMS])
{
    if constexpr (sizeof(ST) == 4) {
#pragma unroll
        for (int e = 0; e < N; e++) out[0][e] = x[e];
    } else if constexpr (std::is_same_v<ST, __bf16>) {
        // Two at a time: one conversion makes both, and their 32 bits hold both floats (gradients of queries of the layer above 246 us, 267 one at a time).
        typedef float float2v __attribute__((ext_vector_type(2)));
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            float2v rest = {x[e], x[e + 1]};
#pragma unroll
            for (int t = 0; t < TERMS; t++) {
                const pair h = __builtin_convertvector(rest, pair);
                out[t][e] = h[0];
                out[t][e + 1] = h[1];
                if (t + 1 < TERMS) {
                    const uint32_t bits = __builtin_bit_cast(uint32_t, h);
                    rest[0] -= __builtin_bit_cast(float, bits << 16);  // (an infinity becomes a NaN)
                    rest[1] -= __builtin_bit_cast(float, bits & 0xffff0000u);
                }
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) {
            float rest = x[e];
#pragma unroll
            for (int t = 0; t < TERMS; t++) {
                // (A product that is rounded to fp16 where it is made is rounded once; what is left must be what that rounding left, and not one's after the
                // product was rounded to fp32: where the two differ, the next term would miss by a whole step.)
                asm("" : "+v"(rest));
                const ST h = (ST)rest;
                out[t][e] = h;
                if (t + 1 < TERMS) rest -= (float)h;
            }
        }
    }
}

// A chunk's tokens by up to D channels in LDS. Sixteen bytes of a row lie where an exclusive or with its number puts them, so that neither
// operand's reads meet in a bank: 16 lanes that read 16 rows at a column have 16 places, and 8 rows of 32 bytes eight times two.
template <typename ST, int D> struct Tile {
    static constexpr int VE = 16 / sizeof(ST), ROW = D / VE, WORDS = Operand<ST>::CHUNK * D * (int)sizeof(ST) / 4;
    ST *p;
    static __device__ __forceinline__ int turn(int row)
    {
        if constexpr (sizeof(ST) == 4) return row & 15;
        else if constexpr (D == 64) return (row >> 1 & 3) * 2 + (row >> 3 & 1);
        else return (row & 7) * 2 + (row >> 3 & 1);
    }
    // Column `col` of a row, a multiple of four.
    __device__ __forceinline__ ST *at(int row, int col) const { return p + row * D + ((col / VE ^ turn(row)) * VE + col % VE); }
    // Operand of 16 of the tile's rows; its own rows are the tile's columns k0 ... k0 + KS - 1.
    __device__ __forceinline__ frag_t<ST> rows(int row0, int k0) const
    {
        const int lane = threadIdx.x & 63, row = row0 + (lane & 15), col = k0 + 4 * (lane >> 4);
        if constexpr (sizeof(ST) == 4) {
            return *reinterpret_cast<const float4v *>(at(row, col));
        } else {
            typedef uint32_t raw8 __attribute__((ext_vector_type(2)));
            const raw8 lo = *reinterpret_cast<const raw8 *>(at(row, col)), hi = *reinterpret_cast<const raw8 *>(at(row, col + 16));
            return __builtin_bit_cast(frag_t<ST>, raw16{lo[0], lo[1], hi[0], hi[1]});
        }
    }
    // Operand of 16 of the tile's columns; its own rows are the tile's rows k0 ... k0 + KS - 1.
    __device__ __forceinline__ frag_t<ST> columns(int col0, int k0) const
    {
        const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
        if constexpr (sizeof(ST) == 4) {
            frag_t<ST> f;
#pragma unroll
            for (int r = 0; r < 4; r++) f[r] = at(k0 + 4 * g + r, col0 + (n & 12))[n & 3];
            return f;
        } else {
            typedef __attribute__((address_space(3))) short4v lds4;
            const int row = k0 + 4 * g + (n >> 2), col = col0 + 4 * (n & 3);
            struct Both { short4v lo, hi; };
            return __builtin_bit_cast(frag_t<ST>, Both{__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)at(row, col)), __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)at(row + 16, col))});
        }
    }
    // Four neighbouring columns of a row.
    __device__ __forceinline__ void four(int row, int col, float (&f)[4]) const
    {
        const Elems<ST, 4> v = __builtin_bit_cast(Elems<ST, 4>, *reinterpret_cast<const typename RawT<4 * sizeof(ST)>::type *>(at(row, col)));
#pragma unroll
        for (int r = 0; r < 4; r++) f[r] = (float)v.e[r];
    }
};

// A tile on its way from memory: asked for a chunk ahead, in registers. Rows from `n` on and columns from `d` on are zeros. EXACT: d is a whole
// number of vectors; then every lane loads, rows past the end the last one again, and what is not there becomes zero on the way to LDS.
template <typename ST, int D, int NT, bool EXACT> struct Staged {
    static constexpr int VE = 16 / sizeof(ST), ROW = D / VE, COUNT = Operand<ST>::CHUNK * ROW / NT, STEP = NT / ROW;
    static_assert(NT % ROW == 0 && Operand<ST>::CHUNK * ROW % NT == 0, "whole rows for all threads");
    raw16 v[COUNT];
    const ST *from;  // this lane's first vector in a tile that would begin at the tensor's first token
    int64_t stride;
    int d, col, drop;  // (drop: elements of this lane's vector that come before its column)
    // Where a row ends inside a vector the vector is the row's last whole one, and what of it belongs to the lane before is shifted out on the way to LDS: loads under a
    // condition of the lanes are waited for one after the other ([25, 656, 5 heads of 194 and 27] in bf16: 237 us that way, 198 this way, before halves).
    __device__ __forceinline__ Staged(const ST *base, int64_t token_stride, int channels) : stride(token_stride), d(channels)
    {
        col = threadIdx.x % ROW * VE;
        drop = !EXACT && d >= VE && col < d && col + VE > d ? col + VE - d : 0;
        from = base + threadIdx.x / ROW * stride + (col < d ? col - drop : 0);
    }
    // Of the tokens from t on, of which there are n.
    __device__ __forceinline__ void load(int64_t t, int n)
    {
        using raw_t = typename RawT<sizeof(ST) * VE>::type;
        typedef raw_t unaligned __attribute__((aligned(sizeof(ST))));
        const int row0 = threadIdx.x / ROW;
        const bool whole = EXACT || d >= VE;
        if (whole && n == Operand<ST>::CHUNK) {
#pragma unroll
            for (int i = 0; i < COUNT; i++) v[i] = *reinterpret_cast<const unaligned *>(from + (t + i * STEP) * stride);
        } else if (whole) {
#pragma unroll
            for (int i = 0; i < COUNT; i++) {
                const int row = row0 + i * STEP;
                v[i] = *reinterpret_cast<const unaligned *>(from + (t + (row < n ? row : n - 1) - row0) * stride);
            }
        } else {
#pragma unroll
            for (int i = 0; i < COUNT; i++) {
                Elems<ST, VE> e;
#pragma unroll
                for (int k = 0; k < VE; k++) e.e[k] = (ST)0.0f;
                if (row0 + i * STEP < n && col < d)
#pragma unroll
                    for (int k = 0; k < VE - 1; k++)
                        if (k < d) e.e[k] = from[(t + i * STEP) * stride + k];
                v[i] = __builtin_bit_cast(raw16, e);
            }
        }
    }
    __device__ __forceinline__ raw16 shifted(raw16 x) const
    {
        const int bytes = drop * (int)sizeof(ST);
        if (bytes & 8) x = raw16{x[2], x[3], 0, 0};
        if (bytes & 4) x = raw16{x[1], x[2], x[3], 0};
        if (sizeof(ST) == 2 && (bytes & 2)) x = raw16{x[0] >> 16 | x[1] << 16, x[1] >> 16 | x[2] << 16, x[2] >> 16 | x[3] << 16, x[3] >> 16};
        return x;
    }
    __device__ __forceinline__ void store(Tile<ST, D> tile, int n) const
    {
        const int row0 = threadIdx.x / ROW;
        if (EXACT && n == Operand<ST>::CHUNK && d == D) {
#pragma unroll
            for (int i = 0; i < COUNT; i++) *reinterpret_cast<raw16 *>(tile.at(row0 + i * STEP, col)) = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < COUNT; i++) {
                const bool there = row0 + i * STEP < n && col < d;
                *reinterpret_cast<raw16 *>(tile.at(row0 + i * STEP, col)) = there ? EXACT ? v[i] : shifted(v[i]) : raw16{0, 0, 0, 0};
            }
        }
    }
};

// The tokens that a workgroup goes through: a part of a sequence, of whole chunks but for the last.
struct Span {
    int64_t sequence, batch, from, begin, end, length;  // from, begin and end: tokens of the batch element; from and length: of the sequence
    int64_t cut;  // the first of the sequence's borders between parts
    int head, part, parts;
};
__device__ __forceinline__ void span_of_sequence(const scanscam_attend &a, Span &s)
{
    int64_t from = 0, to = a.T;
    s.batch = s.sequence;
    if (a.offsets != nullptr) {
        s.batch = 0;
        from = clamp_(index_at(a.offsets, a.offsets64, s.sequence), 0, a.T);
        to = clamp_(index_at(a.offsets, a.offsets64, s.sequence + 1), from, a.T);
    }
    s.from = from;
    s.length = to - from;
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane)
{
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)v, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane);
    return (int64_t)(hi << 32 | lo);
}
// Parts of sequences of different lengths: a long one has more. Every wave counts for itself, 64 sequences at a time: those of the sequences before `sequence`, or where
// that is negative before the one that part `slot` of all belongs to, which s then holds (false if there is none, or no room for its borders).
__device__ __forceinline__ bool count_parts(const AttendArgs &args, int64_t sequence, int64_t slot, Span &s)
{
    const scanscam_attend &a = args.a;
    const int lane = threadIdx.x & 63;
    int64_t before = 0;
    for (int64_t first = 0; first < a.sequences; first += 64) {
        Span at;
        at.sequence = first + lane;
        int64_t parts = 0;
        if (at.sequence < a.sequences) {
            span_of_sequence(a, at);
            const int64_t whole = (at.length + args.per - 1) / args.per;
            parts = whole < 1 ? 1 : whole;
        }
        int64_t upto = parts;
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
            const int64_t other = __shfl_up(upto, step, 64);
            if (lane >= step) upto += other;
        }
        const uint64_t found = __ballot(sequence >= 0 ? at.sequence == sequence : at.sequence < a.sequences && before + upto > slot);
        if (found != 0) {
            const int there = __builtin_ctzll(found);
            s.parts = (int)lane_of(parts, there);
            s.sequence = first + there;
            before += lane_of(upto, there) - s.parts;
            s.part = (int)(slot - before);
            s.cut = before - s.sequence;
            return s.cut + s.parts - 1 <= args.cuts;  // (always, but with offsets that go back)
        }
        before += lane_of(upto, 63);
    }
    return false;
}
// The span of a unit; false if there is none.
__device__ __forceinline__ bool span_of(const AttendArgs &args, int64_t unit, int chunk, Span &s)
{
    const scanscam_attend &a = args.a;
    // (Parts are next to each other: heads of the same tokens, which can share lines of memory, would be on different XCDs. 30001 tokens of 4 heads of 48 and 72
    // in float32, with gradients: 450 us, 428 so.)
    if (args.per == 0 || a.offsets == nullptr) {
        s.parts = args.per == 0 ? 1 : args.parts;
        s.part = (int)(unit % s.parts);
        s.head = (int)(unit / s.parts % a.heads);
        s.sequence = unit / s.parts / a.heads;
        s.cut = s.sequence * (s.parts - 1);
    } else {
        const int64_t slots = a.sequences + args.cuts;
        s.head = (int)(unit / slots);
        if (!count_parts(args, -1, unit % slots, s)) return false;
    }
    span_of_sequence(a, s);
    const int64_t per = args.per == 0 ? s.length : args.per;
    s.begin = s.from + (s.part * per < s.length ? s.part * per : s.length);
    s.end = s.from + ((s.part + 1) * per < s.length ? (s.part + 1) * per : s.length);
    return true;
}
__device__ __forceinline__ int64_t cut_at(const AttendArgs &args, const Span &s, int i) { return s.head * args.cuts + s.cut + i; }
// Where the state lies that a part starts from: the given one, or that at the border before it (gradients: behind it).
__device__ __forceinline__ const float *start_of(const AttendArgs &args, const Span &s, bool back)
{
    const scanscam_attend &a = args.a;
    const int64_t values = (int64_t)a.K * a.V;
    if (s.part != (back ? s.parts - 1 : 0)) return (back ? args.back_ends : args.ends) + cut_at(args, s, s.part - (back ? 0 : 1)) * values;
    const float *given = back ? a.gstate_out : a.state_in;
    return given == nullptr ? nullptr : given + (s.sequence * a.heads + s.head) * values;
}

template <typename ST> __device__ __forceinline__ const ST *tensor_at(const scanscam_tokens &t, const Span &s, int64_t head)
{
    return static_cast<const ST *>(t.p) + s.batch * t.batch + head * t.group;
}

// A token's log of a decay as it is stored: taken apart only where it is used, a chunk after it is asked for.
__device__ __forceinline__ uint32_t decay_at(const scanscam_attend &a, const Span &s, int64_t token, bool there)
{
    uint32_t raw = 0;
    if (there && a.decay.p != nullptr) {
        const int64_t at = s.batch * a.decay.batch + token * a.decay.token + s.head;
        if (a.decay_dtype == SCANSCAM_F32) raw = static_cast<const uint32_t *>(a.decay.p)[at];
        else raw = static_cast<const uint16_t *>(a.decay.p)[at];
    }
    return raw;
}
// ... in powers of two. An infinitely strong one is 2^-1000000, which is zero in fp32 but has differences.
__device__ __forceinline__ double decay_of(const scanscam_attend &a, uint32_t raw)
{
    const float g = a.decay_dtype == SCANSCAM_F32    ? __builtin_bit_cast(float, raw)
                    : a.decay_dtype == SCANSCAM_BF16 ? __builtin_bit_cast(float, raw << 16)
                                                     : (float)__builtin_bit_cast(_Float16, (uint16_t)raw);
    const double d = (double)g * 1.4426950408889634074;
    return d < -1e6 ? -1e6 : d > 1e6 ? 1e6 : d;  // (a NaN stays one)
}
// Sums over the lanes up to each, in 64 bits: differences of them are exponents, and 32 bits would lose what small decays add to large ones.
__device__ __forceinline__ double sums_upto(double v)
{
    v += dpp_move<0x111, 0xf>(0.0, v);
    v += dpp_move<0x112, 0xf>(0.0, v);
    v += dpp_move<0x114, 0xf>(0.0, v);
    v += dpp_move<0x118, 0xf>(0.0, v);
    v += dpp_move<0x142, 0xa>(0.0, v);
    v += dpp_move<0x143, 0xc>(0.0, v);
    return v;
}
__device__ __forceinline__ float exp2_(double x) { return __builtin_amdgcn_exp2f((float)x); }

// Of a chunk, in LDS: the sums of decays, e^G[t] and e^(G[end] - G[t]).
template <int C> struct Decays {
    double *sums;
    float *upto, *after;
    // By the first wave.
    __device__ __forceinline__ void fill(double g)
    {
        const double G = sums_upto(g), end = read_lane(G, 63);
        if (threadIdx.x < C) {
            sums[threadIdx.x] = G;
            upto[threadIdx.x] = exp2_(G);
            after[threadIdx.x] = exp2_(end - G);
        }
    }
    __device__ __forceinline__ float whole() const { return upto[C - 1]; }  // (tokens past the end have no decay)
    static constexpr int WORDS = 4 * C;
};

// sum over 16 neighbouring lanes, in the last of them
__device__ __forceinline__ double row_sum(double v)
{
    v += dpp_move<0x111, 0xf>(0.0, v);
    v += dpp_move<0x112, 0xf>(0.0, v);
    v += dpp_move<0x114, 0xf>(0.0, v);
    v += dpp_move<0x118, 0xf>(0.0, v);
    return v;
}
// sum over the four lanes that hold the same column, in all of them
template <typename T> __device__ __forceinline__ T column_sum4(T v)
{
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Waits for everything asked for before a loop. What is still under way where a loop begins (the state's first values) the compiler takes to be so in every
// turn, and waits there for what the turn itself has asked for meanwhile.
__device__ __forceinline__ void settle()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt 0
    asm volatile("" ::: "memory");
}

// A value that is not known before: what is computed with it is computed there, and not ahead of a loop, to lie in registers all the while.
__device__ __forceinline__ int later(int v)
{
    asm volatile("" : "+v"(v));
    return v;
}

// The same for one of the wave. (With heads over 128 channels a wave has one unit of scores at most, whose addresses would be made before the loop and lie in memory:
// [4, 4096, 8 x 256 x 256] in bf16 380 us for outputs and 1018 for gradients of keys and values, 295 and 804 so.)
__device__ __forceinline__ int later_uniform(int v)
{
    asm volatile("" : "+s"(v));
    return v;
}

// A wave's columns of a state: all rows, in accumulators. Column tile jt of wave w is the state's tile jt * WAVES + w. Products go over the rows that
// there are, 64 at a time.
template <typename ST, int D, int JT, int WAVES> struct State {
    static constexpr int KS = Operand<ST>::KS, PER = KS / 16, RT = D / 16, C = Operand<ST>::CHUNK, STEPS = C / KS;
    float4v s[RT][JT];
    int wave;
    __device__ __forceinline__ int column(int jt) const { return (jt * WAVES + wave) * 16; }
    // value = f(value, row, column) for this lane's values below `rows` and `cols`.
    template <typename F> __device__ __forceinline__ void each(int rows, int cols, F f)
    {
        const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int jt = 0; jt < JT; jt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int row = rt * 16 + 4 * g + r, col = column(jt) + n;
                    if (row < rows && col < cols) s[rt][jt][r] = f(s[rt][jt][r], row, col);
                }
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int jt = 0; jt < JT; jt++) s[rt][jt] = float4v{0, 0, 0, 0};
    }
    // From and to memory where neighbouring rows and columns are so far apart (zeros without memory), and this lane's part of the product with it.
    __device__ __forceinline__ void read(const float *p, int rows, int cols, int row_step, int col_step)
    {
        clear();
        if (p != nullptr) each(rows, cols, [&](float, int row, int col) { return p[row * row_step + col * col_step]; });
    }
    __device__ __forceinline__ void write(float *p, int rows, int cols, int row_step, int col_step)
    {
        each(rows, cols, [&](float v, int row, int col) { return p[row * row_step + col * col_step] = v; });
    }
    __device__ __forceinline__ double dot(const float *p, int rows, int cols, int row_step, int col_step)
    {
        double sum = 0.0;
        each(rows, cols, [&](float v, int row, int col) {
            sum += (double)v * (double)p[row * row_step + col * col_step];
            return v;
        });
        return sum;
    }
    // As the lanes hold it, tile by tile: to memory, and this lane's part of the product with one from there.
    __device__ __forceinline__ void keep(float *p, int rows, int cols) const
    {
        float4v *at = reinterpret_cast<float4v *>(p) + later(threadIdx.x & 63);
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int jt = 0; jt < JT; jt++)
                if (rt * 16 < rows && column(jt) < cols) at[(rt * RT + column(jt) / 16) * 64] = s[rt][jt];
    }
    __device__ __forceinline__ double kept(const float *p, int rows, int cols) const
    {
        const float4v *at = reinterpret_cast<const float4v *>(p) + later(threadIdx.x & 63);
        double sum = 0.0;
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int jt = 0; jt < JT; jt++)
                if (rt * 16 < rows && column(jt) < cols) {
                    const float4v other = at[(rt * RT + column(jt) / 16) * 64];
#pragma unroll
                    for (int r = 0; r < 4; r++) sum += (double)s[rt][jt][r] * (double)other[r];
                }
        return sum;
    }
    // The wave's largest absolute value, or finite one.
    __device__ __forceinline__ float largest(bool finite) const
    {
        float most = 0.0f;
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int jt = 0; jt < JT; jt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float v = __builtin_fabsf(s[rt][jt][r]);
                    most = __builtin_fmaxf(most, finite && !(v < __builtin_inff()) ? 0.0f : v);
                }
        return most_of(most);
    }
    // The power of two that the state is multiplied with in operands.
    __device__ __forceinline__ float scale() const
    {
        if constexpr (!std::is_same_v<ST, _Float16>) return 1.0f;
        return scale_to_fp16([&](bool finite) { return largest(finite); });
    }
    // acc[tt][jt], columns: rows of `of` (tokens), rows: the state's columns: the state's product with them, times the power of two that is returned.
    template <int TERMS> __device__ __forceinline__ float times(Tile<ST, D> of, int rows, float4v (&acc)[C / 16][JT]) const
    {
        const float factor = scale();
#pragma unroll
        for (int tt = 0; tt < C / 16; tt++)
#pragma unroll
            for (int jt = 0; jt < JT; jt++) acc[tt][jt] = float4v{0, 0, 0, 0};
#pragma unroll
        for (int k0 = 0; k0 < D; k0 += 64) {
            if (k0 >= rows) break;
#pragma unroll
            for (int k = k0; k < k0 + 64; k += KS) {
                frag_t<ST> own[JT][TERMS];
#pragma unroll
                for (int jt = 0; jt < JT; jt++) {
                    float x[4 * PER];
#pragma unroll
                    for (int h = 0; h < PER; h++)
#pragma unroll
                        for (int r = 0; r < 4; r++) x[4 * h + r] = s[k / 16 + h][jt][r] * factor;
                    split<ST, TERMS>(x, own[jt]);
                }
#pragma unroll
                for (int tt = 0; tt < C / 16; tt++) {
                    const frag_t<ST> token = of.rows(tt * 16, k);
#pragma unroll
                    for (int jt = 0; jt < JT; jt++)
#pragma unroll
                        for (int t = 0; t < TERMS; t++) acc[tt][jt] = mma(own[jt][t], token, acc[tt][jt]);
                }
            }
        }
        return factor;
    }
    // s = decay s + sum over the chunk's tokens of from[t] (weight[t] factor own[t])^T; scaled: what times() or scale() of this state returned
    template <int TERMS>
    __device__ __forceinline__ void update(Tile<ST, D> from, int rows, const frag_t<ST> (&own)[JT][STEPS], const float *weight, float factor, float decay, float scaled)
    {
        const int g = (threadIdx.x & 63) >> 4;
        float bring = 1.0f;
        if constexpr (std::is_same_v<ST, _Float16>) {
            bring = scale_to_fp16([&](bool finite) {
                float most = 0.0f;
#pragma unroll
                for (int step = 0; step < STEPS; step++)
#pragma unroll
                    for (int h = 0; h < PER; h++) {
                        const float4v w = *reinterpret_cast<const float4v *>(weight + step * KS + 16 * h + 4 * g);
#pragma unroll
                        for (int jt = 0; jt < JT; jt++)
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const float v = __builtin_fabsf((float)own[jt][step][4 * h + r] * (w[r] * factor));
                                most = __builtin_fmaxf(most, finite && !(v < __builtin_inff()) ? 0.0f : v);
                            }
                    }
                return most_of(most);
            });
            // The state is multiplied with it as well, and must stay finite.
            const float most = 32768.0f / scaled * decay;
            if (__builtin_expect(!(most * bring < 0x1p126f), 0)) {
                const float room = most < __builtin_inff() ? __builtin_ldexpf(1.0f, 125 + 127 - (int)(__builtin_bit_cast(uint32_t, most) >> 23)) : 1.0f;
                bring = bring < room ? bring : room;
            }
            factor *= bring;
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int jt = 0; jt < JT; jt++) s[rt][jt] *= decay * bring;
#pragma unroll
        for (int step = 0; step < STEPS; step++) {
            frag_t<ST> scaled[JT][TERMS];
#pragma unroll
            for (int jt = 0; jt < JT; jt++) {
                float x[4 * PER];
#pragma unroll
                for (int h = 0; h < PER; h++) {
                    const float4v w = *reinterpret_cast<const float4v *>(weight + step * KS + 16 * h + 4 * g);
#pragma unroll
                    for (int r = 0; r < 4; r++) x[4 * h + r] = (float)own[jt][step][4 * h + r] * (w[r] * factor);
                }
                split<ST, TERMS>(x, scaled[jt]);
            }
#pragma unroll
            for (int row0 = 0; row0 < D; row0 += 64) {
                if (row0 >= rows) break;
#pragma unroll
                for (int rt = row0 / 16; rt < row0 / 16 + 4; rt++) {
                    const frag_t<ST> row = from.columns(rt * 16, step * KS);
#pragma unroll
                    for (int jt = 0; jt < JT; jt++)
#pragma unroll
                        for (int t = 0; t < TERMS; t++) s[rt][jt] = mma(row, scaled[jt][t], s[rt][jt]);
                }
            }
        }
        if constexpr (std::is_same_v<ST, _Float16>) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int jt = 0; jt < JT; jt++) s[rt][jt] *= 1.0f / bring;
        }
    }
};

// A product of 16 tokens by 16 over their channels, 64 at a time.
template <typename ST, int D> __device__ __forceinline__ float4v score(Tile<ST, D> a, int a0, Tile<ST, D> b, int b0, int channels)
{
    float4v p{0, 0, 0, 0};
#pragma unroll
    for (int k0 = 0; k0 < D; k0 += 64) {
        if (k0 >= channels) break;
#pragma unroll
        for (int k = k0; k < k0 + 64; k += Operand<ST>::KS) p = mma(a.rows(a0, k), b.rows(b0, k), p);
    }
    return p;
}

// Chunks between borders whose products are taken from the states. For 128 x 128 values a head the states stored are 7 % of the bytes of a backward pass.
constexpr int kBorder = 8;
// Of the border before token t of a sequence that begins at token `from`, at a multiple of kBorder chunks: borders of a sequence are so far apart, and
// of the next one's first token's at least the same as of this one's last border, so that each has a place of its own.
__device__ __forceinline__ int64_t border_at(const AttendArgs &args, int64_t batch, int64_t t, int chunk, int head)
{
    return (batch * args.most_borders + t / (kBorder * chunk)) * args.a.heads + head;
}

// The scores of a chunk in LDS, as operands: [term][tile of 16 columns][step of KS rows][lane] of 16 bytes each. In 16 bits they have two terms:
// the rounding of one is that of every result which it is the largest factor of, once more than the result's own.
// In fp16 a token's scores of a step are multiplied with a power of two that brings the largest of them to 2^14, as states are, and sums of products with them by its
// inverse: scores below 2^-14 would be rounded in steps of 2^-24 otherwise, and lost below 2^-25 (queries and keys of 3e-4: outputs 19 % off), and past 65504 infinite.
template <typename ST> struct Scores {
    static constexpr bool SCALED = std::is_same_v<ST, _Float16>;
    static constexpr int KS = Operand<ST>::KS, PER = KS / 16, C = Operand<ST>::CHUNK, TT = C / 16, STEPS = C / KS, TERMS = sizeof(ST) == 2 ? 2 : 1, ONE = TT * STEPS * 64;
    static constexpr int SCALES = SCALED ? STEPS * C : 0, WORDS = TERMS * ONE * 4 + SCALES, UNITS = STEPS * (TT + PER) / 2;
    frag_t<ST> *p;
    __device__ __forceinline__ float *unscale(int step) const { return reinterpret_cast<float *>(p + TERMS * ONE) + step * C; }
    __device__ __forceinline__ frag_t<ST> operand(int tile, int step, int term) const { return p[term * ONE + (tile * STEPS + step) * 64 + (threadIdx.x & 63)]; }
    // A 16 x 16 tile of rows row_tile * 16 ... and columns tile * 16 ...
    __device__ __forceinline__ void put(int tile, int row_tile, float4v v) const
    {
        using raw_t = typename RawT<4 * sizeof(ST)>::type;
        const float f[4] = {v[0], v[1], v[2], v[3]};
        frag_t<ST> terms[TERMS];
        split<ST, TERMS>(f, terms);
#pragma unroll
        for (int term = 0; term < TERMS; term++) {
            Elems<ST, 4> four;
#pragma unroll
            for (int r = 0; r < 4; r++) four.e[r] = terms[term][r];
            *reinterpret_cast<raw_t *>(reinterpret_cast<ST *>(p + term * ONE + (tile * STEPS + row_tile / PER) * 64 + (threadIdx.x & 63)) + row_tile % PER * 4) = __builtin_bit_cast(raw_t, four);
        }
    }
    __device__ __forceinline__ float at(int row, int column) const
    {
        const ST *e = reinterpret_cast<const ST *>(p + (column / 16 * STEPS + row / KS) * 64 + row % 16 / 4 * 16 + column % 16) + row % KS / 16 * 4 + row % 4;
        const float most = (float)*e, back = SCALED ? unscale(row / KS)[column] : 1.0f;
        return (TERMS == 2 && __builtin_isfinite(most) ? most + (float)e[ONE * (16 / sizeof(ST))] : most) * back;
    }
    // The scores of a step's PER row tiles by 16 columns (zeros beyond the diagonal), which lie lane by lane: lane 16 g + n has four rows of column n.
    __device__ __forceinline__ void put_step(int tile, int step, float4v (&v)[PER]) const
    {
        if constexpr (SCALED) {
            float most = 0.0f;
#pragma unroll
            for (int h = 0; h < PER; h++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float x = __builtin_fabsf(v[h][r]);
                    most = __builtin_fmaxf(most, x < __builtin_inff() ? x : 0.0f);  // (what is not finite is no measure for the others)
                }
            most = __builtin_fmaxf(most, __shfl_xor(most, 16));
            most = __builtin_fmaxf(most, __shfl_xor(most, 32));
            const int up = most > 1e-30f ? 14 + 127 - (int)(__builtin_bit_cast(uint32_t, most) >> 23) : 0;
            const float factor = __builtin_bit_cast(float, (uint32_t)(127 + up) << 23);
#pragma unroll
            for (int h = 0; h < PER; h++) v[h] *= factor;
            if ((threadIdx.x & 63) < 16) unscale(step)[tile * 16 + (threadIdx.x & 63)] = __builtin_bit_cast(float, (uint32_t)(127 - up) << 23);
        }
#pragma unroll
        for (int h = 0; h < PER; h++) put(tile, step * PER + h, v[h]);
    }
    // sum += (rows of `own`) x (tile's column of scores), over a step.
    template <int JT> __device__ __forceinline__ void times(const frag_t<ST> (&own)[JT][STEPS], int tile, int step, float4v (&sum)[JT]) const
    {
        float4v part[JT];
#pragma unroll
        for (int jt = 0; jt < JT; jt++) part[jt] = SCALED ? float4v{0, 0, 0, 0} : sum[jt];
#pragma unroll
        for (int term = TERMS; term-- > 0;) {
            const frag_t<ST> f = operand(tile, step, term);
#pragma unroll
            for (int jt = 0; jt < JT; jt++) part[jt] = mma(own[jt][step], f, part[jt]);
        }
        const float back = SCALED ? unscale(step)[tile * 16 + (threadIdx.x & 15)] : 1.0f;
#pragma unroll
        for (int jt = 0; jt < JT; jt++) sum[jt] = SCALED ? sum[jt] + part[jt] * back : part[jt];
    }
};

// The id-th column tile and step of scores that products reach: those of PER row tiles first, so that waves which take two take a whole one and one of a single tile.
// (Row tiles up to the diagonal; for those from it on both count from the other end.)
template <typename ST> __device__ __forceinline__ void unit_of(int id, int &tile, int &step)
{
    if constexpr (Operand<ST>::KS / 16 == 2) {
        static_assert(Operand<ST>::CHUNK == 64, "four column tiles of two steps");
        tile = id < 2 ? 3 : id == 2 ? 2 : id == 3 ? 1 : id == 4 ? 2 : 0;
        step = id == 1 || id == 4 ? 1 : 0;
    } else {
        static_assert(Operand<ST>::CHUNK == 32, "two column tiles of two steps");
        tile = id < 2 ? 1 : 0;
        step = id == 1 ? 1 : 0;
    }
}

// Four neighbouring values of a token's output. EXACT: `cols` is a multiple of four.
template <bool EXACT, typename ST> __device__ __forceinline__ void put4(ST *row, int col, int cols, float4v v)
{
    const float f[4] = {v[0], v[1], v[2], v[3]};
    if (col < cols) store_some<ST, 4>(row + col, EXACT ? 4 : cols - col, f);
}

// Waves of a workgroup, or in the pass over keys and values of each of its kinds: four with up to two tiles of 16 columns each. (Eight waves of one tile
// read the shared operands twice as often: [8, 4096, 16 x 128] in bf16 201 us forwards, 164 so.)
template <int D> constexpr int attend_waves() { return D == 256 ? 8 : 4; }
// Gradients of queries have a third more in registers. With three terms of 128 columns that is more than there are of them: eight waves of one tile take 269 us of
// that layer, four 290. With two (fp16, [2, 4096, 32 x 128]) eight take 120 us, four 118.
template <typename ST, int D> constexpr int query_waves() { return D == 128 && kTerms<ST> == 3 ? 8 : attend_waves<D>(); }

// --- outputs (x, y, z = q, k, v) and, with GRAD, gradients of queries (x, y, z = do, v, k) with what decays read -----------------------
template <typename ST, int W, int D, bool GRAD> struct AttendLds {
    static constexpr int C = Operand<ST>::CHUNK;
    static constexpr int WORDS = 3 * Tile<ST, D>::WORDS + Scores<ST>::WORDS + Decays<C>::WORDS + (GRAD ? W * C + 2 * W : 0);
};
template <typename ST, int D, int JT, int W, bool GRAD, bool EXACT> __global__ __launch_bounds__(64 * W, 2) void attend_kernel(AttendArgs args)
{
    constexpr int C = Operand<ST>::CHUNK, KS = Operand<ST>::KS, NT = 64 * W, STEPS = C / KS, TT = C / 16, PER = KS / 16, TERMS = kTerms<ST>;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const scanscam_attend &a = args.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g = lane >> 4;
    float *at = lds;
    const auto take = [&](int words) { float *p = at; at += words; return p; };
    Tile<ST, D> X{reinterpret_cast<ST *>(take(Tile<ST, D>::WORDS))}, Y{reinterpret_cast<ST *>(take(Tile<ST, D>::WORDS))}, Z{reinterpret_cast<ST *>(take(Tile<ST, D>::WORDS))};
    Scores<ST> scores{reinterpret_cast<frag_t<ST> *>(take(Scores<ST>::WORDS))};
    Decays<C> decays{reinterpret_cast<double *>(take(2 * C)), take(C), take(C)};
    float *red = GRAD ? take(W * C) : nullptr;
    double *last = GRAD ? reinterpret_cast<double *>(take(2 * W)) : nullptr;

    Span span;
    if (!span_of(args, args.first + blockIdx.x, C, span)) return;
    const int64_t shared = span.head / args.each;
    const int K = (int)a.K, V = (int)a.V;
    const scanscam_tokens &xt = GRAD ? a.gy : a.q, &yt = GRAD ? a.v : a.k, &zt = GRAD ? a.k : a.v;
    const ST *x = tensor_at<ST>(xt, span, GRAD ? span.head : shared), *y = tensor_at<ST>(yt, span, GRAD ? span.head : shared), *z = tensor_at<ST>(zt, span, GRAD ? shared : span.head);
    const ST *q = GRAD ? tensor_at<ST>(a.q, span, shared) : nullptr;
    const int inner = GRAD ? V : K, outer = GRAD ? K : V;  // rows and columns of the state as it is held here
    const int row_step = GRAD ? 1 : V, col_step = GRAD ? V : 1;
    const int64_t pair = span.sequence * a.heads + span.head;
    // Where this lane's outputs go: token n16 of a tile, four columns from 4 g on of each of its tiles.
    const int64_t out_step = GRAD ? args.part_q != nullptr ? a.heads * K : a.gq.token : a.y.token;
    const int64_t out_first = GRAD ? args.part_q != nullptr ? (span.batch * a.T * a.heads + span.head) * K : span.batch * a.gq.batch + span.head * a.gq.group
                                   : span.batch * a.y.batch + span.head * a.y.group;
    const int64_t out_lane = out_first + n16 * out_step + 4 * g;

    State<ST, D, JT, W> S;
    S.wave = wave;
    S.read(start_of(args, span, false), inner, outer, row_step, col_step);

    Staged<ST, D, NT, EXACT> sx(x, xt.token, inner), sy(y, yt.token, inner), sz(z, zt.token, outer);
    uint32_t decay = 0;
    const auto ask = [&](int64_t t) {
        const int n = (int)(span.end - t < C ? span.end - t : C);
        if (wave == 0) decay = decay_at(a, span, t + lane, lane < n);
        sx.load(t, n);
        sy.load(t, n);
        sz.load(t, n);
    };
    if (span.begin < span.end) ask(span.begin);
    settle();
    for (int64_t t0 = span.begin; t0 < span.end; t0 += C) {
        const int n = (int)(span.end - t0 < C ? span.end - t0 : C);
        sx.store(X, n);
        sy.store(Y, n);
        sz.store(Z, n);
        if (wave == 0) decays.fill(decay_of(a, decay));
        __syncthreads();
        // This lane's part of the queries, which only the sums over channels need.
        Elems<ST, 4> queries[TT][JT];
        if constexpr (GRAD) {
            using raw_t = typename RawT<4 * sizeof(ST)>::type;
            typedef raw_t unaligned __attribute__((aligned(sizeof(ST))));
#pragma unroll
            for (int tt = 0; tt < TT; tt++)
#pragma unroll
                for (int jt = 0; jt < JT; jt++) {
                    const int t = tt * 16 + n16, col = S.column(jt) + 4 * g;
                    const ST *from = q + (t0 + (t < n ? t : n - 1)) * a.q.token + (col >= outer ? 0 : EXACT || col + 4 <= outer || outer < 4 ? col : outer - 4);
                    if (EXACT || outer >= 4) {  // (a row's last four where there are no four, in the others' order below)
                        const raw_t raw = *reinterpret_cast<const unaligned *>(from);
                        queries[tt][jt] = __builtin_bit_cast(Elems<ST, 4>, raw);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; r++) queries[tt][jt].e[r] = col + r < outer ? from[r] : (ST)0.0f;
                    }
                }
        }
        if (t0 + C < span.end) ask(t0 + C);

        // Scores: tiles of 16 tokens s (rows) by 16 tokens t (columns), t >= s. (The first wave, which has the decays, is not among those with one more.)
        for (int id = D == 256 ? later_uniform((wave + 2) % W) : (wave + 2) % W; id < Scores<ST>::UNITS; id += W) {
            int tt, step;
            unit_of<ST>(id, tt, step);
            const double upto = decays.sums[tt * 16 + n16];
            float4v p[PER];
#pragma unroll
            for (int h = 0; h < PER; h++) {
                const int st = step * PER + h;
                p[h] = float4v{0, 0, 0, 0};
                if (st > tt) continue;
                p[h] = score(Y, st * 16, X, tt * 16, inner);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int s = st * 16 + 4 * g + r, t = tt * 16 + n16;
                    p[h][r] = s <= t ? p[h][r] * (exp2_(upto - decays.sums[s]) * a.scale) : 0.0f;
                }
            }
            scores.put_step(tt, step, p);
        }
        float4v acc[TT][JT];
        const float scaled = S.template times<GRAD ? TERMS : kTermsRounded<ST>>(X, inner, acc), factor = a.scale / scaled;
        if constexpr (GRAD)
            if (args.borders != nullptr && t0 > span.from && (t0 - span.from) % (kBorder * C) == 0)
                S.keep(args.borders + border_at(args, span.batch, t0, C, span.head) * D * D, inner, outer);
        frag_t<ST> own[JT][STEPS];
#pragma unroll
        for (int jt = 0; jt < JT; jt++)
#pragma unroll
            for (int step = 0; step < STEPS; step++) own[jt][step] = Z.columns(S.column(jt), step * KS);
        __syncthreads();

#pragma unroll
        for (int tt = 0; tt < TT; tt++) {
            const int t = tt * 16 + n16;
            const float upto = decays.upto[t] * factor;
            float read = 0.0f, finite = 0.0f;
            float4v sum[JT];
#pragma unroll
            for (int jt = 0; jt < JT; jt++) {
                acc[tt][jt] *= upto;
                if constexpr (GRAD) {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        float query = (float)queries[tt][jt].e[r];
                        if constexpr (!EXACT) {
                            const int col = S.column(jt) + 4 * g, drop = outer < 4 ? 0 : col + 4 - outer;
                            if (drop > 0) {
                                query = 0.0f;
#pragma unroll
                                for (int from = r + 1; from < 4; from++) query = drop == from - r ? (float)queries[tt][jt].e[from] : query;
                            }
                        }
                        read += query * acc[tt][jt][r];
                    }
                }
                sum[jt] = acc[tt][jt];
            }
#pragma unroll
            for (int step = 0; step <= tt / PER; step++) scores.times(own, tt, step, sum);
            if constexpr (!GRAD) {
#pragma unroll
                for (int jt = 0; jt < JT; jt++)
#pragma unroll
                    for (int r = 0; r < 4; r++) finite += sum[jt][r] * 0.0f;
                if (__builtin_expect(__ballot(finite != 0.0f) != 0, 0)) {
                    // A value that is not finite may be a later token's, times a score of zero. Where the tokens up to t alone give a finite sum it is the product's
                    // without such values, in the same order as ever.
                    float4v clean[JT];
#pragma unroll
                    for (int jt = 0; jt < JT; jt++) clean[jt] = acc[tt][jt];
#pragma unroll
                    for (int step = 0; step <= tt / PER; step++) {
                        frag_t<ST> values[JT][STEPS];
#pragma unroll
                        for (int jt = 0; jt < JT; jt++)
#pragma unroll
                            for (int e = 0; e < 4 * PER; e++) values[jt][step][e] = __builtin_isfinite((float)own[jt][step][e]) ? own[jt][step][e] : (ST)0.0f;
                        scores.times(values, tt, step, clean);
                    }
#pragma unroll
                    for (int jt = 0; jt < JT; jt++) {
                        float4v alone = acc[tt][jt];
                        for (int s = 0; s <= t; s++) {
                            float value[4];
                            Z.four(s, S.column(jt) + 4 * g, value);
                            const float p = scores.at(s, t);
#pragma unroll
                            for (int r = 0; r < 4; r++) alone[r] += p * value[r];
                        }
#pragma unroll
                        for (int r = 0; r < 4; r++) sum[jt][r] = __builtin_isfinite(alone[r]) ? clean[jt][r] : alone[r];
                    }
                    settle();
                }
            }
            if (t < n) {
                const int64_t row = out_lane + (t0 + tt * 16) * out_step;
#pragma unroll
                for (int jt = 0; jt < JT; jt++) {
                    const int col = S.column(jt), there = outer - 4 * g;
                    if constexpr (!GRAD) {
                        put4<EXACT>(static_cast<ST *>(a.y.p) + row, col, there, sum[jt]);
                    } else if (args.part_q != nullptr) {
                        put4<EXACT>(args.part_q + row, col, there, sum[jt]);
                    } else {
                        put4<EXACT>(static_cast<ST *>(a.gq.p) + row, col, there, sum[jt]);
                    }
                }
            }
            if constexpr (GRAD) {
                read = column_sum4(read);
                if (g == 0) red[wave * C + t] = read;
            }
        }
        S.template update<TERMS>(Y, inner, own, decays.after, 1.0f, decays.whole(), scaled);
        __syncthreads();
        if constexpr (GRAD) {
            if (threadIdx.x < (unsigned)n && args.reads != nullptr) {
                const int t = threadIdx.x;
                float read = 0.0f;
                for (int w = 0; w < W; w++) read += red[w * C + t];
                args.reads[span.head * args.tokens + span.batch * a.T + t0 + t] = read;
            }
        }
    }
    if (span.part == span.parts - 1) {
        if constexpr (!GRAD) {
            if (a.state_out != nullptr) S.write(a.state_out + pair * K * V, inner, outer, row_step, col_step);
        } else if (args.last != nullptr) {
            double sum = a.gstate_out == nullptr ? 0.0 : S.dot(a.gstate_out + pair * K * V, inner, outer, row_step, col_step);
            sum = sums_upto(sum);
            if (lane == 63) last[wave] = sum;
            __syncthreads();
            if (threadIdx.x == 0) {
                double total = 0.0;
                for (int w = 0; w < W; w++) total += last[w];
                args.last[pair] = total;
            }
        }
    }
}

// --- what a part of a sequence adds to the state (y, z = k, v), or backwards in time to the state's gradient (do, q) --------------------
template <typename ST, int D> struct EndsLds {
    static constexpr int WORDS = 2 * Tile<ST, D>::WORDS + Decays<Operand<ST>::CHUNK>::WORDS;
};
// W waves of JT tiles each. (128 columns are eight waves of one tile, which leave each other twice as much to wait for: 61 us for the first three of four parts of
// [8, 4096, 16 x 128] in bf16, 67 by four waves of two.)
template <typename ST, int D, int JT, int W, bool BACK, int TERMS, bool EXACT> __global__ __launch_bounds__(64 * W, D == 128 && W == 8 ? 4 : 2) void ends_kernel(AttendArgs args)
{
    constexpr int C = Operand<ST>::CHUNK, KS = Operand<ST>::KS, NT = 64 * W, STEPS = C / KS;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const scanscam_attend &a = args.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile<ST, D> Y{reinterpret_cast<ST *>(lds)}, Z{reinterpret_cast<ST *>(lds + Tile<ST, D>::WORDS)};
    float *rest = lds + 2 * Tile<ST, D>::WORDS;
    Decays<C> decays{reinterpret_cast<double *>(rest), rest + 2 * C, rest + 3 * C};
    Span span;
    if (!span_of(args, args.first + blockIdx.x, C, span) || span.part == (BACK ? 0 : span.parts - 1)) return;  // (nothing starts from the last one's end)
    const int K = (int)a.K, V = (int)a.V;
    const scanscam_tokens &yt = BACK ? a.gy : a.k, &zt = BACK ? a.q : a.v;
    const int64_t shared = span.head / args.each;
    const ST *y = tensor_at<ST>(yt, span, BACK ? span.head : shared), *z = tensor_at<ST>(zt, span, BACK ? shared : span.head);
    const int inner = BACK ? V : K, outer = BACK ? K : V, row_step = BACK ? 1 : V, col_step = BACK ? V : 1;
    State<ST, D, JT, W> S;
    S.wave = wave;
    S.clear();
    Staged<ST, D, NT, EXACT> sy(y, yt.token, inner), sz(z, zt.token, outer);
    uint32_t decay = 0;
    double whole = 0.0;
    const auto ask = [&](int64_t t) {
        const int n = (int)(span.end - t < C ? span.end - t : C);
        if (wave == 0) decay = decay_at(a, span, t + lane, lane < n);
        sy.load(t, n);
        sz.load(t, n);
    };
    const int64_t chunks = (span.end - span.begin + C - 1) / C;
    const auto token = [&](int64_t c) { return span.begin + (BACK ? chunks - 1 - c : c) * C; };
    if (chunks > 0) ask(token(0));
    settle();
    for (int64_t c = 0; c < chunks; c++) {
        const int n = (int)(span.end - token(c) < C ? span.end - token(c) : C);
        sy.store(Y, n);
        sz.store(Z, n);
        if (wave == 0) {
            decays.fill(decay_of(a, decay));
            whole += decays.sums[C - 1];
        }
        __syncthreads();
        if (c + 1 < chunks) ask(token(c + 1));
        frag_t<ST> own[JT][STEPS];
#pragma unroll
        for (int jt = 0; jt < JT; jt++)
#pragma unroll
            for (int step = 0; step < STEPS; step++) own[jt][step] = Z.columns(S.column(jt), step * KS);
        S.template update<TERMS>(Y, inner, own, BACK ? decays.upto : decays.after, BACK ? a.scale : 1.0f, decays.whole(), S.scale());
        __syncthreads();
    }
    const int64_t border = cut_at(args, span, span.part - (BACK ? 1 : 0));
    S.write((BACK ? args.back_ends : args.ends) + border * K * V, inner, outer, row_step, col_step);
    if (threadIdx.x == 0) {
        // (the rest is 1 at most, so that the product with it stays finite)
        const bool held = whole >= -4096.0 && whole <= 4096.0;
        const double power = __builtin_ceil(held ? whole : whole < 0.0 ? -4096.0 : 4096.0);
        args.powers[border] = {exp2_(held ? whole - power : 0.0), (int32_t)power};
    }
}

// --- gradients of keys and values, backwards in time ------------------------------------------------------------------------------------
// Two kinds of waves share the tiles: those of dk hold H with the values' channels as rows, those of dv with the keys'. Up to 128 channels four waves of
// each; else (one kind's accumulators alone are half of a CU's registers) a workgroup is of one kind. float32 results come from dk's waves: theirs
// are the products in several terms, and dv's waves compute the scores of both.
template <int D> constexpr bool attend_both() { return D < 256; }
template <int D> constexpr int back_waves() { return attend_waves<D>() * (attend_both<D>() ? 2 : 1); }
template <typename ST, int D> struct BackLds {
    static constexpr int C = Operand<ST>::CHUNK, W = attend_waves<D>();
    static constexpr int WORDS = 4 * Tile<ST, D>::WORDS + (attend_both<D>() ? 2 : 1) * Scores<ST>::WORDS + Decays<C>::WORDS + W * C + 2 * W + 4 * (C / 16) * C;
};
template <typename ST, int D, int JT, bool KEYS, bool EXACT> __device__ __forceinline__ void back_pass(const AttendArgs &args, float *lds)
{
    constexpr bool BOTH = attend_both<D>();
    constexpr int C = Operand<ST>::CHUNK, KS = Operand<ST>::KS, W = attend_waves<D>(), NT = 64 * back_waves<D>(), STEPS = C / KS, TT = C / 16, PER = KS / 16, TERMS = KEYS ? kTerms<ST> : kTermsRounded<ST>;
    const scanscam_attend &a = args.a;
    const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all % W, n16 = lane & 15, g = lane >> 4;
    float *at = lds;
    const auto take = [&](int words) { float *p = at; at += words; return p; };
    Tile<ST, D> Q{reinterpret_cast<ST *>(take(Tile<ST, D>::WORDS))}, Kt{reinterpret_cast<ST *>(take(Tile<ST, D>::WORDS))}, Vt{reinterpret_cast<ST *>(take(Tile<ST, D>::WORDS))},
        O{reinterpret_cast<ST *>(take(Tile<ST, D>::WORDS))};
    // do v, of which dk is made, and q k, of which dv is.
    Scores<ST> of_keys{reinterpret_cast<frag_t<ST> *>(take(Scores<ST>::WORDS))}, of_values{BOTH ? reinterpret_cast<frag_t<ST> *>(take(Scores<ST>::WORDS)) : of_keys.p};
    const Scores<ST> scores = KEYS ? of_keys : of_values;
    Decays<C> decays{reinterpret_cast<double *>(take(2 * C)), take(C), take(C)};
    float *red = take(W * C);
    double *over = reinterpret_cast<double *>(take(2 * W));
    // Sums of M over each tile's rows and columns, in 64 bits: their differences are sums over pairs that pass a token, of which the others' must leave nothing.
    double *rows = reinterpret_cast<double *>(take(2 * TT * C)), *cols = reinterpret_cast<double *>(take(2 * TT * C));

    Span span;
    if (!span_of(args, args.first + blockIdx.x, C, span)) return;
    const int64_t shared = span.head / args.each, pair = span.sequence * a.heads + span.head;
    const int K = (int)a.K, V = (int)a.V;
    const ST *q = tensor_at<ST>(a.q, span, shared), *k = tensor_at<ST>(a.k, span, shared), *v = tensor_at<ST>(a.v, span, span.head), *o = tensor_at<ST>(a.gy, span, span.head);
    const Tile<ST, D> inter = KEYS ? Vt : Kt, update_rows = KEYS ? O : Q, mine = KEYS ? Q : O;
    const int inner = KEYS ? V : K, outer = KEYS ? K : V, row_step = KEYS ? 1 : V, col_step = KEYS ? V : 1;
    const int64_t out_step = !KEYS ? a.gv.token : args.part_k != nullptr ? a.heads * K : a.gk.token;
    const int64_t out_first = !KEYS ? span.batch * a.gv.batch + span.head * a.gv.group
                              : args.part_k != nullptr ? (span.batch * a.T * a.heads + span.head) * K : span.batch * a.gk.batch + span.head * a.gk.group;
    const int64_t out_lane = out_first + n16 * out_step + 4 * g;

    State<ST, D, JT, W> H;
    H.wave = wave;
    H.read(start_of(args, span, true), inner, outer, row_step, col_step);

    Staged<ST, D, NT, EXACT> sq(q, a.q.token, K), sk(k, a.k.token, K), sv(v, a.v.token, V), so(o, a.gy.token, V);
    uint32_t decay = 0;
    const auto ask = [&](int64_t t) {
        const int n = (int)(span.end - t < C ? span.end - t : C);
        if (all == 0) decay = decay_at(a, span, t + lane, lane < n);
        sq.load(t, n);
        sk.load(t, n);
        sv.load(t, n);
        so.load(t, n);
    };
    const int64_t chunks = (span.end - span.begin + C - 1) / C;
    if (chunks > 0) ask(span.begin + (chunks - 1) * C);
    settle();
    for (int64_t c = chunks - 1; c >= 0; c--) {
        const int64_t t0 = span.begin + c * C;
        const int n = (int)(span.end - t0 < C ? span.end - t0 : C);
        sq.store(Q, n);
        sk.store(Kt, n);
        sv.store(Vt, n);
        so.store(O, n);
        if (all == 0) decays.fill(decay_of(a, decay));
        __syncthreads();
        if (c > 0) ask(t0 - C);

        // Scores: tiles of 16 tokens t (rows) by 16 tokens s (columns), t >= s, and of both M.
        if (!BOTH || !KEYS) {
            for (int id = D == 256 ? later_uniform((wave + 2) % W) : (wave + 2) % W; id < Scores<ST>::UNITS; id += W) {
                int st, step;
                unit_of<ST>(id, st, step);
                st = TT - 1 - st;
                step = STEPS - 1 - step;
                const double from_s = decays.sums[st * 16 + n16];
                float4v p[PER], other[PER];
#pragma unroll
                for (int h = 0; h < PER; h++) {
                    const int tt = step * PER + h;
                    p[h] = other[h] = float4v{0, 0, 0, 0};
                    if (tt < st) continue;
                    if (BOTH || KEYS) p[h] = score(O, tt * 16, Vt, st * 16, V);
                    other[h] = score(Q, tt * 16, Kt, st * 16, K);
                    double over_t = 0.0;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int s = st * 16 + n16, t = tt * 16 + 4 * g + r;
                        const float w = exp2_(decays.sums[t] - from_s) * a.scale;
                        if (BOTH || KEYS) {
                            const double m = s < t ? p[h][r] * other[h][r] * w : 0.0f, over_s = row_sum(m);
                            over_t += m;
                            if (n16 == 15) rows[st * C + t] = over_s;
                        }
                        p[h][r] = s <= t ? p[h][r] * w : 0.0f;
                        other[h][r] = s <= t ? other[h][r] * w : 0.0f;
                    }
                    if (BOTH || KEYS) {
                        over_t = column_sum4(over_t);
                        if (g == 0) cols[tt * C + st * 16 + n16] = over_t;
                    }
                }
                if (BOTH || KEYS) of_keys.put_step(st, step, p);
                if (BOTH || !KEYS) of_values.put_step(st, step, other);
            }
        }
        float4v acc[TT][JT];
        const float scaled = H.template times<TERMS>(inter, inner, acc), unscale = 1.0f / scaled;
        frag_t<ST> own[JT][STEPS];
#pragma unroll
        for (int jt = 0; jt < JT; jt++)
#pragma unroll
            for (int step = 0; step < STEPS; step++) own[jt][step] = mine.columns(H.column(jt), step * KS);
        __syncthreads();

#pragma unroll
        for (int st = 0; st < TT; st++) {
            const int s = st * 16 + n16;
            const float after = decays.after[s] * unscale;
            float write = 0.0f;
#pragma unroll
            for (int jt = 0; jt < JT; jt++) {
                acc[st][jt] *= after;
                if constexpr (KEYS) {
                    float key[4];
                    Kt.four(s, H.column(jt) + 4 * g, key);
#pragma unroll
                    for (int r = 0; r < 4; r++) write += key[r] * acc[st][jt][r];
                }
            }
#pragma unroll
            for (int step = st / PER; step < STEPS; step++) scores.times(own, st, step, acc[st]);
            if (s < n) {
                const int64_t row = out_lane + (t0 + st * 16) * out_step;
#pragma unroll
                for (int jt = 0; jt < JT; jt++) {
                    const int col = H.column(jt), there = outer - 4 * g;
                    if constexpr (!KEYS) {
                        put4<EXACT>(static_cast<ST *>(a.gv.p) + row, col, there, acc[st][jt]);
                    } else if (args.part_k != nullptr) {
                        put4<EXACT>(args.part_k + row, col, there, acc[st][jt]);
                    } else {
                        put4<EXACT>(static_cast<ST *>(a.gk.p) + row, col, there, acc[st][jt]);
                    }
                }
            }
            if constexpr (KEYS) {
                write = column_sum4(write);
                if (g == 0) red[wave * C + s] = write;
            }
        }
        H.template update<TERMS>(update_rows, inner, own, decays.upto, a.scale, decays.whole(), scaled);
        if constexpr (KEYS) {
            const bool border = args.cross != nullptr && t0 > span.from && (t0 - span.from) % (kBorder * C) == 0;
            const int64_t at_border = border ? border_at(args, span.batch, t0, C, span.head) : 0;
            if (border) {
                const double sum = sums_upto(H.kept(args.borders + at_border * D * D, inner, outer));
                if (lane == 63) over[wave] = sum;
            }
            __syncthreads();
            if (border && all == 0 && lane == 0) {
                double sum = 0.0;
                for (int w = 0; w < W; w++) sum += over[w];
                args.cross[at_border] = sum;
            }
            if (args.writes != nullptr && threadIdx.x < (unsigned)n) {
                float write = 0.0f;
                for (int w = 0; w < W; w++) write += red[w * C + threadIdx.x];
                const int t = threadIdx.x;
                double inside = 0.0;
                for (int st = 0; st <= t / 16; st++) inside += rows[st * C + t];
                for (int tt = t / 16; tt < TT; tt++) inside -= cols[tt * C + t];
                const int64_t at = span.head * args.tokens + span.batch * a.T + t0 + t;
                args.writes[at] = write;
                args.inside[at] = inside;
            }
        } else {
            __syncthreads();
        }
    }
    if constexpr (KEYS)
        if (span.part == 0 && a.gstate_in != nullptr) H.write(a.gstate_in + pair * K * V, inner, outer, row_step, col_step);
}
// JK, JV: column tiles of dk's and dv's waves. (The kinds meet at the same barriers: each pass has three a chunk.)
template <typename ST, int D, int JK, int JV, bool EXACT> __global__ __launch_bounds__(64 * back_waves<D>(), 2) void attend_back_kernel(AttendArgs args)
{
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (attend_both<D>() ? wave < attend_waves<D>() : blockIdx.y == 0) back_pass<ST, D, JK, true, EXACT>(args, lds);
    else back_pass<ST, D, JV, false, EXACT>(args, lds);
}

// --- launches by type ---------------------------------------------------------------------------------------------------------------------
enum AttendPass { kOutputs, kQueries, kKeysAndValues, kEnds, kBackEnds };

// Channels that a call's tiles have room for.
inline int attend_width(const scanscam_attend &a)
{
    const int64_t most = a.K > a.V ? a.K : a.V;
    return most <= 64 ? 64 : most <= 128 ? 128 : 256;
}

template <typename ST> hipError_t launch_attend(AttendPass pass, int64_t units, hipStream_t stream, const AttendArgs &args);

// Units of several launches where one would have 2^32 threads.
template <auto Kernel, int WORDS> hipError_t launch_attend_units(int64_t units, unsigned kinds, int threads, hipStream_t stream, AttendArgs args)
{
    static_assert(WORDS * 4 <= 160 * 1024, "a workgroup's shared memory");
    constexpr int64_t most = 1 << 22;
    for (int64_t first = 0; first < units; first += most) {
        args.first = first;
        const hipError_t err = launch_wide<Kernel>(dim3((unsigned)(units - first < most ? units - first : most), kinds), threads, WORDS, WORDS, stream, args);
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

// Column tiles of a wave by the columns that there are: a head of up to 64 (of the 256 kind 128) leaves half of the waves' registers and products out.
template <typename ST, int D, bool EXACT> hipError_t launch_attend_with(AttendPass pass, int64_t units, hipStream_t stream, const AttendArgs &args)
{
    constexpr int WAVES = attend_waves<D>(), EJ = D == 256 ? 2 : 1, EW = D / 16 / EJ;  // (EJ, EW: of the ends, whole)
    // HALF: column tiles of a wave for a side that fills no more than half of them ([25, 656, 5 heads of 194 and 27] in bf16: 88 us, 198 with all).
    constexpr int threads = 64 * WAVES, back_threads = 64 * back_waves<D>(), ALL = D == 64 ? 1 : 2, HALF = 1, T = kTerms<ST>;
    constexpr int GW = query_waves<ST, D>(), GJ = D / 16 / GW;  // (of the queries' gradients, whole)
    constexpr int out = AttendLds<ST, WAVES, D, false>::WORDS, grad_half = AttendLds<ST, WAVES, D, true>::WORDS, grad = AttendLds<ST, GW, D, true>::WORDS, back = BackLds<ST, D>::WORDS, ends = EndsLds<ST, D>::WORDS;
    const bool k_half = ALL == 2 && args.a.K <= D / 2, v_half = ALL == 2 && args.a.V <= D / 2;
    const unsigned kinds = attend_both<D>() ? 1 : 2;
    switch (pass) {
    case kOutputs:
        return v_half ? launch_attend_units<attend_kernel<ST, D, HALF, WAVES, false, EXACT>, out>(units, 1, threads, stream, args)
                      : launch_attend_units<attend_kernel<ST, D, ALL, WAVES, false, EXACT>, out>(units, 1, threads, stream, args);
    case kQueries:
        return k_half ? launch_attend_units<attend_kernel<ST, D, HALF, WAVES, true, EXACT>, grad_half>(units, 1, threads, stream, args)
                      : launch_attend_units<attend_kernel<ST, D, GJ, GW, true, EXACT>, grad>(units, 1, 64 * GW, stream, args);
    case kKeysAndValues:  // (both are not halves at once)
        if (k_half) return launch_attend_units<attend_back_kernel<ST, D, HALF, ALL, EXACT>, back>(units, kinds, back_threads, stream, args);
        if (v_half) return launch_attend_units<attend_back_kernel<ST, D, ALL, HALF, EXACT>, back>(units, kinds, back_threads, stream, args);
        return launch_attend_units<attend_back_kernel<ST, D, ALL, ALL, EXACT>, back>(units, kinds, back_threads, stream, args);
    case kEnds:
        return v_half ? launch_attend_units<ends_kernel<ST, D, HALF, WAVES, false, T, EXACT>, ends>(units, 1, threads, stream, args)
                      : launch_attend_units<ends_kernel<ST, D, EJ, EW, false, T, EXACT>, ends>(units, 1, 64 * EW, stream, args);
    default:
        return k_half ? launch_attend_units<ends_kernel<ST, D, HALF, WAVES, true, T, EXACT>, ends>(units, 1, threads, stream, args)
                      : launch_attend_units<ends_kernel<ST, D, EJ, EW, true, T, EXACT>, ends>(units, 1, 64 * EW, stream, args);
    }
}
template <typename ST, int D> hipError_t launch_attend_of(AttendPass pass, int64_t units, hipStream_t stream, const AttendArgs &args)
{
    constexpr int64_t vector = 16 / sizeof(ST);
    return args.a.K % vector == 0 && args.a.V % vector == 0 ? launch_attend_with<ST, D, true>(pass, units, stream, args) : launch_attend_with<ST, D, false>(pass, units, stream, args);
}
#define SCANSCAM_DEFINE_ATTEND_LAUNCH(ST)                                                                                                        \
    template <> hipError_t launch_attend<ST>(AttendPass pass, int64_t units, hipStream_t stream, const AttendArgs &args)                         \
    {                                                                                                                                            \
        const int width = attend_width(args.a);                                                                                                  \
        return width == 64    ? launch_attend_of<ST, 64>(pass, units, stream, args)                                                              \
               : width == 128 ? launch_attend_of<ST, 128>(pass, units, stream, args)                                                             \
                              : launch_attend_of<ST, 256>(pass, units, stream, args);                                                            \
    }

}  // namespace scanscam
