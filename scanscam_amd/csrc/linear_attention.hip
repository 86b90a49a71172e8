// C ABI of linear attention (declared in include/scanscam_attention.h): argument checks, launch shapes, launches; single tokens' steps; and the
// kernels whose work does not depend on the activations' type.
#include "linear_attention_kernels.hpp"

namespace scanscam {

// The states at the borders between parts, out of what each adds: in the parts' order, or from the last part on (gradients). AHEAD borders are asked for
// together: one after the other each would be a trip to memory (128 parts of 4 heads: 37 us, 24 by sixteens). A lane takes VALUES of them.
template <int AHEAD, int VALUES, bool BACK> __global__ __launch_bounds__(256) void join_kernel(AttendArgs args)
{
    const scanscam_attend &a = args.a;
    const int64_t pair = args.first + blockIdx.x, values = a.K * a.V, at = (int64_t)blockIdx.y * 256 * VALUES + threadIdx.x;
    Span s;
    s.sequence = pair / a.heads;
    s.head = (int)(pair % a.heads);
    s.parts = args.parts;
    s.cut = s.sequence * (s.parts - 1);
    if (a.offsets != nullptr && !count_parts(args, s.sequence, 0, s)) return;
    const int borders = s.parts - 1;
    if (borders == 0) return;
    const float *given = BACK ? a.gstate_out : a.state_in;
    float *ends = (BACK ? args.back_ends : args.ends) + at;
    const auto border = [&](int i) { return cut_at(args, s, BACK ? borders - 1 - i : i); };
    float run[VALUES];
#pragma unroll
    for (int v = 0; v < VALUES; v++) run[v] = given != nullptr && at + 256 * v < values ? given[pair * values + at + 256 * v] : 0.0f;
    for (int i0 = 0; i0 < borders; i0 += AHEAD) {
        float adds[AHEAD][VALUES];
        AttendArgs::Power decay[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int there = i0 + i < borders ? i0 + i : borders - 1;
            decay[i] = args.powers[border(there)];
#pragma unroll
            for (int v = 0; v < VALUES; v++) adds[i][v] = at + 256 * v < values ? ends[border(there) * values + 256 * v] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (i0 + i < borders) {
#pragma unroll
                for (int v = 0; v < VALUES; v++) {
                    run[v] = __builtin_ldexpf(run[v] * decay[i].rest, decay[i].whole) + adds[i][v];
                    if (at + 256 * v < values) ends[border(i0 + i) * values + 256 * v] = run[v];
                }
            }
    }
}

// Gradients of decays out of what every token reads and writes (the formula is in linear_attention_kernels.hpp). A workgroup takes the chunks
// between two borders, a wave each, backwards from the later one's product of state and gradient.
template <int C> __global__ __launch_bounds__(64 * kBorder) void decays_kernel(AttendArgs args)
{
    const scanscam_attend &a = args.a;
    AttendArgs whole = args;
    whole.per = 0;
    Span span;
    if (!span_of(whole, args.first + blockIdx.x, C, span)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ double all_reads[kBorder], all_writes[kBorder];
    __shared__ bool closed[kBorder];
    const int64_t chunks = (span.length + C - 1) / C, base = span.head * args.tokens + span.batch * a.T;
    for (int64_t first = (int64_t)blockIdx.y * kBorder; first < chunks; first += (int64_t)gridDim.y * kBorder) {
        const int64_t c = first + kBorder - 1 - wave, t = span.begin + c * C + lane;
        const bool there = lane < C && t < span.end;
        const double read = there ? args.reads[base + t] : 0.0, write = there ? args.writes[base + t] : 0.0, pair = there ? args.inside[base + t] : 0.0;
        const double reads = sums_upto(read), writes = sums_upto(write), pairs = sums_upto(pair), all_pairs = read_lane(pairs, 63), decay = read_lane(sums_upto(decay_of(a, decay_at(a, span, t, there))), 63);
        if (lane == 63) {
            all_reads[wave] = reads;
            all_writes[wave] = writes;
            closed[wave] = exp2_(decay) == 0.0f || (c == 0 && a.state_in == nullptr);  // (as for the states: nothing passes the chunk, or there is nothing before it)
        }
        __syncthreads();
        double end = first + kBorder < chunks ? args.cross[border_at(args, span.batch, span.from + (first + kBorder) * C, C, span.head)] : args.last[args.first + blockIdx.x];
        for (int w = 0; w < wave; w++) end = (closed[w] ? 0.0 : end - all_writes[w]) + all_reads[w];
        const double past = closed[wave] ? 0.0 : end - all_writes[wave];
        if (there)
            args.decays[(span.batch * a.T + t) * a.heads + span.head] =
                (float)(past + (all_reads[wave] - reads + read) + (writes - write) + (all_pairs - pairs + pair));
        __syncthreads();
    }
}

// Gradients of shared queries or keys: over the heads that share them, in order (of no heads they are zero).
struct Shared {
    const float *part;  // [tokens][groups * each][K]
    scanscam_tokens out;
    int64_t tokens, T, token0;
    int32_t groups, each, K;
};
template <typename ST> __global__ __launch_bounds__(256) void shared_kernel(Shared a)
{
    const int fours = (a.K + 3) / 4, row = a.groups * fours;
    const int64_t index = (int64_t)blockIdx.x * 256 + threadIdx.x, token = a.token0 + index / row;
    if (token >= a.tokens) return;
    const int rest = (int)(index % row), group = rest / fours, at = rest % fours * 4, count = a.K - at;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const float *p = a.part + (token * a.groups + group) * a.each * a.K + at;
    for (int h = 0; h < a.each; h++, p += a.K) {
        float f[4];
        load_part<float, 4>(p, count, f);
#pragma unroll
        for (int r = 0; r < 4; r++) sum[r] += f[r];
    }
    store_some<ST, 4>(static_cast<ST *>(a.out.p) + token / a.T * a.out.batch + token % a.T * a.out.token + group * a.out.group + at, count, sum);
}

// One token: S = e^g S + k v^T, y = scale S^T q. Memory bounds it, the states read and written. A workgroup takes `width` columns of a head's
// state; `lanes` lanes hold four columns each, and rows go round the workgroup, four
// under way at once (256 x 16 states of 128 x 128 from HBM, 537 MB: 114 us, 4.7 TB/s; eight 123, sixteen 131, for more registers leave fewer waves).
struct StepArgs {
    scanscam_attend_step a;
    int32_t lanes, pieces, each;
    int64_t first;
};
template <typename ST> __global__ __launch_bounds__(256) void attend_step_kernel(StepArgs args)
{
    const scanscam_attend_step &a = args.a;
    __shared__ float keys[256], queries[256];
    __shared__ __attribute__((aligned(16))) float4v sums[256];
    const int64_t unit = args.first + blockIdx.x, row = unit / args.pieces / a.heads;
    const int piece = (int)(unit % args.pieces), head = (int)(unit / args.pieces % a.heads), shared = head / args.each;
    const int K = (int)a.K, V = (int)a.V, lane = threadIdx.x % args.lanes, row0 = threadIdx.x / args.lanes, stride = 256 / args.lanes;
    const int col = (piece * args.lanes + lane) * 4, count = V - col;
    const int64_t slot = a.slot == nullptr ? row : index_at(a.slot, a.slot64, row);
    ST *y = static_cast<ST *>(a.y.p) + row * a.y.token + head * a.y.group + col;
    if (slot < 0 || slot >= a.slots) {
        const float zeros[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (row0 == 0 && count > 0) store_some<ST, 4>(y, count, zeros);
        return;
    }
    float *state = a.state + (slot * a.heads + head) * (int64_t)K * V + col;
    constexpr int UNROLL = 4;
    float4v s[UNROLL];
    const auto ask = [&](int i0) {
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const int i = i0 + u * stride;
            float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (i < K && count > 0) load_part<float, 4>(state + i * V, count, f);
            s[u] = float4v{f[0], f[1], f[2], f[3]};
        }
    };
    ask(row0);
    if ((int)threadIdx.x < K) {
        keys[threadIdx.x] = (float)static_cast<const ST *>(a.k.p)[row * a.k.token + shared * a.k.group + threadIdx.x];
        queries[threadIdx.x] = (float)static_cast<const ST *>(a.q.p)[row * a.q.token + shared * a.q.group + threadIdx.x];
    }
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (count > 0) load_part<ST, 4>(static_cast<const ST *>(a.v.p) + row * a.v.token + head * a.v.group + col, count, v);
    const float g = a.decay.p == nullptr ? 0.0f : param(scanscam_param{a.decay.p, a.decay_dtype, 0}, row * a.decay.token + head);
    const float decay = __builtin_amdgcn_exp2f((float)((double)g * 1.4426950408889634074));
    __syncthreads();
    float4v sum{0, 0, 0, 0};
    for (int i0 = row0; i0 < K; i0 += UNROLL * stride) {
        if (i0 != row0) ask(i0);
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const int i = i0 + u * stride;
            if (i >= K) continue;
            const float k = keys[i], q = queries[i];
            float f[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                f[r] = __builtin_fmaf(decay, s[u][r], k * v[r]);
                sum[r] = __builtin_fmaf(q, f[r], sum[r]);
            }
            if (count > 0) store_some<float, 4>(state + i * V, count, f);
        }
    }
    sums[threadIdx.x] = sum;
    for (int half = stride / 2; half > 0; half /= 2) {  // (both are powers of two)
        __syncthreads();
        if (row0 < half) sums[threadIdx.x] = sum = sum + sums[threadIdx.x + half * args.lanes];
    }
    if (row0 == 0 && count > 0) {
        const float out[4] = {sum[0] * a.scale, sum[1] * a.scale, sum[2] * a.scale, sum[3] * a.scale};
        store_some<ST, 4>(y, count, out);
    }
}

}  // namespace scanscam

namespace {

using namespace scanscam;

int check_near(const scanscam_tokens &t, int size)
{
    SCANSCAM_CHECK(check_tokens(t, size));
    return t.token >= SCANSCAM_MOST_TOKEN_STRIDE ? SCANSCAM_EINVAL : SCANSCAM_OK;
}

int check_heads(int64_t heads, int64_t groups, int64_t K, int64_t V, int dtype, const scanscam_tokens &decay, int decay_dtype)
{
    if (heads < 0 || groups < 1 || heads % groups != 0 || K < 1 || K > SCANSCAM_MOST_HEAD || V < 1 || V > SCANSCAM_MOST_HEAD) return SCANSCAM_EINVAL;
    if (heads * (K > V ? K : V) > kMostChannels) return SCANSCAM_EINVAL;
    if (activation_size(dtype) == 0) return SCANSCAM_EDTYPE;
    if (decay.p == nullptr) return SCANSCAM_OK;
    if (activation_size(decay_dtype) == 0) return SCANSCAM_EDTYPE;
    return check_tokens(decay, activation_size(decay_dtype));
}

constexpr int64_t kAttendMostParts = 1024;

// `back`: also what a backward call reads and writes.
int check_attend(const scanscam_attend *a, bool back)
{
    if (a == nullptr) return SCANSCAM_EINVAL;
    if (a->batch < 0 || a->T < 0 || a->T >= kMostTokens || a->sequences < 0 || a->sequences >= kMostTokens || a->parts < 0 || a->parts > kAttendMostParts) return SCANSCAM_EINVAL;
    if (a->offsets != nullptr ? a->batch != 1 || a->sequences < 1 : a->sequences != a->batch) return SCANSCAM_EINVAL;
    if (a->batch > 0 && a->T > (kMostTokens - 1) / a->batch) return SCANSCAM_EINVAL;
    SCANSCAM_CHECK(check_heads(a->heads, a->groups, a->K, a->V, a->dtype, a->decay, a->decay_dtype));
    if (misaligned(a->offsets, a->offsets64 ? 8 : 4)) return SCANSCAM_EALIGN;
    if (misaligned(a->saved, 16)) return SCANSCAM_EALIGN;
    for (const void *p : {(const void *)a->state_in, (const void *)a->state_out, (const void *)a->gdecay, (const void *)a->gstate_out, (const void *)a->gstate_in})
        if (misaligned(p, 4)) return SCANSCAM_EALIGN;
    if (a->batch * a->T == 0 || a->heads == 0) return SCANSCAM_OK;
    const int size = activation_size(a->dtype);
    for (const scanscam_tokens *t : {&a->q, &a->k, &a->v}) SCANSCAM_CHECK(check_near(*t, size));
    if (!back) return check_tokens(a->y, size);
    SCANSCAM_CHECK(check_near(a->gy, size));
    for (const scanscam_tokens *t : {&a->gq, &a->gk, &a->gv}) SCANSCAM_CHECK(check_tokens(*t, size));
    return SCANSCAM_OK;
}

int chunk_of(const scanscam_attend &a) { return a.dtype == SCANSCAM_F32 ? Operand<float>::CHUNK : Operand<__bf16>::CHUNK; }

// How time is shared out. Parts cost a second pass over keys and values, and states at their borders; they are for calls with fewer heads of sequences
// than it takes to fill the card: up to 512 parts of no less than four chunks. ([8, 4096, 16 x 128] in bf16 with gradients
// by 1, 2, 4, 8 parts: 1.74, 1.16, 0.99, 1.09 ms; 30001 tokens of four heads in float32 by 64, 128: 425, 416 us.) 512 is two workgroups on each of 256 CUs, which holds for the
// forward pass of up to 128 channels. Backwards, and of more channels, a CU has one, so that where two parts make no round of workgroups fewer one part is better:
// [12, 2048, 16 x 128] in bf16 with gradients takes 940 us by the rule's two and 820 by one; [8, 2048, 8 x 256 x 256] 1810 by its eight and 1530 by four.
// Of sequences behind each other the host knows all tokens only. Their parts have one length, which makes 384 of all tokens, and the sequences' last ones, shorter as
// they are, come on top: 8021 tokens of 13 sequences of 16 heads, from equal ones to one with two thirds of the tokens, 99 - 113 us; with 512 114 - 124,
// 256 117 - 125, and in one part each 114 - 492. A sequence that is no longer than a part is one, and costs an empty workgroup in either of the passes more.
// Every workgroup counts the sequences, 64 in a trip to memory: more than 256 are not shared out, nor heads of sequences that fill the card by themselves
// (6000 tokens and 299 short sequences of four heads: 550 us; with 249 short ones 115).
struct Plan {
    int64_t per;                         // tokens of a part, whole chunks; 0: all of the sequence
    int64_t units, borders;              // heads of parts; borders between parts, at most
    int parts;                           // of a sequence of T tokens
};
Plan plan_of(const scanscam_attend &a)
{
    const int chunk = chunk_of(a);
    const int64_t pairs = a.sequences * a.heads, chunks = ceil_div(a.T, chunk);
    Plan p{0, pairs, 0, 1};
    if (a.offsets != nullptr && a.sequences != 1) {
        int64_t per = a.parts > 0 ? ceil_div(chunks, a.parts) : ceil_div(chunks * a.heads, 384);
        if (a.parts == 0) per = a.sequences > 256 || pairs >= 4096 ? chunks : per < 4 ? 4 : per;
        if (per >= chunks) return p;
        p.per = per * chunk;
        p.borders = a.T / p.per;
        p.units = (a.sequences + p.borders) * a.heads;
        p.parts = (int)ceil_div(chunks, per);
        return p;
    }
    int64_t parts = a.parts;
    if (parts == 0 && pairs > 0 && pairs < 256) parts = 512 / pairs < chunks / 4 ? 512 / pairs : chunks / 4;
    if (parts < 2) return p;
    p.per = ceil_div(chunks, parts) * chunk;
    if (p.per == 0) p.per = chunk;
    p.parts = (int)parts;
    p.borders = a.sequences * (parts - 1);
    p.units = pairs * parts;
    return p;
}

// What the workspace holds, in order; each piece begins on 16 bytes.
struct Pieces {
    size_t ends, back_ends, powers, reads, writes, inside, last, borders, cross, part_q, part_k, decays, bytes;
    int64_t most_borders;
};
int64_t ends_values(const scanscam_attend &a, const Plan &plan) { return plan.borders * a.heads * a.K * a.V; }
Pieces pieces_of(const scanscam_attend &a, bool back, const Plan &plan)
{
    Pieces p{};
    const auto take = [&](bool there, int64_t count, size_t size) {
        const size_t at = p.bytes;
        if (there) p.bytes += ((size_t)count * size + 15) / 16 * 16;
        return at;
    };
    const int64_t pairs = a.sequences * a.heads, values = ends_values(a, plan), tokens = a.batch * a.T;
    p.ends = take(!back, values, 4);  // (a backward call has the forward one's)
    p.powers = take(true, plan.borders * a.heads, sizeof(AttendArgs::Power));
    if (!back) return p;
    p.back_ends = take(true, values, 4);
    p.reads = take(true, tokens * a.heads, 4);
    p.writes = take(true, tokens * a.heads, 4);
    p.inside = take(true, tokens * a.heads, 8);
    p.last = take(true, pairs, 8);
    p.most_borders = a.T / (kBorder * chunk_of(a)) + 1;
    const int64_t borders = a.T > kBorder * chunk_of(a) ? a.batch * p.most_borders * a.heads : 0, width = attend_width(a);
    p.borders = take(borders > 0, borders * width * width, 4);
    p.cross = take(borders > 0, borders, 8);
    p.part_q = take(a.groups < a.heads, tokens * a.heads * a.K, 4);
    p.part_k = take(a.groups < a.heads, tokens * a.heads * a.K, 4);
    p.decays = take(a.decay_fixed != 0, tokens * a.heads, 4);
    return p;
}

hipError_t run(AttendPass pass, int64_t units, hipStream_t stream, const AttendArgs &args)
{
    switch (args.a.dtype) {
    case SCANSCAM_F32: return launch_attend<float>(pass, units, stream, args);
    case SCANSCAM_BF16: return launch_attend<__bf16>(pass, units, stream, args);
    default: return launch_attend<_Float16>(pass, units, stream, args);
    }
}

// The states at the borders between parts.
template <int AHEAD, int VALUES> hipError_t join_with(const AttendArgs &args, bool back, int64_t pairs, hipStream_t stream)
{
    const dim3 grid((unsigned)pairs, (unsigned)ceil_div(args.a.K * args.a.V, 256 * VALUES));
    return launch_op(back ? join_kernel<AHEAD, VALUES, true> : join_kernel<AHEAD, VALUES, false>, grid, dim3(256), 0, stream, args);
}
hipError_t starts(AttendArgs args, bool back, AttendPass pass, int64_t units, hipStream_t stream)
{
    const int64_t pairs = args.a.sequences * args.a.heads;
    hipError_t err = run(pass, units, stream, args);
    constexpr int64_t most = 1 << 22;
    // Four values a lane where their states are half a million or more: there are workgroups enough without. (Packed prompts' 208 states of 128 x 128: 21 us, 56 by one;
    // four parts of 128 of them 10 us, 16 by one; 127 parts of four of 48 x 72 33 us, 19 by one.)
    const bool many = pairs * args.a.K * args.a.V >= 1 << 19, few = args.parts <= 4;
    for (args.first = 0; args.first < pairs && err == hipSuccess; args.first += most) {
        const int64_t now = pairs - args.first < most ? pairs - args.first : most;
        if (few) err = many ? join_with<4, 4>(args, back, now, stream) : join_with<4, 1>(args, back, now, stream);
        else err = many ? join_with<16, 4>(args, back, now, stream) : join_with<16, 1>(args, back, now, stream);
    }
    return err;
}

template <typename ST> hipError_t join_shared(Shared s, hipStream_t stream)
{
    const int64_t row = (int64_t)s.groups * ceil_div(s.K, 4), most = (int64_t(1) << 31) / row;
    const int64_t all = s.tokens;
    hipError_t err = hipSuccess;
    for (; s.token0 < all && err == hipSuccess; s.token0 += most) {
        const int64_t now = all - s.token0 < most ? all - s.token0 : most;
        s.tokens = s.token0 + now;
        err = launch_op(shared_kernel<ST>, dim3((unsigned)ceil_div(now * row, 256)), dim3(256), 0, stream, s);
    }
    return err;
}

// Gradients of queries and keys out of the heads' (each: heads that share one).
hipError_t join_both(const scanscam_attend &a, int32_t each, const float *part_q, const float *part_k, hipStream_t stream)
{
    hipError_t err = hipSuccess;
    for (int i = 0; i < 2 && err == hipSuccess; i++) {
        const Shared sum{i == 0 ? part_q : part_k, i == 0 ? a.gq : a.gk, a.batch * a.T, a.T, 0, (int32_t)a.groups, each, (int32_t)a.K};
        err = a.dtype == SCANSCAM_F32 ? join_shared<float>(sum, stream) : a.dtype == SCANSCAM_BF16 ? join_shared<__bf16>(sum, stream) : join_shared<_Float16>(sum, stream);
    }
    return err;
}

template <typename ST> hipError_t launch_attend_step(const StepArgs &step, hipStream_t stream)
{
    StepArgs args = step;
    const int64_t units = args.a.rows * args.a.heads * args.pieces, most = (int64_t(1) << 32) / 256 - 1;
    hipError_t err = hipSuccess;
    for (args.first = 0; args.first < units && err == hipSuccess; args.first += most)
        err = launch_op(attend_step_kernel<ST>, dim3((unsigned)(units - args.first < most ? units - args.first : most)), dim3(256), 0, stream, args);
    return err;
}

int code(hipError_t err) { return err == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH; }

bool sizes_fit(const scanscam_attend *a)
{
    return a != nullptr && a->batch >= 0 && a->T >= 0 && a->T < kMostTokens && a->sequences >= 0 && a->sequences < kMostTokens && a->parts >= 0 && a->parts <= kAttendMostParts &&
           (a->batch == 0 || a->T <= (kMostTokens - 1) / a->batch) && check_heads(a->heads, a->groups, a->K, a->V, a->dtype, scanscam_tokens{}, 0) == SCANSCAM_OK;
}

}  // namespace

extern "C" {

size_t scanscam_attend_saved_bytes(const scanscam_attend *a)
{
    return sizes_fit(a) ? (size_t)ends_values(*a, plan_of(*a)) * sizeof(float) : 0;
}

size_t scanscam_attend_workspace_bytes(const scanscam_attend *a, int direction)
{
    return sizes_fit(a) ? pieces_of(*a, direction == SCANSCAM_BACKWARD, plan_of(*a)).bytes : 0;
}

int scanscam_attend_fwd(const scanscam_attend *a, void *stream)
{
    SCANSCAM_CHECK(check_attend(a, false));
    if (a->sequences == 0 || a->heads == 0 || (a->batch * a->T == 0 && a->state_out == nullptr)) return SCANSCAM_OK;
    const Plan plan = plan_of(*a);
    const Pieces at = pieces_of(*a, false, plan);
    if (at.bytes > 0 && (a->workspace == nullptr || a->workspace_bytes < at.bytes)) return SCANSCAM_EWORKSPACE;
    if (misaligned(a->workspace, 16)) return SCANSCAM_EALIGN;
    char *w = static_cast<char *>(a->workspace);
    AttendArgs args{};
    args.a = *a;
    args.tokens = a->batch * a->T;
    args.per = plan.per;
    args.parts = plan.parts;
    args.cuts = plan.borders;
    args.each = (int32_t)(a->heads / a->groups);
    args.ends = a->saved != nullptr ? static_cast<float *>(a->saved) : reinterpret_cast<float *>(w + at.ends);
    args.powers = reinterpret_cast<AttendArgs::Power *>(w + at.powers);
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t err = hipSuccess;
    if (plan.borders > 0) err = starts(args, false, kEnds, plan.units, s);
    if (err == hipSuccess) err = run(kOutputs, plan.units, s, args);
    return code(err);
}

int scanscam_attend_bwd(const scanscam_attend *a, void *stream)
{
    SCANSCAM_CHECK(check_attend(a, true));
    if (a->gdecay != nullptr && a->decay.p == nullptr) return SCANSCAM_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a->heads == 0) {
        if (a->batch * a->T == 0) return SCANSCAM_OK;
        if (a->groups > kMostChannels / a->K) return SCANSCAM_EINVAL;
        for (const scanscam_tokens *t : {&a->gq, &a->gk}) SCANSCAM_CHECK(check_tokens(*t, activation_size(a->dtype)));
        return code(join_both(*a, 0, nullptr, nullptr, s));
    }
    if (a->sequences == 0 || (a->batch * a->T == 0 && a->gstate_in == nullptr))
        return a->gdecay != nullptr && a->decay_fixed ? code(column_sum({nullptr, 0, 0, {a->gdecay}, {a->heads}}, s)) : SCANSCAM_OK;
    const Plan plan = plan_of(*a);
    const Pieces at = pieces_of(*a, true, plan);
    if (at.bytes > 0 && (a->workspace == nullptr || a->workspace_bytes < at.bytes)) return SCANSCAM_EWORKSPACE;
    if (misaligned(a->workspace, 16)) return SCANSCAM_EALIGN;
    if (plan.borders > 0 && a->saved == nullptr) return SCANSCAM_EINVAL;
    char *w = static_cast<char *>(a->workspace);
    AttendArgs args{};
    args.a = *a;
    args.tokens = a->batch * a->T;
    args.per = plan.per;
    args.parts = plan.parts;
    args.cuts = plan.borders;
    args.each = (int32_t)(a->heads / a->groups);
    args.ends = static_cast<float *>(a->saved);
    args.back_ends = reinterpret_cast<float *>(w + at.back_ends);
    args.powers = reinterpret_cast<AttendArgs::Power *>(w + at.powers);
    if (a->gdecay != nullptr) {
        args.reads = reinterpret_cast<float *>(w + at.reads);
        args.writes = reinterpret_cast<float *>(w + at.writes);
        args.inside = reinterpret_cast<double *>(w + at.inside);
        args.last = reinterpret_cast<double *>(w + at.last);
        args.most_borders = at.most_borders;
        if (at.cross > at.borders) {  // (some sequence may have one)
            args.borders = reinterpret_cast<float *>(w + at.borders);
            args.cross = reinterpret_cast<double *>(w + at.cross);
        }
        args.decays = a->decay_fixed ? reinterpret_cast<float *>(w + at.decays) : a->gdecay;
    }
    if (args.each > 1) {
        args.part_q = reinterpret_cast<float *>(w + at.part_q);
        args.part_k = reinterpret_cast<float *>(w + at.part_k);
    }
    const int64_t pairs = a->sequences * a->heads;
    hipError_t err = hipSuccess;
    if (plan.borders > 0) err = starts(args, true, kBackEnds, plan.units, s);
    if (err == hipSuccess) err = run(kQueries, plan.units, s, args);
    if (err == hipSuccess) err = run(kKeysAndValues, plan.units, s, args);
    if (a->gdecay != nullptr && err == hipSuccess) {
        constexpr int64_t most = 1 << 21;
        for (args.first = 0; args.first < pairs && err == hipSuccess; args.first += most) {
            const int64_t batches = ceil_div(a->T, kBorder * chunk_of(*a)), rounds = batches < 1 ? 1 : batches < 64 ? batches : 64;
            const dim3 grid((unsigned)(pairs - args.first < most ? pairs - args.first : most), (unsigned)rounds), block(64 * kBorder);
            err = chunk_of(*a) == 32 ? launch_op(decays_kernel<32>, grid, block, 0, s, args) : launch_op(decays_kernel<64>, grid, block, 0, s, args);
        }
        if (a->decay_fixed && err == hipSuccess) err = column_sum({args.decays, args.tokens, a->heads, {a->gdecay}, {a->heads}}, s);
    }
    if (args.each > 1 && err == hipSuccess) err = join_both(*a, args.each, args.part_q, args.part_k, s);
    return code(err);
}

int scanscam_attend_step_fwd(const scanscam_attend_step *a, void *stream)
{
    if (a == nullptr || a->rows < 0 || a->rows >= kMostTokens || a->slots < 0) return SCANSCAM_EINVAL;
    SCANSCAM_CHECK(check_heads(a->heads, a->groups, a->K, a->V, a->dtype, a->decay, a->decay_dtype));
    if (a->rows == 0 || a->heads == 0) return SCANSCAM_OK;
    const int size = activation_size(a->dtype);
    for (const scanscam_tokens *t : {&a->q, &a->k, &a->v, &a->y}) SCANSCAM_CHECK(check_tokens(*t, size));
    if (a->slots > 0 && a->state == nullptr) return SCANSCAM_EINVAL;
    if (misaligned(a->slot, a->slot64 ? 8 : 4) || misaligned(a->state, 4)) return SCANSCAM_EALIGN;
    // Lanes for a whole row of the state, or fewer where that leaves CUs without a workgroup.
    StepArgs args{};
    args.a = *a;
    args.lanes = 1;
    while (args.lanes * 4 < a->V) args.lanes *= 2;
    while (args.lanes > 8 && a->rows * a->heads * ceil_div(a->V, 4 * args.lanes) < 256) args.lanes /= 2;
    args.pieces = (int32_t)ceil_div(a->V, 4 * args.lanes);
    args.each = (int32_t)(a->heads / a->groups);
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (a->dtype) {
    case SCANSCAM_F32: return code(launch_attend_step<float>(args, s));
    case SCANSCAM_BF16: return code(launch_attend_step<__bf16>(args, s));
    default: return code(launch_attend_step<_Float16>(args, s));
    }
}

}  // extern "C"
