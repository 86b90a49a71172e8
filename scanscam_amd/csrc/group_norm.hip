// C ABI of the group norm (declared in include/scanscam_attention.h): argument checks, launch shapes, launches.
#include "group_norm_kernels.hpp"

namespace {

using namespace scanscam;

constexpr int64_t kMostGroup = SCANSCAM_MOST_GROUP, kMostParts = 1024;

int check_group_norm(const scanscam_group_norm *a, bool back)
{
    if (a == nullptr || a->rows < 0 || a->rows >= kMostTokens || a->channels < 0 || a->channels > kMostChannels || a->groups < 1 || a->channels % a->groups != 0 ||
        a->channels / a->groups > kMostGroup || a->x_stride < 0 || a->z_stride < 0 || (a->activation != SCANSCAM_ACT_NONE && a->activation != SCANSCAM_ACT_SILU))
        return SCANSCAM_EINVAL;
    const size_t size = (size_t)activation_size(a->dtype);
    if (size == 0) return SCANSCAM_EDTYPE;
    if (a->channels == 0) return SCANSCAM_OK;
    SCANSCAM_CHECK(check_param(a->weight, false));
    SCANSCAM_CHECK(check_param(a->bias, false));
    if (back && ((a->gweight != nullptr) != (a->weight.p != nullptr) || (a->gbias != nullptr) != (a->bias.p != nullptr))) return SCANSCAM_EINVAL;
    if (back && (misaligned(a->gweight, 4) || misaligned(a->gbias, 4))) return SCANSCAM_EALIGN;
    if (a->rows == 0) return SCANSCAM_OK;
    if (a->x == nullptr || misaligned(a->x, size) || misaligned(a->z, size)) return a->x == nullptr ? SCANSCAM_EINVAL : SCANSCAM_EALIGN;
    if (!back) return a->y == nullptr ? SCANSCAM_EINVAL : misaligned(a->y, size) ? SCANSCAM_EALIGN : SCANSCAM_OK;
    if (a->gy == nullptr || a->gx == nullptr || (a->gz != nullptr) != (a->z != nullptr)) return SCANSCAM_EINVAL;
    return misaligned(a->gy, size) || misaligned(a->gx, size) || misaligned(a->gz, size) ? SCANSCAM_EALIGN : SCANSCAM_OK;
}

GroupNormPlan plan_of(const scanscam_group_norm &a)
{
    const int64_t vectors = ceil_div(a.channels / a.groups, a.dtype == SCANSCAM_F32 ? 4 : 8);
    GroupNormPlan p{1, 1, 1};
    while (p.lanes < 64 && p.lanes < vectors) p.lanes *= 2;
    if (vectors > 64) p.nv = 2;
    if (vectors > 128) {
        p.nv = a.dtype == SCANSCAM_F32 ? group_most<float>() : group_most<__bf16>();
        for (p.waves = 2; p.waves * p.nv * 64 < vectors;) p.waves *= 2;
    }
    return p;
}

// Teams of a group: as many as fill the card, and no more, so that parameters are read by few; backwards fewer, whose sums have to be joined: 1024 of a group at most. With one
// group of few channels these are few workgroups (bf16: 64 for 128 channels, 16 for 32), and the pass is far from memory's rate: [524288, 128] in one group takes 445 us backwards
// for 403 MB, [2097152, 32] 1700; [65536, 1024] in eight groups 117, in one 148.
int64_t parts_of(const scanscam_group_norm &a, const GroupNormPlan &p, bool back)
{
    const int64_t lanes = p.waves > 1 ? 64 * p.waves : p.lanes, most = (back ? int64_t(4096) : int64_t(16384)) * 64 / lanes, parts = ceil_div(most, a.groups);
    const int64_t limit = back && parts > kMostParts ? kMostParts : parts;
    return limit < a.rows ? limit : a.rows > 0 ? a.rows : 1;
}

int64_t columns_of(const scanscam_group_norm &a) { return ((a.weight.p != nullptr ? 1 : 0) + (a.bias.p != nullptr ? 1 : 0)) * a.channels; }

hipError_t run(bool back, const scanscam_group_norm &a, float *part, hipStream_t stream)
{
    const GroupNormPlan plan = plan_of(a);
    const GroupNormArgs args{a, parts_of(a, plan, back), (int32_t)(a.channels / a.groups), plan.waves, part};
    switch (a.dtype) {
    case SCANSCAM_F32: return launch_group_norm<float>(back, plan, stream, args);
    case SCANSCAM_BF16: return launch_group_norm<__bf16>(back, plan, stream, args);
    default: return launch_group_norm<_Float16>(back, plan, stream, args);
    }
}

}  // namespace

extern "C" {

int scanscam_group_norm_fwd(const scanscam_group_norm *a, void *stream)
{
    SCANSCAM_CHECK(check_group_norm(a, false));
    if (a->rows == 0 || a->channels == 0) return SCANSCAM_OK;
    return run(false, *a, nullptr, static_cast<hipStream_t>(stream)) == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
}

size_t scanscam_group_norm_workspace_bytes(const scanscam_group_norm *a)
{
    if (a == nullptr || a->rows <= 0 || a->channels <= 0 || a->channels > kMostChannels || a->groups < 1 || a->channels % a->groups != 0 || a->channels / a->groups > kMostGroup || activation_size(a->dtype) == 0) return 0;
    return (size_t)(parts_of(*a, plan_of(*a), true) * columns_of(*a)) * sizeof(float);
}

int scanscam_group_norm_bwd(const scanscam_group_norm *a, void *stream)
{
    SCANSCAM_CHECK(check_group_norm(a, true));
    if (a->channels == 0) return SCANSCAM_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    ColumnSum sum{nullptr, 0, columns_of(*a), {a->gweight, a->gbias}, {a->gweight != nullptr ? a->channels : 0, a->gbias != nullptr ? a->channels : 0}};
    if (a->rows > 0) {
        const size_t bytes = scanscam_group_norm_workspace_bytes(a);
        if (bytes > 0 && (a->workspace == nullptr || a->workspace_bytes < bytes)) return SCANSCAM_EWORKSPACE;
        if (misaligned(a->workspace, 16)) return SCANSCAM_EALIGN;
        sum.in = static_cast<float *>(a->workspace);
        sum.parts = parts_of(*a, plan_of(*a), true);
        if (run(true, *a, sum.in, s) != hipSuccess) return SCANSCAM_ELAUNCH;
    }
    if (sum.pitch == 0) return SCANSCAM_OK;
    return column_sum(sum, s) == hipSuccess ? SCANSCAM_OK : SCANSCAM_ELAUNCH;
}

}  // extern "C"
