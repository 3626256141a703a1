// Group normalisation: the calls.  See norm.cuh.
#include <algorithm>

#include "norm.cuh"

namespace stdml::collective::train
{
void norm_params_launch(const NormArgs &n, void *dweight, void *dbias, cudaStream_t s);

namespace
{
Rows rows_of(const stdmlc_rows &r) { return {r.ptr, r.image, r.row}; }

// How the work is cut.
//   Channels: chunks of whole groups, of at most 2048 channels and 256 groups (their sums lie in shared memory), and narrower ones, down to 256
//   bytes of a row, while the images' slices alone would leave SMs without work.
//   Positions: slices of 64 at least, up to eight to a cluster; where clusters would fill less than half of the GPU,
//   as many slices as it takes and two launches.
//   (64 images of 112 x 112 x 64 in bf16: 512 blocks of 1568 positions.)
void cut(NormArgs &n, int element)
{
    const int sms = sm_count();
    n.chunks = 1;
    int per_chunk = n.groups;  // groups
    const auto width = [&] { return per_chunk * n.per; };
    while (per_chunk > 1 && (width() > 2048 || per_chunk > kMostGroups || (n.images * ((n.groups + per_chunk - 1) / per_chunk) * kMostSlices < 2 * sms &&
                                                width() / 2 * element >= 256 && per_chunk % 2 == 0))) {
        per_chunk = (per_chunk + 1) / 2;
    }
    n.width = width();
    n.chunks = (n.groups + per_chunk - 1) / per_chunk;
    const long long blocks = n.images * n.chunks, most = std::max(1ll, n.positions / 64);
    long long slices = 1;
    while (slices < kMostSlices && slices * 2 <= most && blocks * slices < 4 * sms) { slices *= 2; }
    n.walks = 3;
    if (blocks * slices < sms / 2 && most > kMostSlices) {
        slices = std::min(most, (2 * sms + blocks - 1) / blocks);
        n.walks = 2;
    }
    n.slices = static_cast<int>(slices);
}

NormArgs checked(const stdmlc_norm *a, bool backward)
{
    require(a != nullptr, "group_norm: null arguments");
    require(float_type(a->dt) && float_type(a->weight_dt), "group_norm: bf16, f16 or f32 expected");
    require(a->act >= STDMLC_ACT_NONE && a->act <= STDMLC_ACT_GELU, "group_norm: unknown activation");
    require(a->images >= 0 && a->positions >= 0 && a->channels > 0, "group_norm: bad sizes");
    require(a->groups > 0 && a->channels % a->groups == 0, "group_norm: the groups must divide the channels");
    require(a->channels / a->groups <= kMostPer, "group_norm: at most 8192 channels in a group");
    require(a->eps >= 0, "group_norm: eps must not be negative");
    const bool any = a->images > 0 && a->positions > 0;
    require(!any || (a->x.ptr != nullptr && a->stats != nullptr), "group_norm: null operand");
    require(!any || (backward ? a->dy.ptr : a->y.ptr) != nullptr, "group_norm: null operand");
    NormArgs n{};
    n.x = rows_of(a->x);
    n.r = rows_of(a->residual);
    n.dy = rows_of(a->dy);
    n.y = rows_of(a->y);
    n.dx = rows_of(a->dx);
    n.dr = rows_of(a->dresidual);
    n.weight = a->weight;
    n.bias = a->bias;
    n.stats = a->stats;
    n.images = a->images;
    n.positions = a->positions;
    n.channels = a->channels;
    n.groups = a->groups;
    n.per = a->channels / a->groups;
    n.weight_dt = a->weight_dt;
    n.eps = a->eps;
    if (any) {
        n.per_position = 1.0 / static_cast<double>(n.positions);
        n.per_value = n.per_position / n.per;
        cut(n, element_size(a->dt));
        require(n.images * n.chunks * n.slices < (1ll << 31), "group_norm: too many images");
    }
    return n;
}

int vector_of(const NormArgs &n, int element, std::initializer_list<const Rows *> all)
{
    int v = 16 / element;
    const auto fits = [&] {
        if (n.channels % v != 0 || n.width % v != 0) { return false; }
        for (const Rows *r : all) {
            if (r->ptr != nullptr && (reinterpret_cast<uintptr_t>(r->ptr) % (v * element) != 0 || r->image % v != 0 || r->row % v != 0)) {
                return false;
            }
        }
        return true;
    };
    while (v > 1 && !fits()) { v /= 2; }
    return v;
}

long long sums_bytes(const NormArgs &n) { return n.walks == 2 ? 16 * n.images * n.slices * n.groups : 0; }
}  // namespace
}  // namespace stdml::collective::train

using namespace stdml::collective::train;

extern "C" long long stdmlc_norm_workspace(const stdmlc_norm *a, int backward)
{
    if (a == nullptr || a->images < 0 || a->positions < 0 || a->channels <= 0 || a->groups <= 0 || a->channels % a->groups != 0) { return -1; }
    if (a->images == 0 || a->positions == 0) { return 0; }
    NormArgs n{};
    n.images = a->images;
    n.positions = a->positions;
    n.channels = a->channels;
    n.groups = a->groups;
    n.per = a->channels / a->groups;
    return bytes_entry([&] {
        cut(n, element_size(a->dt));
        return sums_bytes(n) + (backward != 0 ? 8 * n.images * n.slices * n.channels : 0);
    });
}

extern "C" int stdmlc_norm_forward(const stdmlc_norm *a, int device, void *stream)
{
    return entry(device, [&] {
        NormArgs n = checked(a, false);
        if (n.images == 0 || n.positions == 0) { return; }
        require(n.walks == 3 || a->workspace != nullptr, "group_norm: null workspace");
        n.sums = static_cast<double *>(a->workspace);
        norm_forward_launch(n, a->dt, vector_of(n, element_size(a->dt), {&n.x, &n.r, &n.y}), a->act, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int stdmlc_norm_backward(const stdmlc_norm *a, int device, void *stream)
{
    return entry(device, [&] {
        NormArgs n = checked(a, true);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const bool params = a->dweight != nullptr || a->dbias != nullptr;
        if (n.images == 0 || n.positions == 0) {  // sums of nothing
            for (void *p : {a->dweight, a->dbias}) {
                if (p != nullptr) { cuda_ok(cudaMemsetAsync(p, 0, static_cast<size_t>(element_size(a->weight_dt)) * n.channels, s), "cudaMemsetAsync"); }
            }
            return;
        }
        require(a->workspace != nullptr, "group_norm: null workspace");
        n.sums = static_cast<double *>(a->workspace);
        if (params) { n.param_sums = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + sums_bytes(n)); }
        norm_backward_launch(n, a->dt, vector_of(n, element_size(a->dt), {&n.x, &n.r, &n.dy, &n.dx, &n.dr}), a->act, s);
        if (params) { norm_params_launch(n, a->dweight, a->dbias, s); }
    });
}
