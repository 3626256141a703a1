// Group normalisation with its activation on channels-last images, forward and backward.
//
// With xh = (x - mean) * rstd over the positions and channels of a group, z = xh * w + b + r:
//   y = act(z);  dz = dy * act'(z);  dr = dz;  dw = sum dz * xh;  db = sum dz;
//   dx = rstd * (dz * w - mean(dz * w) - xh * mean(dz * w * xh)).
#include "dispatch.cuh"
#include "host.hpp"

namespace stdml::collective::train
{
namespace
{
constexpr int kThreads = 256;

struct Rows {
    const void *ptr;
    long long image, row;
};

struct NormArgs {
    Rows x, r, dy;
    void *y, *dx, *dr;
    Rows ys, dxs, drs;
    const void *weight, *bias;
    void *dweight, *dbias;
    double *stats, *sums;
    long long images, positions;
    int channels, groups, per, weight_dt;
    double eps;
};

__device__ __forceinline__ float weight_of(const NormArgs &a, int c)
{
    return a.weight != nullptr ? load_any(a.weight, c, a.weight_dt) : 1.f;
}
__device__ __forceinline__ float bias_of(const NormArgs &a, int c)
{
    return a.bias != nullptr ? load_any(a.bias, c, a.weight_dt) : 0.f;
}

// The derivative of relu jumps at zero: a value that 32 bits leave in doubt is placed in 64.
template <int kAct>
__device__ __forceinline__ float pre_activation(float x, double mean, double rstd, float w, float b, float r)
{
    const float k = static_cast<float>(rstd) * w, m = static_cast<float>(mean);
    const float z = (x - m) * k + b + r;
    if constexpr (kAct == STDMLC_ACT_RELU) {
        if (fabsf(z) <= 1e-5f * ((fabsf(x) + fabsf(m)) * fabsf(k) + fabsf(b) + fabsf(r))) {
            return static_cast<float>((x - mean) * rstd * w + b + r);
        }
    }
    return z;
}

template <typename T>
__device__ __forceinline__ float at(const Rows &m, long long n, long long s, int c)
{
    return to_f32(static_cast<const T *>(m.ptr)[n * m.image + s * m.row + c]);
}
template <typename T>
__device__ __forceinline__ void put(void *p, const Rows &m, long long n, long long s, int c, float v)
{
    static_cast<T *>(p)[n * m.image + s * m.row + c] = from_f32<T>(v);
}

template <typename T>
__global__ void stats_kernel(NormArgs a)
{
    __shared__ double slots[32];
    const long long n = blockIdx.x / a.groups, many = a.positions * a.per;
    const int g = blockIdx.x % a.groups;
    double sum = 0;
    for (long long e = threadIdx.x; e < many; e += blockDim.x) {
        sum += at<T>(a.x, n, e / a.per, g * a.per + static_cast<int>(e % a.per));
    }
    const double mean = block_sum(sum, slots) / many;
    double sq = 0;
    for (long long e = threadIdx.x; e < many; e += blockDim.x) {
        const double d = at<T>(a.x, n, e / a.per, g * a.per + static_cast<int>(e % a.per)) - mean;
        sq += d * d;
    }
    const double var = block_sum(sq, slots) / many;
    if (threadIdx.x == 0) {
        a.stats[2 * blockIdx.x] = mean;
        a.stats[2 * blockIdx.x + 1] = 1.0 / sqrt(var + a.eps);
    }
}

template <typename T, int kAct>
__global__ void apply_kernel(NormArgs a)
{
    const long long many = a.images * a.positions * a.channels;
    const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
    for (long long e = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; e < many; e += step) {
        const int c = static_cast<int>(e % a.channels);
        const long long s = e / a.channels % a.positions, n = e / a.channels / a.positions;
        const double *st = a.stats + 2 * (n * a.groups + c / a.per);
        const float r = a.r.ptr != nullptr ? at<T>(a.r, n, s, c) : 0.f;
        const float z = pre_activation<kAct>(at<T>(a.x, n, s, c), st[0], st[1], weight_of(a, c), bias_of(a, c), r);
        put<T>(a.y, a.ys, n, s, c, act<T, kAct>(z));
    }
}

template <typename T, int kAct>
__device__ __forceinline__ float grad_z(const NormArgs &a, long long n, long long s, int c, float &xh)
{
    const double *st = a.stats + 2 * (n * a.groups + c / a.per);
    const float r = a.r.ptr != nullptr ? at<T>(a.r, n, s, c) : 0.f, x = at<T>(a.x, n, s, c);
    const float z = pre_activation<kAct>(x, st[0], st[1], weight_of(a, c), bias_of(a, c), r);
    xh = (x - static_cast<float>(st[0])) * static_cast<float>(st[1]);
    return at<T>(a.dy, n, s, c) * act_grad<T, kAct>(z);
}

template <typename T, int kAct>
__global__ void group_sums_kernel(NormArgs a)
{
    __shared__ double slots[32];
    const long long n = blockIdx.x / a.groups, many = a.positions * a.per;
    const int g = blockIdx.x % a.groups;
    double s1 = 0, s2 = 0;
    for (long long e = threadIdx.x; e < many; e += blockDim.x) {
        const int c = g * a.per + static_cast<int>(e % a.per);
        float xh;
        const float d = grad_z<T, kAct>(a, n, e / a.per, c, xh) * weight_of(a, c);
        s1 += d;
        s2 += d * xh;
    }
    s1 = block_sum(s1, slots);
    s2 = block_sum(s2, slots);
    if (threadIdx.x == 0) {
        a.sums[2 * blockIdx.x] = s1 / many;
        a.sums[2 * blockIdx.x + 1] = s2 / many;
    }
}

template <typename T, int kAct>
__global__ void parameter_sums_kernel(NormArgs a)
{
    __shared__ double slots[32];
    const int c = blockIdx.x;
    const long long many = a.images * a.positions;
    double s1 = 0, s2 = 0;
    for (long long e = threadIdx.x; e < many; e += blockDim.x) {
        float xh;
        const float d = grad_z<T, kAct>(a, e / a.positions, e % a.positions, c, xh);
        s1 += d;
        s2 += d * xh;
    }
    s1 = block_sum(s1, slots);
    s2 = block_sum(s2, slots);
    if (threadIdx.x == 0) {
        if (a.dbias != nullptr) { store_any(a.dbias, c, a.weight_dt, static_cast<float>(s1)); }
        if (a.dweight != nullptr) { store_any(a.dweight, c, a.weight_dt, static_cast<float>(s2)); }
    }
}

template <typename T, int kAct>
__global__ void grad_kernel(NormArgs a)
{
    const long long many = a.images * a.positions * a.channels;
    const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
    for (long long e = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; e < many; e += step) {
        const int c = static_cast<int>(e % a.channels);
        const long long s = e / a.channels % a.positions, n = e / a.channels / a.positions;
        const long long g = n * a.groups + c / a.per;
        float xh;
        const float d = grad_z<T, kAct>(a, n, s, c, xh);
        if (a.dr != nullptr) { put<T>(a.dr, a.drs, n, s, c, d); }
        if (a.dx != nullptr) {
            const float m1 = static_cast<float>(a.sums[2 * g]), m2 = static_cast<float>(a.sums[2 * g + 1]);
            put<T>(a.dx, a.dxs, n, s, c,
                   static_cast<float>(a.stats[2 * g + 1]) * (d * weight_of(a, c) - m1 - xh * m2));
        }
    }
}

Rows rows_of(const stdmlc_rows &r) { return {r.ptr, r.image, r.row}; }

NormArgs checked(const stdmlc_norm *a, bool backward)
{
    require(a != nullptr, "group_norm: null arguments");
    require(float_type(a->dt) && float_type(a->weight_dt), "group_norm: bf16, f16 or f32 expected");
    require(a->act >= STDMLC_ACT_NONE && a->act <= STDMLC_ACT_GELU, "group_norm: unknown activation");
    require(a->images >= 0 && a->positions >= 0 && a->channels > 0, "group_norm: bad sizes");
    require(a->groups > 0 && a->channels % a->groups == 0,
            "group_norm: the groups must divide the channels");
    require(a->images * a->groups < (1ll << 31), "group_norm: too many groups");
    require(a->eps >= 0, "group_norm: eps must not be negative");
    const bool any = a->images > 0 && a->positions > 0;
    require(!any || (a->x.ptr != nullptr && a->stats != nullptr), "group_norm: null operand");
    require(!any || (backward ? a->dy.ptr : a->y.ptr) != nullptr, "group_norm: null operand");
    require(!any || !backward || a->workspace != nullptr, "group_norm: null workspace");
    NormArgs n{};
    n.x = rows_of(a->x);
    n.r = rows_of(a->residual);
    n.dy = rows_of(a->dy);
    n.ys = rows_of(a->y);
    n.dxs = rows_of(a->dx);
    n.drs = rows_of(a->dresidual);
    n.y = a->y.ptr;
    n.dx = a->dx.ptr;
    n.dr = a->dresidual.ptr;
    n.weight = a->weight;
    n.bias = a->bias;
    n.dweight = a->dweight;
    n.dbias = a->dbias;
    n.stats = a->stats;
    n.sums = static_cast<double *>(a->workspace);
    n.images = a->images;
    n.positions = a->positions;
    n.channels = a->channels;
    n.groups = a->groups;
    n.per = a->channels / a->groups;
    n.weight_dt = a->weight_dt;
    n.eps = a->eps;
    return n;
}

unsigned int spread(long long many)
{
    const long long blocks = (many + kThreads - 1) / kThreads;
    return static_cast<unsigned int>(blocks < 4096 ? blocks : 4096);
}
}  // namespace
}  // namespace stdml::collective::train

using namespace stdml::collective::train;

extern "C" long long stdmlc_norm_workspace(const stdmlc_norm *a, int backward)
{
    if (a == nullptr || a->images < 0 || a->groups <= 0) { return -1; }
    return backward ? 16 * a->images * a->groups : 0;
}

extern "C" int stdmlc_norm_forward(const stdmlc_norm *a, int device, void *stream)
{
    return entry(device, [&] {
        const NormArgs n = checked(a, false);
        if (n.images == 0 || n.positions == 0) { return; }
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        by_dtype(a->dt, [&](auto t) {
            using T = decltype(t);
            stats_kernel<T><<<static_cast<unsigned int>(n.images * n.groups), kThreads, 0, s>>>(n);
            by_act(a->act, [&](auto k) {
                apply_kernel<T, decltype(k)::value>
                    <<<spread(n.images * n.positions * n.channels), kThreads, 0, s>>>(n);
            });
        });
    });
}

extern "C" int stdmlc_norm_backward(const stdmlc_norm *a, int device, void *stream)
{
    return entry(device, [&] {
        const NormArgs n = checked(a, true);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        by_dtype(a->dt, [&](auto t) {
            by_act(a->act, [&](auto k) {
                using T = decltype(t);
                constexpr int kAct = decltype(k)::value;
                if (n.dweight != nullptr || n.dbias != nullptr) {
                    parameter_sums_kernel<T, kAct><<<n.channels, kThreads, 0, s>>>(n);
                }
                if (n.images == 0 || n.positions == 0) { return; }
                group_sums_kernel<T, kAct>
                    <<<static_cast<unsigned int>(n.images * n.groups), kThreads, 0, s>>>(n);
                grad_kernel<T, kAct><<<spread(n.images * n.positions * n.channels), kThreads, 0, s>>>(n);
            });
        });
    });
}
