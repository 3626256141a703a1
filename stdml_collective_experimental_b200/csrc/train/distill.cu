// The distillation loss against a teacher's top logits, forward and backward.
//
// A row with logits z, teacher's logits v_j at classes k_j, temperature t, label y:
//   p_j = softmax(v / t)_j;  l = log sum exp z;  m = log sum exp(z / t)
//   loss = a * (l - z_y) + b * t^2 * sum_j p_j * (log p_j - z_kj / t + m)
//   dz_i = a * (exp(z_i - l) - [i = y]) + b * t * (exp(z_i / t - m) * [any p] - sum_{kj = i} p_j)
// with b = 1 - a, or a = 0 and b = 1 without labels.
#include "dispatch.cuh"
#include "host.hpp"

namespace stdml::collective::train
{
namespace
{
constexpr int kThreads = 256;

__device__ __forceinline__ long long index_at(const stdmlc_distill &d, long long r, int j)
{
    const long long i = r * d.index_row + j;
    return d.index_bytes == 8 ? static_cast<const long long *>(d.index)[i] : static_cast<const int *>(d.index)[i];
}

__device__ __forceinline__ long long label_at(const stdmlc_distill &d, long long r)
{
    const long long y = static_cast<const long long *>(d.labels)[r];
    return y != d.ignore && y >= 0 && y < d.classes ? y : -1;
}

// Whether the teacher has an entry in row r (a warp asks).
__device__ __forceinline__ bool has_entry(const stdmlc_distill &d, long long r)
{
    bool any = false;
    for (int j = threadIdx.x & 31; j < d.top_count; j += 32) {
        const long long k = index_at(d, r, j);
        any = any || (k >= 0 && k < d.classes && load_any(d.top, r * d.top_row + j, d.top_dt) != -INFINITY);
    }
    return __any_sync(0xffffffffu, any);
}

// The weight of every row: 1 or 1 / (rows that count), 0 where it does not count.
__global__ void weights_kernel(stdmlc_distill d)
{
    __shared__ long long slots[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    long long live = 0;
    for (long long r = warp; r < d.rows; r += warps) {
        const bool counts = d.labels != nullptr ? label_at(d, r) >= 0 : has_entry(d, r);
        if (lane == 0) { d.row_stats[4 * r + 3] = counts ? 1.f : 0.f; }
        live += counts && lane == 0 ? 1 : 0;
    }
    live = block_sum(live, slots);
    if (d.reduction != 2) { return; }
    const float each = 1.f / static_cast<float>(live > 0 ? live : 1);
    for (long long r = threadIdx.x; r < d.rows; r += blockDim.x) { d.row_stats[4 * r + 3] *= each; }
}

template <typename T>
__global__ void rows_kernel(stdmlc_distill d, float *row_loss)
{
    __shared__ float slots[32];
    const long long r = blockIdx.x;
    const T *z = static_cast<const T *>(d.logits) + r * d.logits_row;
    const float inv_t = 1.f / d.temperature;
    float *st = d.row_stats + 4 * r;
    float most = -INFINITY;
    for (long long i = threadIdx.x; i < d.classes; i += blockDim.x) { most = fmaxf(most, to_f32(z[i])); }
    most = block_max(most, slots);
    float s1 = 0, st_ = 0;
    for (long long i = threadIdx.x; i < d.classes; i += blockDim.x) {
        const float v = to_f32(z[i]);
        s1 += expf(v - most);
        st_ += expf((v - most) * inv_t);
    }
    const float lse = most + logf(block_sum(s1, slots)), lset = most * inv_t + logf(block_sum(st_, slots));
    float top = -INFINITY;
    for (int j = threadIdx.x; j < d.top_count; j += blockDim.x) {
        const long long k = index_at(d, r, j);
        if (k >= 0 && k < d.classes) { top = fmaxf(top, load_any(d.top, r * d.top_row + j, d.top_dt) * inv_t); }
    }
    top = block_max(top, slots);
    const bool some = top != -INFINITY;
    float sp = 0;
    for (int j = threadIdx.x; j < d.top_count; j += blockDim.x) {
        const long long k = index_at(d, r, j);
        if (some && k >= 0 && k < d.classes) { sp += expf(load_any(d.top, r * d.top_row + j, d.top_dt) * inv_t - top); }
    }
    const float lp = some ? top + logf(block_sum(sp, slots)) : -INFINITY;
    float kl = 0;
    for (int j = threadIdx.x; j < d.top_count; j += blockDim.x) {
        const long long k = index_at(d, r, j);
        if (!some || k < 0 || k >= d.classes) { continue; }
        const float logp = load_any(d.top, r * d.top_row + j, d.top_dt) * inv_t - lp;
        if (logp != -INFINITY) { kl += expf(logp) * (logp - (to_f32(z[k]) * inv_t - lset)); }
    }
    kl = block_sum(kl, slots);
    if (threadIdx.x != 0) { return; }
    const float weight = st[3];
    float loss = d.temperature * d.temperature * kl;
    if (d.labels != nullptr) {
        const long long y = label_at(d, r);
        loss = (1.f - d.alpha) * loss + (y >= 0 ? d.alpha * (lse - to_f32(z[y])) : 0.f);
    }
    st[0] = lse;
    st[1] = lset;
    st[2] = lp;
    row_loss[r] = weight != 0.f ? weight * loss : 0.f;
}

__global__ void total_kernel(const float *row_loss, long long rows, float *loss)
{
    __shared__ double slots[32];
    double sum = 0;
    for (long long r = threadIdx.x; r < rows; r += blockDim.x) { sum += row_loss[r]; }
    sum = block_sum(sum, slots);
    if (threadIdx.x == 0) { *loss = static_cast<float>(sum); }
}

template <typename T>
__global__ void grad_kernel(stdmlc_distill d)
{
    extern __shared__ float held[];  // the teacher's probabilities, then their classes
    const long long r = blockIdx.x;
    const T *z = static_cast<const T *>(d.logits) + r * d.logits_row;
    T *dz = static_cast<T *>(d.dlogits) + r * d.classes;
    const float *st = d.row_stats + 4 * r;
    const float inv_t = 1.f / d.temperature, weight = st[3];
    if (weight == 0.f) {
        for (long long i = threadIdx.x; i < d.classes; i += blockDim.x) { dz[i] = from_f32<T>(0.f); }
        return;
    }
    const float up = weight * d.dloss[d.reduction == 0 ? r * d.dloss_row : 0];
    const float lse = st[0], lset = st[1], lp = st[2];
    const float hard = d.labels != nullptr ? up * d.alpha : 0.f;
    const float soft = (d.labels != nullptr ? up * (1.f - d.alpha) : up) * d.temperature;
    const bool some = lp != -INFINITY;
    const long long y = d.labels != nullptr ? label_at(d, r) : -1;
    float *prob = held;
    int *cls = reinterpret_cast<int *>(held + d.top_count);
    for (int j = threadIdx.x; j < d.top_count; j += blockDim.x) {
        const long long k = index_at(d, r, j);
        const bool in = some && k >= 0 && k < d.classes;
        cls[j] = in ? static_cast<int>(k) : -1;
        prob[j] = in ? expf(load_any(d.top, r * d.top_row + j, d.top_dt) * inv_t - lp) : 0.f;
    }
    __syncthreads();
    for (long long i = threadIdx.x; i < d.classes; i += blockDim.x) {
        const float v = to_f32(z[i]);
        float p = 0;
        for (int j = 0; j < d.top_count; ++j) { p += cls[j] == static_cast<int>(i) ? prob[j] : 0.f; }
        float g = some ? soft * (expf(v * inv_t - lset) - p) : 0.f;
        if (hard != 0.f) { g += hard * (expf(v - lse) - (i == y ? 1.f : 0.f)); }
        dz[i] = from_f32<T>(g);
    }
}

void check(const stdmlc_distill *d)
{
    require(d != nullptr, "distill_loss: null arguments");
    require(float_type(d->dt) && float_type(d->top_dt), "distill_loss: bf16, f16 or f32 expected");
    require(d->index_bytes == 4 || d->index_bytes == 8, "distill_loss: 32 or 64-bit indices expected");
    require(d->rows >= 0 && d->rows < (1ll << 31) && d->classes > 0 && d->classes < (1ll << 31),
            "distill_loss: bad sizes");
    require(d->top_count >= 0 && d->top_count <= 4096, "distill_loss: at most 4096 teacher entries in a row");
    require(d->temperature > 0.f, "distill_loss: the temperature must be positive");
    require(d->reduction >= 0 && d->reduction <= 2, "distill_loss: unknown reduction");
    require(d->rows == 0 || (d->logits != nullptr && d->row_stats != nullptr), "distill_loss: null operand");
    require(d->rows == 0 || d->top_count == 0 || (d->top != nullptr && d->index != nullptr),
            "distill_loss: null operand");
}
}  // namespace
}  // namespace stdml::collective::train

using namespace stdml::collective::train;

extern "C" long long stdmlc_distill_workspace(const stdmlc_distill *d)
{
    if (d == nullptr || d->rows < 0) { return -1; }
    return d->reduction == 0 ? 0 : 4 * d->rows;
}

extern "C" int stdmlc_distill_forward(const stdmlc_distill *d, int device, void *stream)
{
    return entry(device, [&] {
        check(d);
        require(d->loss != nullptr || (d->rows == 0 && d->reduction == 0), "distill_loss: null operand");
        require(d->rows == 0 || d->reduction == 0 || d->workspace != nullptr, "distill_loss: null workspace");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        float *row_loss = d->reduction == 0 ? d->loss : static_cast<float *>(d->workspace);
        if (d->rows > 0) {
            weights_kernel<<<1, 1024, 0, s>>>(*d);
            by_dtype(d->dt, [&](auto t) {
                rows_kernel<decltype(t)><<<static_cast<unsigned int>(d->rows), kThreads, 0, s>>>(*d, row_loss);
            });
        }
        if (d->reduction != 0) { total_kernel<<<1, 1024, 0, s>>>(row_loss, d->rows, d->loss); }
    });
}

extern "C" int stdmlc_distill_backward(const stdmlc_distill *d, int device, void *stream)
{
    return entry(device, [&] {
        check(d);
        if (d->rows == 0) { return; }
        require(d->dloss != nullptr && d->dlogits != nullptr, "distill_loss: null operand");
        by_dtype(d->dt, [&](auto t) {
            grad_kernel<decltype(t)><<<static_cast<unsigned int>(d->rows), kThreads, 8 * d->top_count,
                                       static_cast<cudaStream_t>(stream)>>>(*d);
        });
    });
}
