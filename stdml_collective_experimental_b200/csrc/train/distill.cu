// The distillation loss against a teacher's top logits, forward and backward.
//
// A row with logits z, teacher's logits v_j at classes k_j, temperature t, label y:
//   p_j = softmax(v / t)_j;  M = max z;  s = sum exp(z - M);  S = sum exp((z - M) / t)
//   loss = a * (log s - (z_y - M)) + b * t^2 * sum_j p_j * (log p_j - (z_kj - M) / t + log S)
//   dz_i = a * (exp(z_i - M) / s - [i = y]) + b * t * (exp((z_i - M) / t) / S * [any p] - sum_{kj = i} p_j)
// with b = 1 - a, or a = 0 and b = 1 without labels.
//
// Bytes bound it: the logits once in, the gradient once out.  A block (for few rows a cluster of blocks) takes a row,
// walks it once with running maximum and sums, and, where the caller wants gradients, a second time to write
// them: the row comes from the L2 then, since the rows in work at a time are fewer than fit there.  The classes that
// the teacher or the label names are corrected afterwards.
#include <algorithm>

#include "dispatch.cuh"
#include "host.hpp"
#include "ptx.cuh"

namespace stdml::collective::train
{
namespace
{
constexpr int kUnroll = 4;       // vectors of 16 bytes that a thread has on their way
constexpr int kCountBlocks = 256;
constexpr int kMostCluster = 8;

struct Args {
    stdmlc_distill d;
    float *row_loss;
    int *counts;           // rows that count, of each block of the counting kernel; then the ticket
    int count_blocks;      // 0: every row weighs one
    void *grad;            // null: none wanted in the forward pass
    int cluster;
};

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
    for (int base = 0; base < d.top_count; base += 32) {
        const int j = base + (threadIdx.x & 31);
        bool in = false;
        if (j < d.top_count) {
            const long long k = index_at(d, r, j);
            in = k >= 0 && k < d.classes && load_any(d.top, r * d.top_row + j, d.top_dt) * (1.f / d.temperature) != -INFINITY;
        }
        if (__any_sync(0xffffffffu, in)) { return true; }
    }
    return false;
}

// How many rows count: one number for each block, which the rows' blocks add up.
__global__ void __launch_bounds__(1024) count_kernel(stdmlc_distill d, int *counts)
{
    __shared__ int slots[32];
    int live = 0;
    if (d.labels != nullptr) {
        for (long long r = blockIdx.x * 1024ll + threadIdx.x; r < d.rows; r += gridDim.x * 1024ll) {
            live += label_at(d, r) >= 0 ? 1 : 0;
        }
    } else {
        const int lane = threadIdx.x & 31;
        for (long long r = blockIdx.x * 32ll + (threadIdx.x >> 5); r < d.rows; r += gridDim.x * 32ll) {
            const bool counts_ = has_entry(d, r);
            live += counts_ && lane == 0 ? 1 : 0;
        }
    }
    live = block_sum(live, slots);
    if (threadIdx.x == 0) {
        counts[blockIdx.x] = live;
        if (blockIdx.x == 0) { counts[kCountBlocks] = 0; }  // the ticket
    }
}

// A row, or a block's share of it: single elements up to a 16-byte boundary, vectors, single elements.
template <typename T>
struct Share {
    static constexpr int kPer = 16 / sizeof(T);
    const T *z;
    long long head, vectors, from, to, tail;  // vectors [from, to) are the block's; elements from `tail` on the last block's

    __device__ __forceinline__ Share(const T *row, long long classes, int part, int parts) : z(row)
    {
        head = min(classes, static_cast<long long>((16u - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / static_cast<int>(sizeof(T)));
        vectors = (classes - head) / kPer;
        from = vectors * part / parts;
        to = vectors * (part + 1) / parts;
        tail = head + vectors * kPer;
    }
    // f(element index, values, how many), for all of the block's; `several`: kUnroll vectors at once
    template <typename F>
    __device__ __forceinline__ void each(long long classes, bool first, bool last, F f) const
    {
        if (first && threadIdx.x < head) { f.one(threadIdx.x, to_f32(z[threadIdx.x])); }
        const uint4 *v = reinterpret_cast<const uint4 *>(z + head);
        long long i = from + threadIdx.x;
        for (; i + (kUnroll - 1) * blockDim.x < to; i += kUnroll * blockDim.x) {
            uint4 raw[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) { raw[k] = v[i + k * blockDim.x]; }
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) { f.vector(head + (i + k * blockDim.x) * kPer, raw[k]); }
        }
        for (; i < to; i += blockDim.x) { f.vector(head + i * kPer, v[i]); }
        if (last && tail + threadIdx.x < classes) { f.one(tail + threadIdx.x, to_f32(z[tail + threadIdx.x])); }
    }
};

constexpr float kLowest = -3.402823466e38f;

// Maximum and sums of what a thread has seen.
struct Running {
    float most = kLowest, hard = 0, soft = 0;

    __device__ __forceinline__ void raise(float to, float c)
    {
        if (to > most) {
            hard *= fast_exp2((most - to) * kLog2E);
            soft *= fast_exp2((most - to) * c);
            most = to;
        }
    }
};

// (z - M) / t in powers of two: a difference and a product, or for 16-bit logits one multiply-add, where neither product can
// overflow (a mask's lowest value, as the only one in the row, would).
template <typename T>
struct Reach {
    float most, c, shift;
    bool fused;
    __device__ __forceinline__ Reach(float most_, float c_) : most(most_), c(c_), shift(-most_ * c_), fused(sizeof(T) == 2 && fabsf(shift) < 1e30f) {}
    __device__ __forceinline__ float operator()(float v) const { return fused ? fmaf(v, c, shift) : (v - most) * c; }
};

// exp((z - M) / t) and exp(z - M).  kPower: t where it is 1, 2 or 4, so that the one is a power of the other (0: another
// t); the exponential unit takes 8 cycles for what the others do in one (bf16, 2048 x 30522: 87 us at t = 2, 99 at t = 3; 4096 x 128256:
// 545 and 658).  In 32 bits the gradient of a class that nobody names is 1.0e-7 to 3.9e-7 off (root mean square, relative), with powers or
// without; CUDA's expf makes that 0.9e-7 to 2.5e-7, as elementary operations have it, and 2048 x 30522 takes 198 us instead of 144.
template <bool kHard, bool kSoft, int kPower>
__device__ __forceinline__ void exponentials(float x, float t, float &hard, float &soft)
{
    if constexpr (kSoft) { soft = fast_exp2(x); }
    if constexpr (kHard && kSoft && kPower != 0) {
        hard = kPower == 1 ? soft : kPower == 2 ? soft * soft : (soft * soft) * (soft * soft);
    } else if constexpr (kHard) {
        hard = fast_exp2(x * t);
    }
}

template <typename T, bool kHard, bool kSoft, int kPower>
struct Walk {
    Running &r;
    float c, t;  // c: log2(e) / t

    __device__ __forceinline__ void one(long long, float v)
    {
        r.raise(v, c);
        add(v, Reach<T>(r.most, c));
    }
    __device__ __forceinline__ void vector(long long, const uint4 &raw)
    {
        float v[16 / sizeof(T)];
        unpack16<T>(raw, v);
        float most = v[0];
#pragma unroll
        for (int i = 1; i < static_cast<int>(16 / sizeof(T)); ++i) { most = fmaxf(most, v[i]); }
        r.raise(most, c);
        const Reach<T> x(r.most, c);
        if (x.fused) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) { add(v[i], x); }
        } else {
#pragma unroll
            for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) { add(v[i], x); }
        }
    }
    __device__ __forceinline__ void add(float v, const Reach<T> &x)
    {
        float h = 0, q = 0;
        exponentials<kHard, kSoft, kPower>(x(v), t, h, q);
        if constexpr (kHard) { r.hard += h; }
        if constexpr (kSoft) { r.soft += q; }
    }
};

template <typename T, bool kHard, bool kSoft, int kPower>
struct Write {
    T *dz;
    float most, hard, soft, c, t;  // factors of the two exponentials; c: log2(e) / t
    bool same;                     // the gradient's rows lie on the same boundaries as the logits'

    __device__ __forceinline__ float grad(float v, const Reach<T> &x) const
    {
        float h = 0, q = 0;
        exponentials<kHard, kSoft, kPower>(x(v), t, h, q);
        return kHard && kSoft ? hard * h + soft * q : kHard ? hard * h : soft * q;
    }
    __device__ __forceinline__ void one(long long i, float v) { dz[i] = from_f32<T>(grad(v, Reach<T>(most, c))); }
    __device__ __forceinline__ void vector(long long i, const uint4 &raw)
    {
        float v[16 / sizeof(T)];
        unpack16<T>(raw, v);
        const Reach<T> x(most, c);
        if (x.fused) {
#pragma unroll
            for (int k = 0; k < static_cast<int>(16 / sizeof(T)); ++k) { v[k] = grad(v[k], x); }
        } else {
#pragma unroll
            for (int k = 0; k < static_cast<int>(16 / sizeof(T)); ++k) { v[k] = grad(v[k], x); }
        }
        if (same) {
            __stcs(reinterpret_cast<uint4 *>(dz + i), pack16<T>(v));
        } else {
#pragma unroll
            for (int k = 0; k < static_cast<int>(16 / sizeof(T)); ++k) { dz[i + k] = from_f32<T>(v[k]); }
        }
    }
};

// The teacher's side of a row: the largest of its v / t (-inf without an entry, NaN with one), and the sum of exp(v / t - most).  (Their
// logarithm in one number would cost a probability what 32 bits lose of v / t.)
struct Teacher {
    float most, sum;

    __device__ __forceinline__ bool some() const { return most != -INFINITY; }
    __device__ __forceinline__ float prob(float v) const { return some() ? expf(v - most) / sum : 0.f; }
};

// That of row r, with v / t and the classes (-1: no entry) in shared memory.
__device__ __forceinline__ Teacher teacher_row(const stdmlc_distill &d, long long r, float *prob, int *cls, float *slots)
{
    const float inv_t = 1.f / d.temperature;
    float top = -INFINITY;
    for (int j = threadIdx.x; j < d.top_count; j += blockDim.x) {
        const long long k = index_at(d, r, j);
        const bool in = k >= 0 && k < d.classes;
        const float v = in ? load_any(d.top, r * d.top_row + j, d.top_dt) * inv_t : -INFINITY;
        cls[j] = in ? static_cast<int>(k) : -1;
        prob[j] = v;
        top = v > top || v != v ? v : top;  // (NaN stays)
    }
    if (d.top_count <= 32) {
        // one warp has them all
        __syncthreads();
        if (threadIdx.x < 32) {
            const bool nan = __any_sync(0xffffffffu, top != top);
            const float m = warp_max(top);
            const float sum = warp_sum(threadIdx.x < d.top_count && m != -INFINITY ? expf(prob[threadIdx.x] - m) : 0.f);
            if (threadIdx.x == 0) {
                slots[32] = nan ? NAN : m;
                slots[33] = sum;
            }
        }
        __syncthreads();
        return {slots[32], slots[33]};
    }
    const bool nan = __syncthreads_or(top != top ? 1 : 0) != 0;
    const float m = block_max(top, slots);
    float sum = 0;
    for (int j = threadIdx.x; j < d.top_count; j += blockDim.x) { sum += m != -INFINITY ? expf(prob[j] - m) : 0.f; }
    sum = block_sum(sum, slots);
    return {nan ? NAN : m, sum};
}

// Gradients at the classes that teacher or label name, over what the walk has written (by all threads of a block).
template <typename T, typename Writer>
__device__ __forceinline__ void correct(const stdmlc_distill &d, const Writer &w, const T *z, long long y, float hard, float soft,
                                        const float *prob, const int *cls)
{
    const Reach<T> x(w.most, w.c);
    bool y_named = false;
    for (int j = threadIdx.x; j < d.top_count; j += blockDim.x) {
        const int k = cls[j];
        const float v = k >= 0 ? to_f32(z[k]) : 0.f;
        bool again = false;  // a class that is named twice is written once, for both
        float p = 0;
#pragma unroll 8
        for (int i = 0; i < d.top_count; ++i) {
            const bool same = cls[i] == k;
            again = again | (same & (i < j));
            p += same ? prob[i] : 0.f;
        }
        y_named = y_named | (k == y);
        if (k >= 0 && !again) { w.dz[k] = from_f32<T>(w.grad(v, x) - soft * p - (k == y ? hard : 0.f)); }
    }
    if (y < 0) { return; }  // (the same for all of them)
    y_named = __syncthreads_or(y_named ? 1 : 0) != 0;
    if (threadIdx.x == 0 && !y_named) { w.dz[y] = from_f32<T>(w.grad(to_f32(z[y]), x) - hard); }
}

constexpr int kStats = 5;  // of a row: maximum, the two sums, the teacher's maximum, the row's weight

// A row's gradient from its statistics.  kBlocks: threads of the cluster share it.
template <typename T, bool kHard, bool kSoft, int kPower>
__device__ __forceinline__ void write_row(const stdmlc_distill &d, long long r, void *grad, float up, float most, float hard_sum,
                                          float soft_sum, bool some, const float *prob, const int *cls, int part, int parts)
{
    const T *z = static_cast<const T *>(d.logits) + r * d.logits_row;
    T *dz = static_cast<T *>(grad) + r * d.classes;
    const bool labels = d.labels != nullptr;
    const float hard = labels ? up * d.alpha : 0.f, soft = some ? (labels ? up * (1.f - d.alpha) : up) * d.temperature : 0.f;
    const bool same = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15u) == 0;
    const Write<T, kHard, kSoft, kPower> w{dz, most, hard / hard_sum, soft != 0.f ? soft / soft_sum : 0.f, kLog2E / d.temperature, d.temperature, same};
    Share<T>(z, d.classes, part, parts).each(d.classes, part == 0, part == parts - 1, w);
    if (parts > 1) {
        cluster_sync();
    } else {
        __syncthreads();
    }
    const long long y = labels ? label_at(d, r) : -1;
    if (part == 0) { correct(d, w, z, y, kHard ? hard : 0.f, kSoft ? soft : 0.f, prob, cls); }
}

template <typename T>
__device__ __forceinline__ void zero_row(T *dz, long long classes, int part, int parts)
{
    const long long from = classes * part / parts, to = classes * (part + 1) / parts;
    for (long long i = from + threadIdx.x; i < to; i += blockDim.x) { dz[i] = from_f32<T>(0.f); }
}

// kHard, kSoft: whether either softmax of the student is needed.  (Two blocks of 512 threads or four of 256 to an SM.)
template <typename T, bool kHard, bool kSoft, int kPower>
__global__ void __launch_bounds__(1024) rows_kernel(Args a)
{
    extern __shared__ float held[];  // the teacher's probabilities, then their classes
    __shared__ float slots[34];
    __shared__ float shares[3 * kMostCluster];
    __shared__ int counted;
    const stdmlc_distill &d = a.d;
    const int parts = a.cluster, part = parts > 1 ? static_cast<int>(cta_rank()) : 0;
    if (parts > 1) { cluster_begin(); }
    const long long r = blockIdx.x / parts;
    const T *z = static_cast<const T *>(d.logits) + r * d.logits_row;
    float *prob = held;
    int *cls = reinterpret_cast<int *>(held + d.top_count);
    int live = 0;
    if (threadIdx.x < a.count_blocks) { live = a.counts[threadIdx.x]; }
    for (int i = threadIdx.x + blockDim.x; i < a.count_blocks; i += blockDim.x) { live += a.counts[i]; }
    const Teacher teacher = teacher_row(d, r, prob, cls, slots);
    const long long y = d.labels != nullptr ? label_at(d, r) : -1;
    const bool counts = d.labels != nullptr ? y >= 0 : teacher.some();
    if (parts > 1) { cluster_runs(); }
    if (!counts) {  // (the same in all blocks of the row)
        if (a.grad != nullptr) { zero_row(static_cast<T *>(a.grad) + r * d.classes, d.classes, part, parts); }
        if (part == 0 && threadIdx.x == 0) {
            d.row_stats[kStats * r + 4] = 0.f;
            a.row_loss[r] = 0.f;
        }
    } else {
        float weight = 1.f;
        if (a.count_blocks > 0) {
            live = block_sum(live, reinterpret_cast<int *>(slots));
            weight = 1.f / static_cast<float>(live);
        }
        const float c = kLog2E / d.temperature;
        Running run;
        Share<T>(z, d.classes, part, parts).each(d.classes, part == 0, part == parts - 1, Walk<T, kHard, kSoft, kPower>{run, c, d.temperature});
        float most = block_max(run.most, slots);
        const bool bad = __syncthreads_or(run.hard != run.hard || run.soft != run.soft ? 1 : 0) != 0;  // (fmaxf drops NaN)
        run.raise(most, c);
        float hard = kHard ? block_sum(run.hard, slots) : 1.f, soft = kSoft ? block_sum(run.soft, slots) : 1.f;
        if (bad) { hard = soft = NAN; }
        if (parts > 1) {
            // every block gets every block's
            if (threadIdx.x < parts) {
                const uint32_t at = smem_at(shares + 3 * part);
                uint32_t there;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(static_cast<uint32_t>(threadIdx.x)));
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(most) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there + 4), "f"(hard) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there + 8), "f"(soft) : "memory");
            }
            cluster_sync();
            float all = kLowest;
            for (int k = 0; k < parts; ++k) { all = fmaxf(all, shares[3 * k]); }
            hard = soft = 0;
            for (int k = 0; k < parts; ++k) {
                hard += shares[3 * k + 1] * (kHard ? fast_exp2((shares[3 * k] - all) * kLog2E) : 1.f / parts);
                soft += shares[3 * k + 2] * (kSoft ? fast_exp2((shares[3 * k] - all) * c) : 1.f / parts);
            }
            most = all;
        }
        // the teacher's side
        const float inv_t = 1.f / d.temperature, log_soft = kSoft ? logf(soft) : 0.f;
        const float log_sum = teacher.some() ? logf(teacher.sum) : 0.f;
        float kl = 0;
        for (int j = threadIdx.x; j < d.top_count; j += blockDim.x) {
            const float p = cls[j] >= 0 ? teacher.prob(prob[j]) : 0.f;
            // (an entry whose weight has vanished has no term, wherever the student is: 0 log 0; NaN stays)
            if (kSoft && p != 0.f) {
                kl += p * (((prob[j] - teacher.most) - log_sum) - ((to_f32(z[cls[j]]) - most) * inv_t - log_soft));
            }
            prob[j] = p;
        }
        if (part == 0) {
            kl = block_sum(kl, slots);
            if (threadIdx.x == 0) {
                float loss = d.temperature * d.temperature * kl;
                if (d.labels != nullptr) {
                    loss = (kSoft ? (1.f - d.alpha) * loss : 0.f) + (kHard ? d.alpha * (logf(hard) - (to_f32(z[y]) - most)) : 0.f);
                }
                float *st = d.row_stats + kStats * r;
                st[0] = most;
                st[1] = hard;
                st[2] = soft;
                st[3] = teacher.most;
                st[4] = weight;
                a.row_loss[r] = weight * loss;
            }
        }
        __syncthreads();
        if (a.grad != nullptr) { write_row<T, kHard, kSoft, kPower>(d, r, a.grad, weight, most, hard, soft, teacher.some(), prob, cls, part, parts); }
    }
    // Whoever comes last adds up the rows, in their order.
    if (d.reduction == 0 || part != 0) { return; }
    if (threadIdx.x == 0) {
        __threadfence();
        counted = atomicAdd(a.counts + kCountBlocks, 1);
    }
    __syncthreads();
    if (counted != static_cast<int>(d.rows) - 1) { return; }
    __threadfence();
    __shared__ double sums[32];
    double sum = 0;
    for (long long i = threadIdx.x; i < d.rows; i += blockDim.x) { sum += __ldcg(a.row_loss + i); }
    sum = block_sum(sum, sums);
    if (threadIdx.x == 0) { *d.loss = static_cast<float>(sum); }
}

// The gradient of a loss of gradient d.dloss.  Where the forward pass has written that of a loss of gradient one (d.written), there is
// nothing to do for one, and for another the whole of it is computed again: multiplied, it would be rounded twice.
template <typename T, bool kHard, bool kSoft, int kPower>
__global__ void __launch_bounds__(1024) grad_kernel(Args a)
{
    extern __shared__ float held[];
    __shared__ float slots[34];
    const stdmlc_distill &d = a.d;
    const int parts = a.cluster, part = parts > 1 ? static_cast<int>(cta_rank()) : 0;
    if (d.written != 0 && *d.dloss == 1.f) { return; }
    for (long long r = blockIdx.x / parts; r < d.rows; r += gridDim.x / parts) {
        const float *st = d.row_stats + kStats * r;
        const float weight = st[4];
        if (weight == 0.f) {
            zero_row(static_cast<T *>(a.grad) + r * d.classes, d.classes, part, parts);
            continue;
        }
        const float up = weight * d.dloss[d.reduction == 0 ? r * d.dloss_row : 0];
        float *prob = held;
        int *cls = reinterpret_cast<int *>(held + d.top_count);
        if (part == 0) {
            const Teacher teacher = teacher_row(d, r, prob, cls, slots);
            for (int j = threadIdx.x; j < d.top_count; j += blockDim.x) { prob[j] = cls[j] >= 0 ? teacher.prob(prob[j]) : 0.f; }
            __syncthreads();
        }
        write_row<T, kHard, kSoft, kPower>(d, r, a.grad, up, st[0], st[1], st[2], st[3] != -INFINITY, prob, cls, part, parts);
        __syncthreads();  // (prob and cls are the next row's)
    }
}

void check(const stdmlc_distill *d)
{
    require(d != nullptr, "distill_loss: null arguments");
    require(float_type(d->dt) && float_type(d->top_dt), "distill_loss: bf16, f16 or f32 expected");
    require(d->index_bytes == 4 || d->index_bytes == 8, "distill_loss: 32 or 64-bit indices expected");
    require(d->rows >= 0 && d->rows < (1ll << 28) && d->classes > 0 && d->classes < (1ll << 31),
            "distill_loss: at most 2^28 rows of 2^31 classes");
    require(d->top_count >= 0 && d->top_count <= 4096, "distill_loss: at most 4096 teacher entries in a row");
    require(d->temperature > 0.f, "distill_loss: the temperature must be positive");
    require(d->reduction >= 0 && d->reduction <= 2, "distill_loss: unknown reduction");
    require(d->rows == 0 || (d->logits != nullptr && d->row_stats != nullptr), "distill_loss: null operand");
    require(d->rows == 0 || d->top_count == 0 || (d->top != nullptr && d->index != nullptr),
            "distill_loss: null operand");
}

// How many blocks share a row, and their threads.
//   Rows that are fewer than the SMs are spread over clusters, down to 4 KB for each block.
//   An SM has 1024 threads of these kernels.  The smaller the blocks, the more rows are in work at a time, some waiting
//   while others load; but rows in work have to stay in the L2 (126 MB) until they are written: 256 threads up to
//   64 KB of a row (38 MB in work), 512 up to 256 KB (76 MB), 1024 beyond.
//   With 1024 throughout, 2048 rows of 61 KB took 245 us, and 4096 of 256 KB 691.
void launch_shape(const stdmlc_distill &d, int &cluster, int &threads)
{
    const long long bytes = d.classes * element_size(d.dt);
    cluster = 1;
    while (cluster < kMostCluster && d.rows * cluster * 2 <= 2 * sm_count() && bytes / (cluster * 2) >= 4096) { cluster *= 2; }
    const long long share = bytes / cluster;
    threads = share <= 4096 ? 128 : share <= (64 << 10) ? 256 : share <= (256 << 10) ? 512 : 1024;
}

template <typename F>
void by_need(const stdmlc_distill &d, F f)
{
    const bool hard = d.labels != nullptr && d.alpha != 0.f, soft = d.labels == nullptr || d.alpha != 1.f;
    if (hard && soft) {
        if (d.temperature == 1.f) {
            f(Int<1>{}, Int<1>{}, Int<1>{});
        } else if (d.temperature == 2.f) {
            f(Int<1>{}, Int<1>{}, Int<2>{});
        } else if (d.temperature == 4.f) {
            f(Int<1>{}, Int<1>{}, Int<4>{});
        } else {
            f(Int<1>{}, Int<1>{}, Int<0>{});
        }
    } else if (hard) {
        f(Int<1>{}, Int<0>{}, Int<0>{});
    } else {
        f(Int<0>{}, Int<1>{}, Int<0>{});
    }
}

template <typename Kernel>
void launch_rows(Kernel kernel, const Args &a, long long rows, int threads, cudaStream_t s)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned int>(rows * a.cluster));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = 8 * static_cast<size_t>(a.d.top_count);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {static_cast<unsigned int>(a.cluster), 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cuda_ok(cudaLaunchKernelEx(&cfg, kernel, a), "distill_loss: launch");
}

constexpr long long up16(long long n) { return (n + 15) / 16 * 16; }
}  // namespace
}  // namespace stdml::collective::train

using namespace stdml::collective::train;

extern "C" long long stdmlc_distill_workspace(const stdmlc_distill *d)
{
    if (d == nullptr || d->rows < 0) { return -1; }
    return d->reduction == 0 ? 0 : up16(4 * d->rows) + 4 * (kCountBlocks + 1);
}

extern "C" int stdmlc_distill_forward(const stdmlc_distill *d, int device, void *stream)
{
    return entry(device, [&] {
        check(d);
        require(d->loss != nullptr || (d->rows == 0 && d->reduction == 0), "distill_loss: null operand");
        require(d->rows == 0 || d->reduction == 0 || d->workspace != nullptr, "distill_loss: null workspace");
        require(d->dlogits == nullptr || (d->reduction != 0 && d->dt != kF16), "distill_loss: no gradient in the forward pass here");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (d->rows == 0) {
            if (d->reduction != 0) { cuda_ok(cudaMemsetAsync(d->loss, 0, 4, s), "cudaMemsetAsync"); }
            return;
        }
        Args a{*d, d->loss, nullptr, 0, d->dlogits, 1};
        int threads;
        launch_shape(*d, a.cluster, threads);
        if (d->reduction != 0) {
            a.row_loss = static_cast<float *>(d->workspace);
            a.counts = reinterpret_cast<int *>(static_cast<char *>(d->workspace) + up16(4 * d->rows));
            const long long each = d->labels != nullptr ? 1024 : 32, blocks = (d->rows + each - 1) / each;
            const int used = static_cast<int>(blocks < kCountBlocks ? blocks : kCountBlocks);
            count_kernel<<<static_cast<unsigned int>(used), 1024, 0, s>>>(*d, a.counts);
            a.count_blocks = d->reduction == 2 ? used : 0;
        }
        by_dtype(d->dt, [&](auto t) {
            by_need(*d, [&](auto hard, auto soft, auto power) {
                launch_rows(rows_kernel<decltype(t), decltype(hard)::value != 0, decltype(soft)::value != 0, decltype(power)::value>, a, d->rows, threads, s);
            });
        });
    });
}

extern "C" int stdmlc_distill_backward(const stdmlc_distill *d, int device, void *stream)
{
    return entry(device, [&] {
        check(d);
        if (d->rows == 0) { return; }
        require(d->dloss != nullptr && d->dlogits != nullptr, "distill_loss: null operand");
        Args a{*d, nullptr, nullptr, 0, d->dlogits, 1};
        int threads;
        require(d->written == 0 || d->reduction != 0, "distill_loss: no gradient in the forward pass here");
        launch_shape(*d, a.cluster, threads);
        // Blocks that find nothing to do cost a launch of thousands some microseconds, so each takes several rows where there may be
        // nothing: as many blocks as fit on the GPU twice (4096 rows of 256 KB: 5.5 us with four times as many).
        long long rows = d->rows;
        if (d->written != 0 && a.cluster == 1) {
            const long long most = 2ll * sm_count() * (1024 / threads), each = (rows + most - 1) / most;
            rows = (rows + each - 1) / each;
        }
        by_dtype(d->dt, [&](auto t) {
            by_need(*d, [&](auto hard, auto soft, auto power) {
                launch_rows(grad_kernel<decltype(t), decltype(hard)::value != 0, decltype(soft)::value != 0, decltype(power)::value>, a, rows, threads,
                            static_cast<cudaStream_t>(stream));
            });
        });
    });
}

extern "C" long long stdmlc_stream_capturing(void *stream)
{
    cudaStreamCaptureStatus how = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &how, &id) != cudaSuccess) { (void)cudaGetLastError(); }
    return how != cudaStreamCaptureStatusNone ? static_cast<long long>(id) : 0;
}
