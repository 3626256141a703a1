// Group normalisation with its activation on channels-last images: what its two directions share.
//
// With xh = (x - mean) * rstd over the positions and channels of a group, z = xh * w + b + r:
//   y = act(z);  dz = dy * act'(z);  dr = dz;  db_c = sum dz;  dw_c = sum dz * xh;
//   dx = rstd * (dz * w - m1 - xh * m2),  m1 = sum_c w_c db_c / count,  m2 = sum_c w_c dw_c / count  (of the image and group).
//
// Bytes bound it: images in and out once.  A block takes a slice of an image's positions, of all channels or of a chunk of
// whole groups; a thread has the same few channels in all its rows, so that sums and factors stay in its registers.
// Either direction walks its slice twice, first for sums and then for results.  The blocks of an image are a
// cluster that exchanges its sums through shared memory.  The second walk goes back from where the first ended and finds in the L2 what is
// still there; of large batches that is a part, since all their images are in work at once (48 images of 112 x 112 x 64 in bf16: 112 MB
// read forward and 265 backward, of 77 and 154).  (Keeping them in shared memory instead took a third longer at its best: too few
// blocks then share an SM, and nothing is under way while one sums.)  Where there are too few images for that to fill the GPU, the two walks are two launches
// of slices of all images, with the sums in memory between them.
#pragma once
#include <algorithm>

#include "dispatch.cuh"
#include "host.hpp"
#include "ptx.cuh"

namespace stdml::collective::train
{
constexpr int kNormThreads = 256;  // four blocks to an SM: while some sum, others load (with two of 512, a tenth slower)
constexpr int kMostSlices = 8;  // of an image, in a cluster
constexpr int kMostGroups = 256;  // of a chunk
constexpr int kMostPer = 8192;  // channels of a group

struct Rows {
    const void *ptr;
    long long image, row;
};

struct NormArgs {
    Rows x, r, dy, y, dx, dr;  // (results too; null: not wanted)
    const void *weight, *bias;
    double *stats;      // [images][groups][2]: mean, 1 / sqrt(var + eps)
    double *sums;       // [images][slices][groups][2], between two launches
    float *param_sums;  // [images][slices][2][channels]; null: not wanted
    long long images, positions;
    int channels, groups, per, weight_dt;
    int chunks, width;  // of an image's channels: `width` channels in all but the last
    int slices;         // of an image's positions
    int walks;          // 1: first walk alone, 2: second, 3: both, the slices being a cluster
    double eps;
    double per_position, per_value;  // 1 / positions, 1 / (positions * channels of a group)
};

__device__ __forceinline__ float weight_of(const NormArgs &a, int c)
{
    return a.weight != nullptr ? load_any(a.weight, c, a.weight_dt) : 1.f;
}
__device__ __forceinline__ float bias_of(const NormArgs &a, int c)
{
    return a.bias != nullptr ? load_any(a.bias, c, a.weight_dt) : 0.f;
}

// kCh channels side by side.
template <typename T, int kCh>
struct Vec {
    static constexpr int kBytes = kCh * static_cast<int>(sizeof(T));
    alignas(kBytes) T v[kCh];

    __device__ __forceinline__ float at(int i) const { return to_f32(v[i]); }
    __device__ __forceinline__ void set(const float (&f)[kCh])
    {
        if constexpr (sizeof(T) == 2 && kCh % 2 == 0) {
#pragma unroll
            for (int i = 0; i < kCh; i += 2) { reinterpret_cast<uint32_t *>(v)[i / 2] = pack2(f[i], f[i + 1], T{}); }
        } else {
#pragma unroll
            for (int i = 0; i < kCh; ++i) { v[i] = from_f32<T>(f[i]); }
        }
    }
};

// n * i / of, in 32 bits where that does.
__device__ __forceinline__ long long portion(long long n, int i, int of)
{
    return n < (1ll << 27) ? static_cast<unsigned int>(n) * static_cast<unsigned int>(i) / static_cast<unsigned int>(of) : n * i / of;
}

// What a block works on.
struct Part {
    long long n;      // image
    int slice;
    int c0, width;    // channels
    long long from, to;  // positions

    __device__ __forceinline__ explicit Part(const NormArgs &a)
    {
        const unsigned int i = blockIdx.x / static_cast<unsigned int>(a.slices);
        slice = blockIdx.x - i * a.slices;
        n = i / static_cast<unsigned int>(a.chunks);
        c0 = (i - static_cast<int>(n) * a.chunks) * a.width;
        width = min(a.width, a.channels - c0);
        from = a.slices <= 32 ? portion(a.positions, slice, a.slices) : a.positions * slice / a.slices;
        to = a.slices <= 32 ? portion(a.positions, slice + 1, a.slices) : a.positions * (slice + 1) / a.slices;
    }
};

// A block's threads as columns of kCh channels by rows; more columns than threads are passed over one after the other.
template <int kCh>
struct Grid {
    int columns, across, down, passes;

    __device__ __forceinline__ explicit Grid(int width)
    {
        columns = (width + kCh - 1) / kCh;
        across = min(columns, static_cast<int>(blockDim.x));
        down = blockDim.x / across;
        passes = (columns + across - 1) / across;
    }
    __device__ __forceinline__ int column(int pass) const { return pass * across + threadIdx.x % across; }
    __device__ __forceinline__ int row() const { return threadIdx.x / across; }
};

// Two sums for each channel of a block, over its rows of threads: into `total`.  A thread adds up few rows in 32 bits, and has the sums of
// those in 64 here, in `lines`: value i of a thread's channels at line_of(i).  All threads take part in adding them up: some rows
// each, then the shares.  `shares`: blockDim.x pairs.
__device__ __forceinline__ int line_of(int i) { return i * kNormThreads + threadIdx.x; }

template <int kCh>
__device__ __forceinline__ void column_sums(const Grid<kCh> &g, int pass, int width, const double2 *lines, double2 *shares, double2 *total)
{
    __syncthreads();
    const int span = g.across * kCh;  // (the first channels of all columns, the second ones, ...)
    const auto sum_of = [&](int at, int first, int step) {
        const double2 *line = lines + at / g.across * kNormThreads + at % g.across;
        double a = 0, b = 0;
        for (int r = first; r < g.down; r += step) {
            a += line[r * g.across].x;
            b += line[r * g.across].y;
        }
        return make_double2(a, b);
    };
    const int helpers = span < kNormThreads ? kNormThreads / span : 1;
    if (helpers > 1) {
        const int part = threadIdx.x / span;
        if (part < helpers) { shares[threadIdx.x] = sum_of(threadIdx.x % span, part, helpers); }
        __syncthreads();
    }
    for (int at = threadIdx.x; at < span; at += kNormThreads) {
        const int c = pass * span + at % g.across * kCh + at / g.across;
        if (c >= width) { continue; }
        double2 sum;
        if (helpers > 1) {
            sum = make_double2(0, 0);
            for (int k = 0; k < helpers; ++k) {
                sum.x += shares[k * span + at].x;
                sum.y += shares[k * span + at].y;
            }
        } else {
            sum = sum_of(at, 0, 1);
        }
        total[c] = sum;
    }
    __syncthreads();
}

// f(group, first channel's lane, lanes): a thread takes a group of few channels, a warp one of many.  f's values are
// added up by `gather`.
constexpr int kFewPer = 16;
template <typename F>
__device__ __forceinline__ void each_group(int groups, int per, F f)
{
    if (per <= kFewPer) {
        for (int k = threadIdx.x; k < groups; k += kNormThreads) { f(k, 0, 1, [](double v) { return v; }); }
    } else {
        for (int k = threadIdx.x >> 5; k < groups; k += kNormThreads / 32) {
            f(k, static_cast<int>(threadIdx.x & 31), 32, [](double v) { return warp_sum(v); });
        }
    }
}

// A thread's rows of a matrix, one after the other.
template <typename V>
struct Walker {
    const char *at;
    long long step;  // bytes to the next row

    template <typename T>
    __device__ __forceinline__ Walker(const T *image, long long row, long long first, int column, int channels, int down)
        : at(reinterpret_cast<const char *>(image + first * row + column * channels)), step(static_cast<long long>(sizeof(T)) * row * down)
    {
    }
    __device__ __forceinline__ V load(int k) const { return *reinterpret_cast<const V *>(at + k * step); }
    __device__ __forceinline__ void store(int k, const V &v) const { *reinterpret_cast<V *>(const_cast<char *>(at) + k * step) = v; }
    __device__ __forceinline__ void next(int k) { at += k * step; }
    // From the last of `rows` rows back to the first.
    __device__ __forceinline__ void turn(int rows)
    {
        at += (rows - 1) * step;
        step = -step;
    }
};

// Two doubles to the same place in a block of the cluster.  (Sent, not fetched: eight reads one after the other took 10 us.)
__device__ __forceinline__ void send(const double2 *place, int block, const double2 &v)
{
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_at(place)), "r"(block));
    asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(at), "d"(v.x), "d"(v.y) : "memory");
}

// A slice's sums of a group go to all blocks of the image: [slice][group] in shared memory, or in memory for the second launch.
__device__ __forceinline__ void publish(const NormArgs &a, const Part &p, double2 *all, int groups, int g0, int k, const double2 &v)
{
    if (a.walks == 1) {
        reinterpret_cast<double2 *>(a.sums)[(p.n * a.slices + p.slice) * a.groups + g0 + k] = v;
    } else if (a.slices == 1) {
        all[k] = v;
    } else {
        for (int i = 0; i < a.slices; ++i) { send(all + p.slice * groups + k, i, v); }
    }
}
__device__ __forceinline__ double2 published(const NormArgs &a, const Part &p, const double2 *all, int groups, int g0, int k, int slice)
{
    return a.walks == 2 ? reinterpret_cast<const double2 *>(a.sums)[(p.n * a.slices + slice) * a.groups + g0 + k] : all[slice * groups + k];
}

// `vector`: how many channels side by side all addresses allow to be read at once.
void norm_forward_launch(const NormArgs &n, int dt, int vector, int act, cudaStream_t s);
void norm_backward_launch(const NormArgs &n, int dt, int vector, int act, cudaStream_t s);

// One launch of clusters, or one for each walk (the second only where there are `results` beyond sums).
template <typename Kernel>
void norm_walks(Kernel kernel, NormArgs n, int channels_per_thread, bool results, cudaStream_t s)
{
    const long long blocks = n.images * n.chunks * n.slices;
    // lines of sums, first values, shares of the lines, totals of channels, sums of groups (of all slices)
    const size_t sums = sizeof(double2) * kNormThreads * channels_per_thread + sizeof(float) * ((n.width + 3) / 4 * 4) +
                        sizeof(double2) * (kNormThreads + n.width + (n.walks == 3 ? n.slices : 1) * (n.width / n.per));
    // (the most that any sizes take, always: another thread may be about to launch the same kernel with more)
    cuda_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 << 10), "shared memory");
    for (int walk : {1, 2}) {
        if (walk == 2 && (n.walks == 3 || !results)) { return; }
        NormArgs args = n;
        args.walks = n.walks == 3 ? 3 : walk;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned int>(blocks));
        cfg.blockDim = dim3(kNormThreads);
        cfg.dynamicSmemBytes = sums;
        cfg.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {static_cast<unsigned int>(n.walks == 3 ? n.slices : 1), 1, 1};
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cuda_ok(cudaLaunchKernelEx(&cfg, kernel, args), "group_norm: launch");
    }
}
}  // namespace stdml::collective::train
