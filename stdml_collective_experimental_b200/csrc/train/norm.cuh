// Group normalisation with its activation on channels-last images: what its two directions share.
//
// With xh = (x - mean) * rstd over the positions and channels of a group, z = xh * w + b + r:
//   y = act(z);  dz = dy * act'(z);  dr = dz;  db_c = sum dz;  dw_c = sum dz * xh;
//   dx = rstd * (dz * w - m1 - xh * m2),  m1 = sum_c w_c db_c / count,  m2 = sum_c w_c dw_c / count  (of the image and group).
//
// Bytes bound it: images in and out once.  A block takes a slice of an image's positions, of all channels or of a chunk of
// whole groups; a thread has the same few channels in all its rows, so that sums and factors stay in its registers.
// Either direction walks its slice twice, first for sums and then for results.  The blocks of an image are a
// cluster that exchanges its sums through shared memory, and few enough images are in work at a time that the second walk
// reads from the L2.  Where there are too few images for that to fill the GPU, the two walks are two launches
// of slices of all images, with the sums in memory between them.
#pragma once
#include "dispatch.cuh"
#include "host.hpp"
#include "ptx.cuh"

namespace stdml::collective::train
{
constexpr int kNormThreads = 512;
constexpr int kMostSlices = 8;  // of an image, in a cluster
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

// What a block works on.
struct Part {
    long long n;      // image
    int slice;
    int c0, width;    // channels
    long long from, to;  // positions

    __device__ __forceinline__ explicit Part(const NormArgs &a)
    {
        const int i = blockIdx.x / a.slices;
        slice = blockIdx.x - i * a.slices;
        n = i / a.chunks;
        c0 = (i - static_cast<int>(n) * a.chunks) * a.width;
        width = min(a.width, a.channels - c0);
        from = a.positions * slice / a.slices;
        to = a.positions * (slice + 1) / a.slices;
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

// The sums of two values for each channel of a block, over its rows of threads: into `total`, in 64 bits.
// `lines`: blockDim.x * kCh pairs.
template <int kCh>
__device__ __forceinline__ void column_sums(const Grid<kCh> &g, int pass, int width, const float (&s1)[kCh], const float (&s2)[kCh],
                                            float2 *lines, double2 *total)
{
    __syncthreads();
    const int span = g.across * kCh;
    if (g.row() < g.down) {
#pragma unroll
        for (int i = 0; i < kCh; ++i) { lines[g.row() * span + (threadIdx.x % g.across) * kCh + i] = make_float2(s1[i], s2[i]); }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < span; c += blockDim.x) {
        if (pass * span + c >= width) { break; }
        double a = 0, b = 0;
        for (int r = 0; r < g.down; ++r) {
            const float2 v = lines[r * span + c];
            a += v.x;
            b += v.y;
        }
        total[pass * span + c] = make_double2(a, b);
    }
}

// Two doubles of a group at the same place in another block of the cluster.
__device__ __forceinline__ double2 of_block(const double2 *mine, int block)
{
    uint32_t at;
    double2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_at(mine)), "r"(block));
    asm volatile("ld.shared::cluster.v2.f64 {%0, %1}, [%2];" : "=d"(v.x), "=d"(v.y) : "r"(at) : "memory");
    return v;
}

// `vector`: how many channels side by side all addresses allow to be read at once.
void norm_forward_launch(const NormArgs &n, int dt, int vector, int act, cudaStream_t s);
void norm_backward_launch(const NormArgs &n, int dt, int vector, int act, cudaStream_t s);

// One launch of clusters, or one for each walk.
template <typename Kernel>
void norm_walks(Kernel kernel, NormArgs n, int channels_per_thread, cudaStream_t s)
{
    const long long blocks = n.images * n.chunks * n.slices;
    // lines of sums, totals of channels, sums of groups
    const size_t smem = sizeof(float2) * kNormThreads * channels_per_thread + sizeof(double2) * (n.width + n.width / n.per);
    cuda_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)), "shared memory");
    for (int walk : {1, 2}) {
        if (n.walks == 3 && walk == 2) { return; }
        NormArgs args = n;
        args.walks = n.walks == 3 ? 3 : walk;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned int>(blocks));
        cfg.blockDim = dim3(kNormThreads);
        cfg.dynamicSmemBytes = smem;
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
