// Matrix products on the tensor cores: a persistent kernel in which one warp brings tiles of the operands
// into shared memory (TMA), one thread issues the products (tcgen05), and eight warps take finished tiles out of tensor
// memory and through an epilogue while the next tile is summed.
//
// A tile is 128 (kCtas == 1) or 256 (2: a pair of CTAs works on one) by 256, summed in 32 bits.
#pragma once
#include "math.cuh"
#include "ptx.cuh"

namespace stdml::collective::train
{
constexpr int kTileM = 128;       // rows of a CTA
constexpr int kTileN = 256;       // columns of a tile
constexpr int kStepK = 64;        // of the reduction: 128 bytes
constexpr int kChunk = 128 * 128; // bytes of 128 rows (or columns) by one step
constexpr int kEpilogueWarps = 8;
constexpr int kProductThreads = 32 * (4 + kEpilogueWarps);
constexpr int kMostSegments = 12;

// What a product reads: a sum over segments, each a product over the whole reduction.  A and B are slabs of their maps.
struct Segment {
    signed char a_slab, b_map, b_slab;
};

struct Product {
    CUtensorMap a, b[2];
    Segment segments[kMostSegments];
    int segment_count;
    int steps;                // of the reduction, per segment
    long long m, n;           // of the result (n: of each half in a gated tile)
    int m_tiles, n_tiles, z;  // z results side by side: A's slabs z_slabs apart
    int z_slabs, z_first;
    uint32_t kind;            // instruction descriptor
    unsigned int *status;
};

// Why a kernel gave up: a wait ran out.
constexpr unsigned int kWaitRanOut = 1;
constexpr unsigned long long kWaitLimitNs = 10ull * 1000 * 1000 * 1000;

__device__ __forceinline__ unsigned long long clock_ns()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// False: the block gives up (`dead` in its shared memory says so to all its warps).
static __device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile int *dead, unsigned int *status)
{
    const unsigned long long t0 = clock_ns();
    for (unsigned int spins = 0; spins < (1u << 28); ++spins) {
        if (bar_try(bar, parity)) { return true; }
        if (*dead != 0) { return false; }
        if ((spins & 63u) == 63u && clock_ns() - t0 > kWaitLimitNs) { break; }
    }
    *dead = 1;
    atomicExch(status, kWaitRanOut);
    return false;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int *dead, unsigned int *status)
{
    return bar_try(bar, parity) || wait_slow(bar, parity, dead, status);
}

struct Tile {
    long long m, n;
    int z;
};

// Tiles that run at the same time share operands: bands of kBand tile rows, column by column.
template <int kCtas>
__device__ __forceinline__ Tile tile_at(const Product &p, int i)
{
    constexpr int kBand = 16 / kCtas;
    const int per = p.m_tiles * p.n_tiles, z = i / per;
    i -= z * per;
    const int band = i / (kBand * p.n_tiles), first = band * kBand;
    const int high = min(kBand, p.m_tiles - first);
    i -= band * kBand * p.n_tiles;
    return {static_cast<long long>(first + i % high) * (kTileM * kCtas), static_cast<long long>(i / high), z + p.z_first};
}

template <int kCtas>
constexpr int stages()
{
    return kCtas == 2 ? 6 : 4;
}
template <int kCtas>
constexpr int stage_bytes()
{
    return kChunk + kChunk * 2 / kCtas;
}
template <int kCtas>
constexpr int product_smem()
{
    return stages<kCtas>() * stage_bytes<kCtas>() + 1024 /* alignment */ + 256 /* barriers */;
}

// kAcrossA, kAcrossB: the operand's rows lie along the reduction (its reduction runs across them).
// Epilogue: void tile(const Product &, m0 of the CTA, n tile, z, warp 0..7, tensor memory address).
template <int kCtas, bool kAcrossA, bool kAcrossB, bool kTwoB, typename Epilogue>
__global__ void __launch_bounds__(kProductThreads, 1) product_kernel(const __grid_constant__ Product p,
                                                                     const __grid_constant__ Epilogue epilogue)
{
    extern __shared__ unsigned char raw[];
    constexpr int kStages = stages<kCtas>(), kBytes = stage_bytes<kCtas>(), kChunksB = 2 / kCtas;
    __shared__ uint32_t tmem_at;
    __shared__ int dead_flag;
    unsigned char *ring = raw + ((1024u - (smem_at(raw) & 1023u)) & 1023u);
    uint64_t *bars = reinterpret_cast<uint64_t *>(ring + kStages * kBytes);
    const uint32_t ring_at = smem_at(ring), full = smem_at(bars), empty = full + 8 * kStages,
                   summed = empty + 8 * kStages, taken = summed + 16;
    volatile int *dead = &dead_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = kCtas == 2 ? cta_rank() : 0u;

    if (threadIdx.x == 0) {
        dead_flag = 0;
        for (int i = 0; i < kStages; ++i) {
            bar_init(full + 8 * i, 1);
            bar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(summed + 8 * i, 1);
            bar_init(taken + 8 * i, kCtas * kEpilogueWarps);
        }
        bar_init_visible();
    }
    if (warp == 2) { tmem_alloc<kCtas>(smem_at(&tmem_at), 512); }
    tmem_before_sync();
    __syncthreads();
    if constexpr (kCtas == 2) { cluster_sync(); }
    tmem_after_sync();
    const uint32_t tmem = tmem_at;

    const int tiles = p.m_tiles * p.n_tiles * p.z, workers = gridDim.x / kCtas, first = blockIdx.x / kCtas;

    if (warp == 0 && lane == 0) {
        // ---- loads
        map_prefetch(&p.a);
        map_prefetch(&p.b[0]);
        if constexpr (kTwoB) { map_prefetch(&p.b[1]); }
        int it = 0;
        bool ok = true;
        for (int t = first; ok && t < tiles; t += workers) {
            const Tile tile = tile_at<kCtas>(p, t);
            const int m0 = static_cast<int>(tile.m) + static_cast<int>(rank) * kTileM;
            for (int s = 0; ok && s < p.segment_count; ++s) {
                const Segment seg = p.segments[s];
                const int a_slab = seg.a_slab + tile.z * p.z_slabs;
                for (int k = 0; k < p.steps; ++k, ++it) {
                    const int st = it % kStages;
                    ok = it < kStages || wait_for(empty + 8 * st, (it / kStages - 1) & 1, dead, p.status);
                    if (!ok) { break; }
                    const uint32_t bar = full + 8 * st, at = ring_at + st * kBytes;
                    if (rank == 0) { bar_expect(bar, kCtas * kBytes); }
                    if constexpr (kAcrossA) {
                        for (int i = 0; i < 2; ++i) {
                            box_load<kCtas>(at + i * (kChunk / 2), &p.a, m0 + 64 * i, k * kStepK, a_slab, bar);
                        }
                    } else {
                        box_load<kCtas>(at, &p.a, k * kStepK, m0, a_slab, bar);
                    }
#pragma unroll
                    for (int c = 0; c < kChunksB; ++c) {
                        const int chunk = static_cast<int>(rank) * kChunksB + c;  // of the tile's two
                        const uint32_t to = at + kChunk * (1 + c);
                        const CUtensorMap *map = &p.b[kTwoB ? chunk : seg.b_map];
                        const int n0 = kTwoB ? static_cast<int>(tile.n) * 128 : static_cast<int>(tile.n) * kTileN + 128 * chunk;
                        if constexpr (kAcrossB) {
                            for (int i = 0; i < 2; ++i) {
                                box_load<kCtas>(to + i * (kChunk / 2), map, n0 + 64 * i, k * kStepK, seg.b_slab, bar);
                            }
                        } else {
                            box_load<kCtas>(to, map, k * kStepK, n0, seg.b_slab, bar);
                        }
                    }
                }
            }
        }
        // The copies asked for end before the block does: with the products that read them (an arrival on `empty`).
        for (int i = max(0, it - kStages); i < it; ++i) {
            if (!wait_for(empty + 8 * (i % kStages), (i / kStages) & 1, dead, p.status)) { break; }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        // ---- products
        int it = 0, round = 0;
        bool ok = true;
        for (int t = first; ok && t < tiles; t += workers, ++round) {
            const int buf = round & 1;
            ok = round < 2 || wait_for(taken + 8 * buf, (round / 2 - 1) & 1, dead, p.status);
            if (!ok) { break; }
            tmem_after_sync();
            const uint32_t d = tmem + buf * kTileN;
            const int steps = p.segment_count * p.steps;
            for (int k = 0; k < steps; ++k, ++it) {
                const int st = it % kStages;
                ok = wait_for(full + 8 * st, (it / kStages) & 1, dead, p.status);
                if (!ok) { break; }
                tmem_after_sync();
                const uint32_t at = ring_at + st * kBytes;
                const uint64_t a = operand_desc(at, kAcrossA ? kChunk / 2 : 16, 1024);
                const uint64_t b = operand_desc(at + kChunk, kAcrossB ? kChunk / 2 : 16, 1024);
#pragma unroll
                for (int j = 0; j < kStepK / 16; ++j) {
                    // 16 further: 32 bytes along the rows, or 16 rows
                    mma16<kCtas>(d, a + j * (kAcrossA ? 128 : 2), b + j * (kAcrossB ? 128 : 2), p.kind, k > 0 || j > 0);
                }
                mma_commit<kCtas>(empty + 8 * st);
            }
            if (ok) { mma_commit<kCtas>(summed + 8 * buf); }
        }
    } else if (warp >= 4) {
        // ---- epilogue
        int round = 0;
        for (int t = first; t < tiles; t += workers, ++round) {
            const int buf = round & 1;
            if (!__all_sync(0xffffffffu, wait_for(summed + 8 * buf, (round / 2) & 1, dead, p.status))) { break; }
            tmem_after_sync();
            const Tile tile = tile_at<kCtas>(p, t);
            epilogue.tile(p, tile.m + rank * kTileM, tile.n, tile.z, warp - 4, tmem + buf * kTileN);
            tmem_before_sync();
            __syncwarp();
            if (lane == 0) { bar_arrive_first(taken + 8 * buf); }
        }
    }
    __syncwarp();
    tmem_before_sync();
    __syncthreads();
    if constexpr (kCtas == 2) { cluster_sync(); }
    tmem_after_sync();
    if (warp == 2) { tmem_free<kCtas>(tmem, 512); }
}
}  // namespace stdml::collective::train
