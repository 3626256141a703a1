// Matrix products on the tensor cores: a persistent kernel in which one warp brings tiles of the operands
// into shared memory (TMA), one thread issues the products (tcgen05), and sixteen warps take finished tiles out of tensor
// memory and through an epilogue while the next tile is summed.
//
// A tile is 256 by kN (256 or 128); a pair of CTAs works on it (each loads its own 128 rows of A and half the columns of
// B), and it is summed in 32 bits.  What a launch computes is cut into units: a tile, or one of
// `split` parts of its reduction, where whole tiles would not keep all SMs busy.  Whoever comes last to a tile that was
// split sums its parts, in their order, so that results do not depend on who that is.
#pragma once
#include "math.cuh"
#include "ptx.cuh"

namespace stdml::collective::train
{
constexpr int kCtas = 2;
constexpr int kTileM = 128;        // rows of a CTA
constexpr int kStepK = 64;         // of the reduction: 128 bytes
constexpr int kChunkA = kTileM * 128;  // bytes of A's 128 rows by one step
constexpr int kEpilogueWarps = 16;     // (with 8 the epilogue of a gated tile of 12 steps took three times its products)
constexpr int kSlices = kEpilogueWarps / 4;
constexpr int kProductThreads = 32 * (4 + kEpilogueWarps);
constexpr int kStagingBytes = 4096;  // of an epilogue warp: 32 rows of 128 bytes

// 32-bit operands come in pieces, of which the pairs that reach 2^-24 of the largest are multiplied, smallest first.
constexpr int kPieces = 3, kPairs = 6;
__device__ constexpr int kPairA[kPairs] = {0, 2, 1, 0, 1, 0}, kPairB[kPairs] = {2, 0, 1, 1, 0, 0};

// What depends on the width of a tile, and on the operands (kWide: in pieces, of which a stage has all).
template <int kN, bool kWide>
struct Shape {
    static constexpr int kChunkB = kN / kCtas * 128, kOf = kWide ? kPieces : 1;
    static constexpr int kStageBytes = kOf * (kChunkA + kChunkB);
    static constexpr int kStages = kWide ? 2 : kN == 256 ? 5 : 6;
    static constexpr int kSmem = kStages * kStageBytes + kEpilogueWarps * kStagingBytes + 1024 /* alignment */ + 256 /* barriers */;
    static constexpr int kValues = kN / kSlices;  // of a tile that an epilogue thread takes
    static constexpr int kBlocks = kValues / 16;
    static constexpr long long kPart = static_cast<long long>(kCtas) * kEpilogueWarps * 32 * kValues;  // values of a part
};

// A result, or several (z) of one shape, as sums of products over a reduction.
struct Product {
    CUtensorMap a, b[2];
    int across_a, across_b;   // the operand's rows lie along the reduction (it runs across them)
    int two_b;                // half of a tile's columns by b[0], the same columns by b[1] in the other half
    int steps;                // of the reduction
    int halves;               // reductions one after the other: A's slabs half_slabs apart, the second with b[1]
    int half_slabs, z_slabs;  // A's slabs from one half, from one result to the next
    int m, n;                 // of the result (n: of either half in a tile with two B)
    int m_tiles, n_tiles, z, z_first;
    int split, first_unit, first_tile, first_part;
    uint32_t kind;            // instruction descriptor
};

struct Work {
    Product product[2];
    int products, units;
    int chunk;          // steps that are summed in tensor memory before 32-bit registers take over (0: all)
    float *parts;       // kPart values for each unit of a split product, then (kWide) for each cluster, from own_part on
    int own_part;
    unsigned int *tickets;  // zero: [tile][CTA of the pair][epilogue warp]
    unsigned int *status;
    unsigned long long wait_ns;  // how long a wait may last; 0: the kernel gives up with its first loads under way
};

// Why a kernel gave up: a wait ran out.
constexpr unsigned int kWaitRanOut = 1;
constexpr unsigned long long kSettleNs = 1000 * 1000 * 1000;

__device__ __forceinline__ unsigned long long clock_ns()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ void give_up(volatile int *dead, unsigned int *status)
{
    *dead = 1;
    atomicExch(status, kWaitRanOut);
}

// False: the block gives up (`dead` in its shared memory says so to all its warps).
static __device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile int *dead, unsigned int *status, unsigned long long limit)
{
    const unsigned long long t0 = clock_ns();
    for (unsigned int spins = 0; limit != 0 && spins < (1u << 28); ++spins) {
        if (bar_try(bar, parity)) { return true; }
        if (*dead != 0) { return false; }
        if ((spins & 63u) == 63u && clock_ns() - t0 > limit) { break; }
    }
    give_up(dead, status);
    return false;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int *dead, const Work &w)
{
    return bar_try(bar, parity) || wait_slow(bar, parity, dead, w.status, w.wait_ns);
}

// What a CTA has asked for when its roles have ended.
struct Asked {
    int dead;
    int loads;         // steps whose copies it has asked for
    int steps, sums;   // (of the pair's first CTA) steps, and tiles or chunks of them, whose products it has asked for
};

// Where either CTA of a pair has given up: what is under way into their shared and tensor memory ends before they do.  One thread of
// each; both CTAs know what either has asked for.  The waits are bounded too, and nothing comes of one that runs out.
static __device__ __noinline__ void settle(uint32_t full, uint32_t empty, uint32_t summed, int stages, uint32_t stage_bytes, bool first,
                                           const volatile Asked &mine, const volatile Asked &other)
{
    const auto wait = [](uint32_t bar, int phase) {
        const unsigned long long t0 = clock_ns();
        while (!bar_try(bar, phase & 1) && clock_ns() - t0 < kSettleNs) {}
    };
    // products arrive at the barriers of both
    const int steps = first ? mine.steps : other.steps, sums = first ? mine.sums : other.sums;
    for (int i = max(0, steps - stages); i < steps; ++i) { wait(empty + 8 * (i % stages), i / stages); }
    for (int i = max(0, sums - 2); i < sums; ++i) { wait(summed + 8 * (i & 1), i / 2); }
    if (!first) { return; }
    // The copies of both arrive at the first one's.  A CTA that is ahead of the other in a stage has the other's bytes to go without
    // (its own arrival counts on them), or, as the second, no arrival that counts on its own.
    for (int s = 0; s < stages; ++s) {
        const auto last = [&](int loads) { return loads > s ? (loads - 1 - s) / stages : -1; };  // use of this stage
        const int a = last(mine.loads), b = last(other.loads);
        if (a < 0 && b < 0) { continue; }
        if (a > b) { bar_forgo(full + 8 * s, stage_bytes); }
        if (b > a) { bar_expect(full + 8 * s, stage_bytes); }
        wait(full + 8 * s, max(a, b));
    }
}

// What a unit is: a part of a tile of a product.
struct Unit {
    int product, tile, part;  // (the tile's number counts all products' tiles)
    int m, n, z;              // first row, tile column, result
    int from, to;             // steps of the reduction, over all halves
};

// n / d for 0 <= n < 2^23 by the quotient in 32-bit floats, which is off by one at most.  (The compiler's division, five in
// a row, cost each unit 1 us.)
__device__ __forceinline__ int divided(int n, int d)
{
    const int q = __float2int_rz(__fdividef(static_cast<float>(n), static_cast<float>(d)));
    const int r = n - q * d;
    return r < 0 ? q - 1 : r >= d ? q + 1 : q;
}

__device__ __forceinline__ Unit unit_at(const Work &w, int i)
{
    // Tiles that run at the same time share operands: bands of kBand tile rows, column by column.
    constexpr int kBand = 8;
    Unit u;
    u.product = i >= w.product[1].first_unit ? 1 : 0;
    const Product &p = w.product[u.product];
    i -= p.first_unit;
    const int steps = p.steps * p.halves;
    int tile = i;
    u.part = 0;
    u.from = 0;
    u.to = steps;
    if (p.split > 1) {  // (steps * split < 2^23 too)
        tile = divided(i, p.split);
        u.part = i - tile * p.split;
        u.from = divided(steps * u.part, p.split);
        u.to = divided(steps * (u.part + 1), p.split);
    }
    u.tile = p.first_tile + tile;
    const int per = p.m_tiles * p.n_tiles;
    int z = 0;
    for (; z + 1 < p.z && tile >= per; ++z) { tile -= per; }
    const int band = divided(tile, kBand * p.n_tiles), first = band * kBand, high = min(kBand, p.m_tiles - first);
    const int in_band = tile - first * p.n_tiles;
    u.n = divided(in_band, high);
    u.m = (first + in_band - u.n * high) * (kTileM * kCtas);
    u.z = z + p.z_first;
    return u;
}

// Where the 16 values of a block of a thread's lie in a tile's tensor memory: those of a slice side by side, of a
// gated tile half of them in either half.
template <int kN>
__device__ __forceinline__ int block_column(bool two_b, int slice, int block)
{
    constexpr int kOf = Shape<kN, false>::kValues, kHalf = Shape<kN, false>::kBlocks / 2;
    return two_b ? kOf / 2 * slice + 16 * (block % kHalf) + block / kHalf * (kN / 2) : kOf * slice + 16 * block;
}

// The values of a finished tile: in tensor memory, or in parts that are added up.
template <int kN>
struct FromTensorMemory {
    uint32_t at;
    bool two_b;
    int slice;
    uint32_t taken;
    __device__ __forceinline__ void load(int block, float (&v)[16]) const
    {
        tmem_load16(at + block_column<kN>(two_b, slice, block), v);
    }
    __device__ __forceinline__ void loaded(float (&v)[16]) const { tmem_loaded(v); }
    // The warp has all that it wanted: the memory is free for another tile.
    __device__ __forceinline__ void done() const
    {
        tmem_before_sync();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) { bar_arrive_first(taken); }
    }
};
template <int kN>
struct FromParts {
    const float *at;  // of the first part, this thread's first value
    int count;
    __device__ __forceinline__ void load(int block, float (&v)[16]) const
    {
        const float *p = at + block * 16 * 32;
        int k = 1;
        if (count > 1) {  // two parts at a time on their way
            float second[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) { v[i] = __ldcg(p + 32 * i); }
#pragma unroll
            for (int i = 0; i < 16; ++i) { second[i] = __ldcg(p + Shape<kN, false>::kPart + 32 * i); }
#pragma unroll
            for (int i = 0; i < 16; ++i) { v[i] += second[i]; }
            k = 2;
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) { v[i] = __ldcg(p + 32 * i); }
        }
        for (; k < count; k += 2) {
            float first[16], second[16];
            const bool two = k + 1 < count;
            const float *q = p + k * Shape<kN, false>::kPart;
#pragma unroll
            for (int i = 0; i < 16; ++i) { first[i] = __ldcg(q + 32 * i); }
#pragma unroll
            for (int i = 0; i < 16; ++i) { second[i] = two ? __ldcg(q + Shape<kN, false>::kPart + 32 * i) : 0.f; }
#pragma unroll
            for (int i = 0; i < 16; ++i) { v[i] = v[i] + first[i] + second[i]; }
        }
    }
    __device__ __forceinline__ void loaded(float (&)[16]) const {}
    __device__ __forceinline__ void done() const {}
};

// kWide: operands in pieces, sums of `chunk` steps added up in registers.  An Epilogue has
//   template <int kN, typename Source> void tile(const Product &, product, row of the warp's first lane, tile column, z,
//                                                slice, staging memory of the warp, Source)
// which calls the source's done() once, after its last load.
template <bool kWide, int kN, typename Epilogue>
__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kProductThreads, 1)
    product_kernel(const __grid_constant__ Work w, const __grid_constant__ Epilogue epilogue)
{
    extern __shared__ unsigned char raw[];
    __shared__ uint32_t tmem_at;
    __shared__ Asked asked[2];  // this CTA's, the other's
    using S = Shape<kN, kWide>;
    constexpr int kStages = S::kStages, kStageBytes = S::kStageBytes;
    constexpr uint32_t kColumns = 2 * kN;  // of tensor memory: one tile is summed while the other is taken
    unsigned char *ring = raw + ((1024u - (smem_at(raw) & 1023u)) & 1023u);
    unsigned char *staging = ring + kStages * kStageBytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(staging + kEpilogueWarps * kStagingBytes);
    const uint32_t ring_at = smem_at(ring), full = smem_at(bars), empty = full + 8 * kStages,
                   summed = empty + 8 * kStages, taken = summed + 16;
    volatile int *dead = &asked[0].dead;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cta_rank();

    if (threadIdx.x == 0) {
        asked[0] = Asked{};
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
    if (warp == 2) { tmem_alloc(smem_at(&tmem_at), kColumns); }
    tmem_before_sync();
    __syncthreads();
    cluster_sync();
    tmem_after_sync();
    const uint32_t tmem = tmem_at;
    const int workers = gridDim.x / kCtas, mine = blockIdx.x / kCtas;

    if (warp == 0 && lane == 0) {
        // ---- loads
        int it = 0;
        bool ok = true;
        for (int i = mine; ok && i < w.units; i += workers) {
            const Unit u = unit_at(w, i);
            const Product &p = w.product[u.product];
            const int m0 = u.m + static_cast<int>(rank) * kTileM;
            const int n0 = u.n * (p.two_b ? kN / 2 : kN) + (p.two_b ? 0 : kN / 2 * static_cast<int>(rank));
            for (int step = u.from; step < u.to; ++step, ++it) {
                const int st = it % kStages;
                ok = it < kStages || wait_for(empty + 8 * st, (it / kStages - 1) & 1, dead, w);
                if (!ok) { break; }
                const uint32_t bar = full + 8 * st, at_a = ring_at + st * kStageBytes, at_b = at_a + S::kOf * kChunkA;
                if (rank == 0) { bar_expect(bar, kCtas * kStageBytes); }
                const int second = step >= p.steps ? 1 : 0, k = (step - second * p.steps) * kStepK;
                const int slab = second * p.half_slabs + u.z * p.z_slabs;
                const CUtensorMap *b = &p.b[p.two_b ? static_cast<int>(rank) : second];
#pragma unroll
                for (int piece = 0; piece < S::kOf; ++piece) {
                    const uint32_t a_to = at_a + piece * kChunkA, b_to = at_b + piece * S::kChunkB;
                    if (p.across_a) {
                        box_load(a_to, &p.a, m0, k, slab + piece, bar);
                        box_load(a_to + kChunkA / 2, &p.a, m0 + 64, k, slab + piece, bar);
                    } else {
                        box_load(a_to, &p.a, k, m0, slab + piece, bar);
                    }
                    if (p.across_b) {
#pragma unroll
                        for (int j = 0; j < kN / kCtas; j += 64) { box_load(b_to + 128 * j, b, n0 + j, k, piece, bar); }
                    } else {
                        box_load(b_to, b, k, n0, piece, bar);
                    }
                }
            }
        }
        // The copies asked for end before the block does: with the products that read them (an arrival on `empty`).
        for (int i = max(0, it - kStages); i < it; ++i) {
            if (!wait_for(empty + 8 * (i % kStages), (i / kStages) & 1, dead, w)) { break; }
        }
        asked[0].loads = it;
    } else if (warp == 1 && lane == 0 && rank == 0) {
        // ---- products
        int it = 0, round = 0, sums = 0;
        bool ok = w.wait_ns != 0;
        if (!ok) { give_up(dead, w.status); }
        for (int i = mine; ok && i < w.units; i += workers) {
            const Unit u = unit_at(w, i);
            const Product &p = w.product[u.product];
            const uint32_t kind = p.kind;
            const bool across_a = p.across_a != 0, across_b = p.across_b != 0;
            // 16 further in the reduction: 32 bytes along the rows, or 16 rows
            const uint64_t next_a = across_a ? 128 : 2, next_b = across_b ? 128 : 2;
            const int chunk = kWide ? w.chunk : u.to - u.from;
            for (int c = u.from; ok && c < u.to; c += chunk, ++round) {
                const int buf = round & 1;
                ok = round < 2 || wait_for(taken + 8 * buf, (round / 2 - 1) & 1, dead, w);
                if (!ok) { break; }
                tmem_after_sync();
                const uint32_t d = tmem + buf * kN;
                const int steps = min(c + chunk, u.to) - c;
                for (int k = 0; k < steps; ++k, ++it) {
                    const int st = it % kStages;
                    ok = wait_for(full + 8 * st, (it / kStages) & 1, dead, w);
                    if (!ok) { break; }
                    tmem_after_sync();
                    const uint32_t at_a = ring_at + st * kStageBytes, at_b = at_a + S::kOf * kChunkA;
#pragma unroll
                    for (int pair = 0; pair < (kWide ? kPairs : 1); ++pair) {
                        const uint64_t a = operand_desc(at_a + (kWide ? kPairA[pair] * kChunkA : 0), across_a ? 64 * 128 : 16, 1024);
                        const uint64_t b = operand_desc(at_b + (kWide ? kPairB[pair] * S::kChunkB : 0), across_b ? 64 * 128 : 16, 1024);
#pragma unroll
                        for (int j = 0; j < kStepK / 16; ++j) {
                            mma16(d, a + j * next_a, b + j * next_b, kind, k > 0 || pair > 0 || j > 0);
                        }
                    }
                    mma_commit(empty + 8 * st);
                }
                if (ok) {
                    mma_commit(summed + 8 * buf);
                    ++sums;
                }
            }
        }
        asked[0].steps = it;
        asked[0].sums = sums;
    } else if (warp >= 4) {
        // ---- epilogue
        const int quarter = warp & 3, slice = (warp - 4) >> 2;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
        unsigned char *mem = staging + (warp - 4) * kStagingBytes;
        const long long place = ((static_cast<long long>(rank) * kEpilogueWarps + (warp - 4)) * S::kValues) * 32 + lane;
        int round = 0;
        bool ok = true;
        for (int i = mine; ok && i < w.units; i += workers) {
            const Unit u = unit_at(w, i);
            const Product &p = w.product[u.product];
            const bool two_b = p.two_b != 0;
            const int row = u.m + static_cast<int>(rank) * kTileM + 32 * quarter;
            const long long slot = p.split > 1 ? p.first_part + (i - p.first_unit) : w.own_part + mine;
            float *part = w.parts + slot * S::kPart + place;
            if constexpr (kWide) {
                float sum[S::kValues];
#pragma unroll
                for (int j = 0; j < S::kValues; ++j) { sum[j] = 0.f; }
                for (int c = u.from; c < u.to; c += w.chunk, ++round) {
                    const int buf = round & 1;
                    ok = __all_sync(0xffffffffu, wait_for(summed + 8 * buf, (round / 2) & 1, dead, w));
                    if (!ok) { break; }
                    tmem_after_sync();
#pragma unroll
                    for (int b = 0; b < S::kBlocks; ++b) {
                        float v[16];
                        tmem_load16(lanes + buf * kN + block_column<kN>(two_b, slice, b), v);
                        tmem_loaded(v);
#pragma unroll
                        for (int j = 0; j < 16; ++j) { sum[16 * b + j] += v[j]; }
                    }
                    tmem_before_sync();
                    __syncwarp();
                    if (lane == 0) { bar_arrive_first(taken + 8 * buf); }
                }
                if (!ok) { break; }
#pragma unroll
                for (int j = 0; j < S::kValues; ++j) { __stcg(part + 32 * j, sum[j]); }
            } else {
                const int buf = round++ & 1;
                ok = __all_sync(0xffffffffu, wait_for(summed + 8 * buf, ((round - 1) / 2) & 1, dead, w));
                if (!ok) { break; }
                tmem_after_sync();
                const FromTensorMemory<kN> from{lanes + buf * kN, two_b, slice, taken + 8 * buf};
                if (p.split == 1) {
                    epilogue.template tile<kN>(p, u.product, row, u.n, u.z, slice, mem, from);
                    continue;
                }
#pragma unroll 1
                for (int b = 0; b < S::kBlocks; ++b) {
                    float v[16];
                    from.load(b, v);
                    from.loaded(v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) { __stcg(part + 32 * (16 * b + j), v[j]); }
                }
                from.done();
            }
            // This warp's share of the tile: whoever stores the last part adds them up.
            bool last = true;
            if (p.split > 1) {
                __threadfence();
                __syncwarp();
                unsigned int before = 0;
                if (lane == 0) {
                    before = atomicAdd(w.tickets + (static_cast<long long>(u.tile) * kCtas + rank) * kEpilogueWarps + (warp - 4), 1u);
                }
                last = __shfl_sync(0xffffffffu, before, 0) + 1u == static_cast<unsigned int>(p.split);
                __threadfence();
            }
            if (last) {
                epilogue.template tile<kN>(p, u.product, row, u.n, u.z, slice, mem,
                                           FromParts<kN>{part - (p.split > 1 ? u.part * S::kPart : 0), p.split});
            }
        }
    }
    __syncwarp();
    tmem_before_sync();
    __syncthreads();
    if (threadIdx.x < 4) {
        send_word(reinterpret_cast<volatile int *>(&asked[1]) + threadIdx.x, rank ^ 1u, reinterpret_cast<volatile int *>(&asked[0])[threadIdx.x]);
    }
    cluster_sync();
    tmem_after_sync();
    if (*dead != 0 || *static_cast<volatile int *>(&asked[1].dead) != 0) {  // (the same in both CTAs)
        if (threadIdx.x == 0) { settle(full, empty, summed, kStages, kStageBytes, rank == 0, asked[0], asked[1]); }
        __syncthreads();
        cluster_sync();
        tmem_after_sync();
    }
    if (warp == 2) { tmem_free(tmem, kColumns); }
}
}  // namespace stdml::collective::train
