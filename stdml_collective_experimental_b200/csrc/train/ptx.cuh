// The instructions of sm_100a that the products are made of, each under a name.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace stdml::collective::train
{
__device__ __forceinline__ uint32_t smem_at(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ uint32_t cta_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The two halves of it.  A block's shared memory may be written by the others only once it runs: they arrive as they begin, and
// wait before they send.
__device__ __forceinline__ void cluster_begin() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_runs() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// ------------------------------------------------------------ barriers in shared memory
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_visible()
{
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Bytes that will not come count as if they had.
__device__ __forceinline__ void bar_forgo(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// To the same place in a CTA of the cluster.
__device__ __forceinline__ void send_word(const volatile int *place, uint32_t cta, int v)
{
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_at(const_cast<const int *>(place))), "r"(cta));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
// On the barrier at the same place in the cluster's first CTA.  Orders nothing: a release would wait for the stores under
// way (a third of the time of an epilogue).
__device__ __forceinline__ void bar_arrive_first(uint32_t bar)
{
    asm volatile("{\n\t"
                 ".reg .b32 at;\n\t"
                 "mapa.shared::cluster.u32 at, %0, 0;\n\t"
                 "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [at];\n\t"
                 "}" ::"r"(bar)
                 : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n\t"
                 ".reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t"
                 "}"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done != 0;
}

// ------------------------------------------------------------ TMA
// A box at (x, y, z) of a tensor of this GPU; the bytes are counted on the barrier of the pair's first CTA, at the same
// place.
__device__ __forceinline__ void box_load(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
                 "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar & 0xFEFFFFFFu)
                 : "memory");
}

// ------------------------------------------------------------ tensor memory and products
__device__ __forceinline__ void tmem_alloc(uint32_t to, uint32_t columns)
{
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns)
{
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void tmem_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 16 columns of the warp's 32 lanes, one lane to a thread.
__device__ __forceinline__ void tmem_load16(uint32_t at, float (&v)[16])
{
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}
// Waits for the loads so far; the values pass through, so that nothing uses them earlier.
__device__ __forceinline__ void tmem_loaded(float (&v)[16])
{
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

// Shared-memory operand in tiles of 128-byte rows, swizzled over 8 of them (1024 bytes).
//   reduction along the rows: groups of 8 rows `group` bytes apart
//   reduction across them: the same for 8 steps of the reduction, the next 64 elements of the other dimension `lead` bytes on
__device__ __forceinline__ uint64_t operand_desc(uint32_t at, uint32_t lead, uint32_t group)
{
    return static_cast<uint64_t>((at & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) |
           (static_cast<uint64_t>(group >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// D (+)= A B over 16 of the reduction; issued by one thread.
__device__ __forceinline__ void mma16(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add)
{
    const uint32_t on = add ? 1u : 0u;
    asm volatile("{\n\t"
                 ".reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
                 "}" ::"r"(d),
                 "l"(a), "l"(b), "r"(kind), "r"(on)
                 : "memory");
}
// The barrier of both CTAs of the pair is arrived at when all products issued so far are done.
__device__ __forceinline__ void mma_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
}
}  // namespace stdml::collective::train
