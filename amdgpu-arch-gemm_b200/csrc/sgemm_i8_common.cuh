// ---------------------------------------------------------------------------------------------
// Shared device code of the 8-bit kernels: typed loads and stores, mbarriers with bounded waits, TMA, tcgen05.
// An 8-bit matrix here is a column-major K x N matrix of int8 (leading dimension >= K) with one FP32 scale per column:
// column j stands for scale[j] * q[:, j].  A token's features, or an output channel's weights, are one column.
// ---------------------------------------------------------------------------------------------
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#define I8_TIMEOUT_NS 2000000000ull

extern "C" __device__ const uint32_t sgemm_i8_layout[SGEMM_I8_LAYOUT_WORDS] = SGEMM_I8_LAYOUT;   // read by sgemm_open

struct alignas(64) I8TensorMap { uint64_t opaque[16]; };

// ------------------------------------------------------------------------------- element types
template <uint32_t TYPE> struct I8Elem;
template <> struct I8Elem<SGEMM_I8_FP32> {
    using type = float;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct I8Elem<SGEMM_I8_FP16> {
    using type = __half;
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <> struct I8Elem<SGEMM_I8_BF16> {
    using type = __nv_bfloat16;
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
// element `index` of a matrix whose type is only known at run time
__device__ __forceinline__ float i8_load(const void *p, uint64_t index, uint32_t type) {
    if (type == SGEMM_I8_FP32) return static_cast<const float *>(p)[index];
    if (type == SGEMM_I8_FP16) return __half2float(static_cast<const __half *>(p)[index]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[index]);
}
__device__ __forceinline__ void i8_store(void *p, uint64_t index, uint32_t type, float v) {
    if (type == SGEMM_I8_FP32) static_cast<float *>(p)[index] = v;
    else if (type == SGEMM_I8_FP16) static_cast<__half *>(p)[index] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[index] = __float2bfloat16_rn(v);
}
// The four int8 of a word as FP32, without the conversion unit: with the sign bit flipped a byte u = q + 128 placed
// under the exponent of 2^23 is the float 2^23 + u, and the subtraction is exact.
__device__ __forceinline__ void i8_widen4(uint32_t word, float (&v)[4]) {
    const uint32_t u = word ^ 0x80808080u;
    v[0] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440)) - 8388736.0f;
    v[1] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7441)) - 8388736.0f;
    v[2] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7442)) - 8388736.0f;
    v[3] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7443)) - 8388736.0f;
}

// --------------------------------------------------------------------------------- PTX wrappers
__device__ __forceinline__ uint32_t i8_smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t i8_globaltimer() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ uint32_t i8_cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t i8_cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// True in one lane of the (converged) warp, the same one every time.  The warps that issue MMAs and copies run their loops with all lanes
// and elect one around the issuing instructions only: the compiler then knows the loop's values to be uniform and keeps
// descriptors and addresses where those instructions take them from.  With a loop inside `if (lane == 0)` a stage of four MMAs took
// its issuer 780 cycles, more than the 512 the tensor core needs for it.
__device__ __forceinline__ bool i8_elect() {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    return elected != 0u;
}
__device__ __forceinline__ void i8_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// shared::cluster address of `addr` (a shared::cta address of this CTA) in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t i8_map_to_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// Shared memory by its 32-bit address.  (Through a pointer that was aligned by hand the compiler no longer knows the address
// space and takes the generic instructions, whose latency is several times as long.  Volatile keeps their order among themselves
// and to the barriers; loads issued before their values are needed stay under way together.)
__device__ __forceinline__ uint4 i8_lds4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float i8_ldsf(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ void i8_sts4(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void i8_sts(uint32_t addr, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
// Loads from a peer's shared memory.  (No "memory" clobber: several may be under way together; the cluster barriers before and
// after them carry one.)
__device__ __forceinline__ uint4 i8_ld_cluster4u(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float4 i8_ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void i8_mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void i8_mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void i8_mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void i8_mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// The same with the instruction's default scope, for arrivals that publish nothing the waiting thread itself reads.  A release at cluster
// scope makes the warp wait until all its earlier writes are visible to the whole cluster (900 cycles beside a busy tensor core).  What such an arrival
// announces lies in this CTA's own shared memory and is read by the tensor core on the waiting thread's order: the
// writes were handed to the asynchronous proxy by a proxy fence before (or were reads of TMEM, ordered by tcgen05 fences).
__device__ __forceinline__ void i8_mbar_arrive_peer(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ uint32_t i8_mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
__device__ __forceinline__ void i8_prefetch_map(const I8TensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// TMA tile load into this CTA's shared memory, completion reported to a barrier of this CTA ...
__device__ __forceinline__ void i8_tma_load(uint32_t dst, const I8TensorMap *map, uint32_t bar, int32_t x, int32_t y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
// ... or, in a CTA pair, to a barrier of the pair's leader (`bar` is then a shared::cluster address)
__device__ __forceinline__ void i8_tma_load_pair(uint32_t dst, const I8TensorMap *map, uint32_t bar, int32_t x, int32_t y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void i8_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void i8_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
template <int GROUP> __device__ __forceinline__ void i8_tmem_alloc(uint32_t slot, uint32_t cols) {
    if (GROUP == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <int GROUP> __device__ __forceinline__ void i8_tmem_dealloc(uint32_t base, uint32_t cols) {
    if (GROUP == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
// One MMA of 32 bytes of K per operand row: int8 x int8 -> int32, or 16-bit x 16-bit -> FP32.
template <int GROUP> __device__ __forceinline__ void i8_mma_s8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if (GROUP == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void i8_mma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrive on `bar` once every MMA issued so far by this thread has completed.  In a CTA pair the barrier exists in both CTAs
// at the same offset: the leader's one commit arrives on its own and on the peer's copy (`pair_mask`: the bits of the two CTAs'
// ranks in the cluster).
template <int GROUP> __device__ __forceinline__ void i8_commit(uint32_t bar, uint16_t pair_mask) {
    if (GROUP == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"(pair_mask) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void i8_tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void i8_tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void i8_tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void i8_tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// 64-bit shared-memory matrix descriptor: start address and the two byte offsets in 16-byte units, version 1, 128-byte
// swizzle of 16-byte units.  Moving the start address by `bytes` adds bytes / 16 to the descriptor (the field never carries: shared
// memory ends below 256 KB), so the issuing thread keeps one descriptor per operand and adds constants: it issues an MMA every 128
// cycles and has little time for address arithmetic.
__device__ __forceinline__ uint64_t i8_smem_desc(uint32_t addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo_bytes >> 4) << 16) | ((uint64_t)(sbo_bytes >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}

// ------------------------------------------------------------------------------ bounded waiting
struct I8Wait {
    volatile uint32_t *abort_flag;  // shared memory, CTA-wide
    uint32_t *status;               // global memory, SGEMM_STATUS_WORDS words
    uint64_t timeout_ns;            // how long one wait may go without the barrier completing
};
__device__ __forceinline__ bool i8_wait_slow(const I8Wait &w, uint32_t bar, uint32_t parity, uint32_t tag, uint32_t tile, uint32_t kb) {
    const uint64_t t0 = i8_globaltimer();
    uint32_t spins = 0;
    for (;;) {
        if (i8_mbar_try_wait(bar, parity)) return true;
        if ((++spins & 31u) == 0u) {
            if (*w.abort_flag) return false;
            if (i8_globaltimer() - t0 > w.timeout_ns) {
                *w.abort_flag = 1u;
                if (atomicCAS(w.status, SGEMM_STATUS_OK, SGEMM_STATUS_TIMEOUT) == SGEMM_STATUS_OK) {
                    w.status[1] = tag;
                    w.status[2] = tile;
                    w.status[3] = kb;
                    w.status[4] = blockIdx.x;
                    w.status[5] = parity;
                }
                __threadfence();
                return false;
            }
        }
    }
}
__device__ __forceinline__ bool i8_wait(const I8Wait &w, uint32_t bar, uint32_t parity, uint32_t tag, uint32_t tile, uint32_t kb) {
    if (i8_mbar_try_wait(bar, parity)) return true;
    return i8_wait_slow(w, bar, parity, tag, tile, kb);
}
// The same for a whole warp: true when the barrier completed for every lane.
__device__ __forceinline__ bool i8_wait_warp(const I8Wait &w, uint32_t bar, uint32_t parity, uint32_t tag, uint32_t tile, uint32_t kb) {
    return __all_sync(0xffffffffu, i8_wait(w, bar, parity, tag, tile, kb));
}
// After a wait gave up: copies and MMAs that may still be in flight get time to land before TMEM is released.
__device__ __forceinline__ void i8_settle() {
    const uint64_t t0 = i8_globaltimer();
    while (i8_globaltimer() - t0 < 2000000ull) __nanosleep(1000);
}

// Self-test of the bounded wait (see sgemm_wait_selftest in the runner's header): a barrier nothing arrives on.
extern "C" __global__ void sgemm_wait_selftest(uint32_t *status, uint64_t timeout_ns, uint32_t tag) {
    __shared__ __align__(8) uint64_t barrier_storage;
    __shared__ uint32_t abort_flag;
    sgemm_grid_dependency_wait();
    if (threadIdx.x == 0) {
        i8_mbar_init(i8_smem_u32(&barrier_storage), 1);
        abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const I8Wait waiter{&abort_flag, status, timeout_ns};
    const bool completed = i8_wait(waiter, i8_smem_u32(&barrier_storage), 0u, tag, 0u, threadIdx.x);
    if (completed && threadIdx.x == 0) status[6] = 0xBAD0BAD0u;   // cannot happen: nobody arrives
    __syncthreads();
}
