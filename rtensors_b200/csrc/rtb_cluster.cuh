// What kernels that work in thread-block clusters share: vectors, asynchronous copies into a ring of shared-memory stages, the
// exchange of small values between the CTAs of a cluster, and the launch.
#pragma once
#include "rtb_internal.h"

namespace rtb {

constexpr unsigned kMaxCluster = 8;                     // the portable size
constexpr unsigned kWideCluster = 16;                   // what a kernel may opt in to; a device need not be able to place it
constexpr unsigned long long kWaitNs = 2000000000ull;   // limit of a wait for another CTA's values
constexpr uint64_t kMaxGrid = 0x7fffffffull;

// A limit by device that only ever rises, shared by all contexts and threads: `set` is what raises it, never while another raise
// is under way, so that a smaller one cannot come last.
class RisingLimit {
    std::mutex mu;
    std::atomic<size_t> reached[64] = {};

  public:
    template <typename F> int raise(int device, size_t to, F set) {
        std::atomic<size_t> &mark = reached[device & 63];
        if (mark.load(std::memory_order_acquire) >= to) return RTB_OK;
        std::lock_guard<std::mutex> lock(mu);
        if (mark.load(std::memory_order_relaxed) >= to) return RTB_OK;
        if (int rc = set()) return rc;
        mark.store(to, std::memory_order_release);
        return RTB_OK;
    }
};

#ifdef __CUDACC__
template <typename T, int V> struct alignas(sizeof(T) * V) Pack {
    T e[V];
};
template <typename T, int V> __device__ __forceinline__ Pack<T, V> ld(const T *p) { return *reinterpret_cast<const Pack<T, V> *>(p); }
template <typename T, int V> __device__ __forceinline__ void st(T *p, const Pack<T, V> &v) { *reinterpret_cast<Pack<T, V> *>(p) = v; }

// asynchronous copy of BYTES (4, 8 or 16) into shared memory
template <int BYTES> __device__ __forceinline__ void copy_async(void *smem, const void *gmem) {
    const unsigned dst = (unsigned)__cvta_generic_to_shared(smem);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(gmem) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(gmem), "n"(BYTES) : "memory");
}
// the same for 16 bytes of which only `valid` lie in the source; the rest becomes zero and is not read
__device__ __forceinline__ void copy_async_16(void *smem, const void *gmem, unsigned valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(smem)), "l"(gmem), "r"(valid) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
// Values travel between the CTAs of a cluster as asynchronous stores that count their bytes on a barrier of the receiver: unlike
// a cluster-wide barrier they do not wait for the sender's own global stores.
__device__ __forceinline__ unsigned smem_addr(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ unsigned in_cta(unsigned addr, unsigned rank) {
    unsigned at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    return at;
}
template <typename P> __device__ __forceinline__ void send(unsigned to, const P &v, unsigned mbar) {
    static_assert(sizeof(P) == 4 || sizeof(P) == 8 || sizeof(P) == 16, "one store");
    if constexpr (sizeof(P) == 16) {
        uint4 q;
        memcpy(&q, &v, 16);
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "r"(q.x),
                     "r"(q.y), "r"(q.z), "r"(q.w), "r"(mbar) : "memory");
    } else if constexpr (sizeof(P) == 8) {
        unsigned long long q;
        memcpy(&q, &v, 8);
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(to), "l"(q), "r"(mbar) : "memory");
    } else {
        unsigned q;
        memcpy(&q, &v, 4);
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(to), "r"(q), "r"(mbar) : "memory");
    }
}
__device__ __forceinline__ void mbar_init(unsigned long long *bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(bar)) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_expect(unsigned long long *bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// -> whether the phase completed within the limit
__device__ __forceinline__ bool mbar_wait(unsigned long long *bar, unsigned parity) {
    unsigned long long began = 0;
    for (;;) {
        unsigned done;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                     : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
        if (done) return true;
        if (!began) began = now_ns();
        else if (now_ns() - began > kWaitNs) return false;
    }
}

// Allows a kernel `smem` bytes of dynamic shared memory (on first use on a device; each kernel instantiates this function).
template <typename A, void (*kernel)(A)> int allow_smem(Ctx *ctx, size_t smem) {
    static RisingLimit limit;
    return limit.raise(ctx->device, smem, [&]() -> int {
        RTB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        return RTB_OK;
    });
}

// How many clusters of `cluster` CTAs (1 to 16) of a kernel an idle device runs at once; above 8 it may be none, and a size must
// have been asked for before it is launched.  Asked once per device and size.
template <typename A, void (*kernel)(A)> int clusters_at_once(Ctx *ctx, unsigned threads, unsigned cluster, size_t smem, unsigned *out) {
    static std::atomic<unsigned> known[64][kWideCluster + 1];   // one more than the answer
    std::atomic<unsigned> &mark = known[ctx->device & 63][cluster];
    unsigned n = mark.load(std::memory_order_relaxed);
    if (!n) {
        if (int rc = allow_smem<A, kernel>(ctx, smem)) return rc;
        if (cluster > kMaxCluster) RTB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        int got = 0;
        if (cluster == 1) {
            RTB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&got, kernel, (int)threads, smem));
            got *= ctx->sm_count;
        } else {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(cluster);
            cfg.blockDim = dim3(threads);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            RTB_CUDA(cudaOccupancyMaxActiveClusters(&got, kernel, &cfg));
        }
        n = got > 0 ? (unsigned)got + 1 : cluster > kMaxCluster ? 1 : 2;
        mark.store(n, std::memory_order_relaxed);
    }
    *out = n - 1;
    return RTB_OK;
}

// Launches `kernel` with `smem` bytes of dynamic shared memory in clusters of `cluster` CTAs.  early: the grid may start beside
// its predecessor's last CTAs (programmatic dependent launch).  A long-running grid of one wave should not: it lands on
// the SMs that happen to be free and stays there (f32 (1, 65536, 256) with 4 heads, backward: 126 us early, 78 us not).
template <typename A, void (*kernel)(A)>
int launch_cluster(Ctx *ctx, const char *name, uint64_t grid, unsigned threads, unsigned cluster, size_t smem, bool early, const A &args) {
    if (grid > kMaxGrid) return fail(RTB_ERR_TOO_LARGE, "%s: %zu CTAs are beyond one launch", name, (size_t)grid);
    if (int rc = allow_smem<A, kernel>(ctx, smem)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster, attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (early) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = n ? attr : nullptr;
    cfg.numAttrs = n;
    (void)cudaLaunchKernelEx(&cfg, kernel, args);
    return check_launch(ctx, name);
}
#endif

}  // namespace rtb
