// Softmax cross-entropy of (rows, classes) logits against one class per row, with its gradient map:
//
//   loss = sum_r [ log sum_j exp(x_rj - m_r) - (x_rt - m_r) ]  [ / count ],   m_r = max_j x_rj
//   map_rj = (exp(x_rj - m_r) / sum_r - [j = t_r])  [ / count ]
//
// A row is read once: its logits stay in registers as exp(x - m) for a maximum m of the thread's own, (m, sum) pairs are merged
// over the threads of the row, and the map is what is in the registers times one factor.  HBM-bound: 4 bytes read
// and 4 written per element in f32.
//   up to 16 classes      a thread for each row
//   up to 4 KB a row      4 to 32 threads of a warp
//   up to 1 MB a row      a CTA of up to 512 threads, 256 bytes of the row in each; beyond 128 KB a cluster of up to 8 CTAs that exchange
//                         their pairs through shared memory
//   beyond                a CTA reads the row twice (the second time mostly from L2)
// A CTA copies the rows ahead into shared memory, vector by vector as it takes a row's vectors from there into registers.
//
// A row with t < 0 does not count (padding): its map is zero and its logits are not read.  t >= classes gives NaN for the row
// and the loss.  Rows are dealt out statically and every sum has a fixed order: results are deterministic.
#include <algorithm>

#include "rtb_internal.h"
#include "rtb_cluster.cuh"

namespace rtb {
namespace {

constexpr size_t kWsHeader = 65536;   // completion counters in front of the workspace (rtb_context.cpp)
constexpr int kCountCtas = 64;

template <typename T> struct alignas(16) Vec {
    static constexpr int N = 16 / sizeof(T);
    T e[N];
};

__device__ __forceinline__ float exp_(float x) { return expf(x); }
__device__ __forceinline__ double exp_(double x) { return exp(x); }
__device__ __forceinline__ float log_(float x) { return logf(x); }
__device__ __forceinline__ double log_(double x) { return log(x); }
__device__ __forceinline__ float max_(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double max_(double a, double b) { return fmax(a, b); }
// exp for the bulk: 2^(x log2 e), the argument rounded once more, off by (|x| + 2) 2^-23 of the result at most
__device__ __forceinline__ float fast_exp(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}
__device__ __forceinline__ double fast_exp(double x) { return exp(x); }
template <typename T> __device__ __forceinline__ T lowest() { return -(T)INFINITY; }
template <typename T> __device__ __forceinline__ T nan_() { return (T)NAN; }

__device__ __forceinline__ float warp_max(float v) {
    float m;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

// (maximum m, sum of exp(x - m)) of some logits.  Entries of -inf add nothing and keep a maximum of -inf harmless; a NaN is
// skipped by the maximum and kept by the sum.
template <typename T> struct alignas(2 * sizeof(T)) Lse {
    T m, s;
    __device__ __forceinline__ T factor(T top) const { return m == lowest<T>() ? (T)1 : exp_(m - top); }
    __device__ __forceinline__ void merge(T m2, T s2) {
        const Lse o{m2, s2};
        const T top = max_(m, m2);
        s = s * factor(top) + o.s * o.factor(top);
        m = top;
    }
    template <int N> __device__ __forceinline__ void add(const T *x) {
        T top = m;
#pragma unroll
        for (int k = 0; k < N; ++k) top = max_(top, x[k]);
        if (top > m) {
            s = m == lowest<T>() ? s : s * exp_(m - top);
            m = top;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) s += x[k] == lowest<T>() ? (T)0 : exp_(x[k] - m);
    }
};

// x becomes exp(x - m) for the maximum of these n values (0 in place of a maximum of -inf)
template <typename T, int N> __device__ __forceinline__ Lse<T> exponentials(T (&x)[N]) {
    Lse<T> l{lowest<T>(), (T)0};
#pragma unroll
    for (int k = 0; k < N; ++k) l.m = max_(l.m, x[k]);
    const T base = l.m == lowest<T>() ? (T)0 : l.m;
    T part[4] = {};
#pragma unroll
    for (int k = 0; k < N; ++k) {
        x[k] = fast_exp(x[k] - base);
        part[k % 4] += x[k];
    }
    l.s = (part[0] + part[1]) + (part[2] + part[3]);
    return l;
}

// number of rows that count, as kCountCtas partial counts
__global__ void __launch_bounds__(256) xent_count_kernel(const int64_t *targets, size_t rows, unsigned long long *counts) {
    grid_dep_sync();
    unsigned long long n = 0;
    for (size_t r = (size_t)blockIdx.x * 256 + threadIdx.x; r < rows; r += (size_t)gridDim.x * 256) n += targets[r] >= 0;
    __shared__ unsigned long long sn[8];
#pragma unroll
    for (int d = 16; d; d >>= 1) n += __shfl_down_sync(0xffffffffu, n, d);
    if ((threadIdx.x & 31) == 0) sn[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) n += sn[w];
        counts[blockIdx.x] = n;
    }
}

struct XentPartial {
    double loss;
    unsigned long long rows;
};

template <typename T> struct XentArgs {
    const T *logits;
    size_t rows, classes;
    int64_t pitch;
    const int64_t *targets;
    int mean;
    const unsigned long long *counts;   // kCountCtas partial counts, or null: every CTA counts for itself
    T *loss, *map;
    XentPartial *partials;              // one for each CTA
    unsigned *done;                     // completion counter, left at zero
    unsigned cluster;
};

template <int THREADS> __device__ __forceinline__ unsigned long long block_sum(unsigned long long n, unsigned long long *smem) {
#pragma unroll
    for (int d = 16; d; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = n;
    __syncthreads();
    n = smem[0];
    for (int w = 1; w < THREADS / 32; ++w) n += smem[w];
    __syncthreads();
    return n;
}

// what the map is divided by, as a factor
template <typename T, int THREADS> __device__ __forceinline__ T map_factor(const XentArgs<T> &p, unsigned long long *smem) {
    if (!p.map || !p.mean) return (T)1;
    unsigned long long n = 0;
    if (p.counts) {
        if (threadIdx.x < kCountCtas) n = p.counts[threadIdx.x];
    } else {
        for (size_t r = threadIdx.x; r < p.rows; r += THREADS) n += p.targets[r] >= 0;
    }
    return (T)1 / (T)block_sum<THREADS>(n, smem);
}

// sum over the CTA in a fixed order, for thread 0
template <int THREADS> __device__ __forceinline__ XentPartial block_total(XentPartial v, XentPartial *smem) {
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        v.loss += __shfl_down_sync(0xffffffffu, v.loss, d);
        v.rows += __shfl_down_sync(0xffffffffu, v.rows, d);
    }
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < THREADS / 32; ++w) v.loss += smem[w].loss, v.rows += smem[w].rows;
    return v;
}

// One partial per CTA; the last CTA adds them in order.
template <typename T, int THREADS> __device__ __forceinline__ void finish_loss(const XentArgs<T> &p, XentPartial mine) {
    __shared__ XentPartial sp[THREADS / 32];
    __shared__ bool last;
    mine = block_total<THREADS>(mine, sp);
    if (threadIdx.x == 0) {
        p.partials[blockIdx.x] = mine;
        __threadfence();
        last = atomicAdd(p.done, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    XentPartial all{0.0, 0};
    for (unsigned k = threadIdx.x; k < gridDim.x; k += THREADS) {
        all.loss += __ldcg(&p.partials[k].loss);
        all.rows += __ldcg(&p.partials[k].rows);
    }
    all = block_total<THREADS>(all, sp);
    if (threadIdx.x == 0) {
        *p.loss = (T)(p.mean ? all.loss / (double)all.rows : all.loss);
        *p.done = 0;   // ready for the next launch on this stream
    }
}

// a row's loss from its maximum, sum and target logit
template <typename T> __device__ __forceinline__ double row_loss(const Lse<T> &l, T target, bool bad) {
    return bad ? (double)NAN : (double)(log_(l.s) - (target - l.m));
}

// ---- rows of up to TPR * NV packs of N: TPR threads of a warp hold a row ---------------------------------------
template <typename T, int TPR, int NV, int N>
__global__ void __launch_bounds__(256) xent_warp_kernel(const __grid_constant__ XentArgs<T> p) {
    constexpr int G = 256 / TPR;
    __shared__ unsigned long long sn[8];
    const int in_row = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    grid_dep_sync();
    const T inv_n = map_factor<T, 256>(p, sn);
    XentPartial mine{0.0, 0};
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < p.rows; r0 += (size_t)gridDim.x * G) {
        const size_t r = r0 + slot;
        const int64_t t = r < p.rows ? p.targets[r] : -1;
        const bool counted = t >= 0, bad = (uint64_t)t >= p.classes;
        const T *x = p.logits + (counted ? (int64_t)r * p.pitch : 0);
        T e[NV * N];
        T xt = (T)0;          // the target's logit, in the thread that holds it: the map may take the logits' place
        bool mine_t = false;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const size_t j = (size_t)(k * TPR + in_row) * N;
            if (counted && j < p.classes) {
                if constexpr (N > 1) {
                    const Vec<T> q = *reinterpret_cast<const Vec<T> *>(x + j);
#pragma unroll
                    for (int i = 0; i < N; ++i) e[k * N + i] = q.e[i];
                } else {
                    e[k] = x[j];
                }
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (j + i == (size_t)t) xt = e[k * N + i], mine_t = true;
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) e[k * N + i] = lowest<T>();
            }
        }
        Lse<T> l = exponentials(e);
        const Lse<T> own = l;
        // the row's maximum first: one rescaling, then a plain sum
        T top = l.m;
#pragma unroll
        for (int d = TPR / 2; d; d >>= 1) top = max_(top, __shfl_xor_sync(0xffffffffu, top, d));
        const T f = own.factor(top);
        T sum = own.s * f;
#pragma unroll
        for (int d = TPR / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        l = Lse<T>{top, sum};
        if (counted) {
            if (mine_t || (bad && in_row == 0)) mine.loss += row_loss(l, xt, bad);
            if (in_row == 0) mine.rows += 1;
        }
        if (p.map && r < p.rows) {
            T *g = p.map + r * p.classes;
            const T inv_s = bad ? nan_<T>() : (T)1 / sum;
            const T to_p = f * inv_s;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const size_t j = (size_t)(k * TPR + in_row) * N;
                if (j >= p.classes) continue;
                Vec<T> q;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    q.e[i] = counted ? (e[k * N + i] * to_p - (j + i == (size_t)t ? (T)1 : (T)0)) * inv_n : (T)0;
                if constexpr (N > 1) *reinterpret_cast<Vec<T> *>(g + j) = q;
                else g[j] = q.e[0];
            }
        }
    }
    finish_loss<T, 256>(p, mine);
}

// ---- a CTA, or each CTA of a cluster, holds THREADS * NV vectors of 16 bytes of a row ----------------------------
// Vectors lie at 16-byte boundaries of the logits; where a row starts in the middle of one (an odd number of classes), its first
// and last vectors are partly the row's.
// AHEAD rows are in shared memory or on their way; a row's vectors are taken, and replaced, in kGroups parts, so that copies never
// all wait for the last of a row.
template <typename T, int THREADS, int NV, int AHEAD>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) xent_cta_kernel(const __grid_constant__ XentArgs<T> p) {
    constexpr int kWarps = THREADS / 32, N = Vec<T>::N, kGroups = 4, kGroup = NV / kGroups;
    extern __shared__ __align__(16) unsigned char ring[];   // [row ahead][vector][thread]: a thread copies what it reads itself
    __shared__ alignas(16) Lse<T> pairs[2][kMaxCluster * kWarps];
    __shared__ unsigned long long arrived[2];
    __shared__ unsigned long long sn[kWarps];
    using P = Pack<T, N>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned nc = p.cluster, rank = nc > 1 ? cluster_rank() : 0;
    const size_t stride = gridDim.x / nc;
    const size_t row0 = blockIdx.x / nc;
    const int classes = (int)p.classes;
    grid_dep_wait();
    const T inv_n = map_factor<T, THREADS>(p, sn);
    auto target_of = [&](size_t r) { return r < p.rows ? p.targets[r] : (int64_t)-1; };
    auto slot = [&](int ahead, int k) { return reinterpret_cast<P *>(ring) + (ahead * NV + k) * THREADS + threadIdx.x; };
    auto row_at = [&](size_t r) { return p.logits + (int64_t)r * p.pitch; };
    // elements of the row's first vector that lie in front of the row
    auto phase_of = [&](const T *x) { return (int)(((uintptr_t)x & 15u) / sizeof(T)); };
    // the class of vector k's first element: below zero, or the vector beyond `classes`, at the row's ends
    auto class_of = [&](int k, int phase) { return ((int)(rank * NV + k) * THREADS + (int)threadIdx.x) * N - phase; };
    auto copy_group = [&](size_t r, int64_t t, int ahead, int group) {
        if (t >= 0) {
            const T *x = row_at(r);
            const int phase = phase_of(x);
#pragma unroll
            for (int k = group * kGroup; k < (group + 1) * kGroup; ++k) {
                const int j = class_of(k, phase);
                if (j >= classes) continue;
                if (j >= 0) {
                    copy_async_16(slot(ahead, k), x + j, j + N <= classes ? 16 : (unsigned)(classes - j) * (unsigned)sizeof(T));
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (j + i >= 0 && j + i < classes) copy_async<sizeof(T)>(&slot(ahead, k)->e[i], x + j + i);
                }
            }
        }
        copy_commit();
    };
    int64_t t_of[AHEAD + 1];   // targets of this row and of those ahead
#pragma unroll
    for (int a = 0; a <= AHEAD; ++a) t_of[a] = target_of(row0 + a * stride);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
#pragma unroll
        for (int g = 0; g < kGroups; ++g) copy_group(row0 + a * stride, t_of[a], a, g);
    int ahead = 0;
    if (nc > 1) {
        if (threadIdx.x == 0) mbar_init(&arrived[0]), mbar_init(&arrived[1]);
        cluster_barrier();   // every CTA runs, its barriers are set, before any is written to
    }
    bool lost = false;
    XentPartial mine{0.0, 0};
    unsigned counted = 0;    // rows worked on: which buffer, which phase
    for (size_t r = row0; r < p.rows; r += stride) {
        const int64_t t_far = target_of(r + (AHEAD + 1) * stride), t = t_of[0];
        const int phase = t < 0 ? 0 : phase_of(row_at(r));
        T e[NV * N];
        T xt = (T)0;          // the target's logit, in the thread that holds it: the map may take the logits' place
        bool mine_t = false;
        const bool bad = t >= (int64_t)classes, first = rank == 0 && threadIdx.x == 0;
        const int tt = bad ? -N : (int)t;   // no class in any vector where the target is beyond them
#pragma unroll
        for (int group = 0; group < kGroups; ++group) {
            copy_wait<AHEAD * kGroups - 1>();
            if (t >= 0) {
#pragma unroll
                for (int k = group * kGroup; k < (group + 1) * kGroup; ++k) {
                    const int j = class_of(k, phase);
                    P q;
                    if (j < classes) q = *slot(ahead, k);
#pragma unroll
                    for (int i = 0; i < N; ++i) e[k * N + i] = j < classes ? q.e[i] : lowest<T>();
                    if (j < 0 || j + N > classes) {
#pragma unroll
                        for (int i = 0; i < N; ++i)
                            if (j + i < 0 || j + i >= classes) e[k * N + i] = lowest<T>();
                    }
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (j + i == tt) xt = e[k * N + i], mine_t = true;
                }
            }
            copy_group(r + AHEAD * stride, t_of[AHEAD], ahead, group);
        }
        if (t < 0) {
            if (p.map) {
                T *g = p.map + r * p.classes;
                for (int j = (int)(rank * NV * THREADS * N + threadIdx.x), k = 0; k < NV * N; ++k, j += THREADS)
                    if (j < classes) g[j] = (T)0;
            }
        } else {
            const Lse<T> own = exponentials(e);
            Lse<T> l{warp_max(own.m), (T)0};
            l.s = own.s * own.factor(l.m);
#pragma unroll
            for (int d = 16; d; d >>= 1) l.s += __shfl_xor_sync(0xffffffffu, l.s, d);
            const int buf = (int)(counted & 1);   // a warp is never a whole row ahead of another: two buffers suffice
            if (nc > 1) {
                if (threadIdx.x == 0) mbar_expect(&arrived[buf], nc * kWarps * sizeof(Lse<T>));
                if (lane < (int)nc) send(in_cta(smem_addr(&pairs[buf][rank * kWarps + warp]), lane), l, in_cta(smem_addr(&arrived[buf]), lane));
                if (!lost && !mbar_wait(&arrived[buf], (counted >> 1) & 1u)) lost = true;
            } else {
                if (lane == 0) pairs[buf][warp] = l;
                __syncthreads();
            }
            ++counted;
            // all warps merge the pairs the same way
            T m = lowest<T>();
            for (unsigned k = lane; k < nc * kWarps; k += 32) m = max_(m, pairs[buf][k].m);
            m = warp_max(m);
            T sum = (T)0;
            for (unsigned k = lane; k < nc * kWarps; k += 32) sum += pairs[buf][k].s * pairs[buf][k].factor(m);
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lost) sum = nan_<T>();
            if (mine_t || (bad && first)) mine.loss += row_loss(Lse<T>{m, sum}, xt, bad);
            if (first) mine.rows += 1;
            if (p.map) {
                T *g = p.map + r * p.classes;
                const bool whole = ((uintptr_t)(g - phase) & 15u) == 0;   // the map's vectors lie as the logits' do
                const T inv_s = bad ? nan_<T>() : (T)1 / sum;
                const T to_p = own.factor(m) * inv_s, to_map = to_p * inv_n;
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int j = class_of(k, phase);
                    if (j >= classes) continue;
                    P q;
#pragma unroll
                    for (int i = 0; i < N; ++i) q.e[i] = e[k * N + i] * to_map;
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (j + i == tt) q.e[i] = (e[k * N + i] * to_p - (T)1) * inv_n;
                    if (whole && j >= 0 && j + N <= classes) {
                        st<T, N>(g + j, q);
                    } else {
#pragma unroll
                        for (int i = 0; i < N; ++i)
                            if (j + i >= 0 && j + i < classes) g[j + i] = q.e[i];
                    }
                }
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) t_of[a] = t_of[a + 1];
        t_of[AHEAD] = t_far;
        ahead = ahead + 1 == AHEAD ? 0 : ahead + 1;
    }
    grid_dep_launch();
    if (nc > 1) cluster_barrier();   // no CTA leaves while another may still write to it
    finish_loss<T, THREADS>(p, mine);
}

// ---- any row: a CTA reads it twice ------------------------------------------------------------------------
template <typename T, int N>
__global__ void __launch_bounds__(512) xent_twice_kernel(const __grid_constant__ XentArgs<T> p) {
    constexpr int THREADS = 512, kWarps = THREADS / 32;
    __shared__ Lse<T> pairs[kWarps];
    __shared__ unsigned long long sn[kWarps];
    using P = Pack<T, N>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dep_sync();
    const T inv_n = map_factor<T, THREADS>(p, sn);
    XentPartial mine{0.0, 0};
    const size_t packs = p.classes / N;
    for (size_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const int64_t t = p.targets[r];
        const T *x = p.logits + (t < 0 ? 0 : (int64_t)r * p.pitch);
        T *g = p.map ? p.map + r * p.classes : nullptr;
        if (t < 0) {
            if (g)
                for (size_t k = threadIdx.x; k < packs; k += THREADS) st<T, N>(g + k * N, P{});
            continue;
        }
        Lse<T> l{lowest<T>(), (T)0};
        for (size_t k = threadIdx.x; k < packs; k += THREADS) l.template add<N>(ld<T, N>(x + k * N).e);
#pragma unroll
        for (int d = 16; d; d >>= 1) l.merge(__shfl_xor_sync(0xffffffffu, l.m, d), __shfl_xor_sync(0xffffffffu, l.s, d));
        if (lane == 0) pairs[warp] = l;
        __syncthreads();
        l = pairs[0];
        for (int w = 1; w < kWarps; ++w) l.merge(pairs[w].m, pairs[w].s);
        const bool bad = (uint64_t)t >= p.classes;
        if (threadIdx.x == 0) {
            mine.loss += row_loss(l, bad ? (T)0 : x[t], bad);
            mine.rows += 1;
        }
        __syncthreads();   // the pairs are written again for the next row, x[t] may be overwritten below
        if (g) {
            const T inv_s = bad ? nan_<T>() : (T)1 / l.s;
            for (size_t k = threadIdx.x; k < packs; k += THREADS) {
                P q = ld<T, N>(x + k * N);
#pragma unroll
                for (int j = 0; j < N; ++j) q.e[j] = (exp_(q.e[j] - l.m) * inv_s - (k * N + j == (size_t)t ? (T)1 : (T)0)) * inv_n;
                st<T, N>(g + k * N, q);
            }
        }
    }
    finish_loss<T, THREADS>(p, mine);
}

// ---- host ------------------------------------------------------------------------------------------------
// Every CTA counts the targets for itself up to this many rows (32 KB of them, from L2); beyond, a kernel of its own counts.
constexpr size_t kCountRows = 4096;

template <typename T, void (*kernel)(XentArgs<T>)> int run(Ctx *ctx, const char *name, XentArgs<T> &p, size_t grid, unsigned threads, size_t smem) {
    void *ws = nullptr;
    if (int rc = workspace(ctx, 1024 + grid * sizeof(XentPartial), &ws)) return rc;
    unsigned long long *counts = (unsigned long long *)((char *)ws + kWsHeader);
    p.partials = (XentPartial *)((char *)ws + kWsHeader + 1024);
    p.done = (unsigned *)ws;
    if (p.map && p.mean && p.rows > kCountRows) {
        launch_dep(ctx, kCountCtas, 256, xent_count_kernel, p.targets, p.rows, counts);
        if (int rc = check_launch(ctx, "xent_count_kernel")) return rc;
        p.counts = counts;
    }
    // behind the tiny count, or short itself: it may start early
    return launch_cluster<XentArgs<T>, kernel>(ctx, name, grid, threads, p.cluster, smem, p.counts || p.rows * p.classes <= (size_t(1) << 24), p);
}

template <typename T, int TPR, int NV, int N> int run_warp(Ctx *ctx, XentArgs<T> &p) {
    constexpr size_t G = 256 / TPR;
    const size_t grid = std::min<size_t>(std::max<size_t>(1, (p.rows + G - 1) / G), (size_t)ctx->sm_count * 8);
    return run<T, xent_warp_kernel<T, TPR, NV, N>>(ctx, "xent_warp_kernel", p, grid, 256, 0);
}

template <typename T, int THREADS, int NV, int AHEAD> int run_cta(Ctx *ctx, XentArgs<T> &p, unsigned cluster) {
    constexpr size_t smem = (size_t)AHEAD * THREADS * NV * 16;
    p.cluster = cluster;
    // as many clusters as run at once (a CTA of 512 threads fills an SM, four of 128 do), the rows dealt out among them
    unsigned fit = 0;
    if (int rc = clusters_at_once<XentArgs<T>, xent_cta_kernel<T, THREADS, NV, AHEAD>>(ctx, THREADS, cluster, smem, &fit)) return rc;
    const size_t clusters = std::max<size_t>(1, std::min<size_t>(p.rows, fit));
    return run<T, xent_cta_kernel<T, THREADS, NV, AHEAD>>(ctx, "xent_cta_kernel", p, clusters * cluster, THREADS, smem);
}

template <typename T> int pick_size(Ctx *ctx, XentArgs<T> &p, bool vec) {
    constexpr int N = Vec<T>::N;
    const size_t n = p.classes, bytes = n * sizeof(T);
    if (n <= 16) return run_warp<T, 1, 16, 1>(ctx, p);
    if (vec) {
        if (n <= 64) return run_warp<T, 4, 16 / N, N>(ctx, p);
        if (n <= 128) return run_warp<T, 8, 16 / N, N>(ctx, p);
        if (n <= 256) return run_warp<T, 16, 16 / N, N>(ctx, p);
        if (bytes <= 4096) return run_warp<T, 32, 8, N>(ctx, p);
    } else {
        if (n <= 64) return run_warp<T, 8, 8, 1>(ctx, p);
        if (n <= 256) return run_warp<T, 32, 8, 1>(ctx, p);
        if (bytes <= 4096) return run_warp<T, 32, 128 / (int)sizeof(T), 1>(ctx, p);
    }
    const size_t room = bytes + 16;   // a row that starts inside a vector takes one more
    if (room <= 128 * 8 * 16) return run_cta<T, 128, 8, 3>(ctx, p, 1);
    if (room <= 128 * 16 * 16) return run_cta<T, 128, 16, 1>(ctx, p, 1);
    if (room <= 256 * 16 * 16) return run_cta<T, 256, 16, 1>(ctx, p, 1);
    for (unsigned cluster = 1; cluster <= kMaxCluster; cluster *= 2)
        if (room <= (size_t)cluster * 512 * 16 * 16) return run_cta<T, 512, 16, 1>(ctx, p, cluster);
    const size_t grid = std::min<size_t>(p.rows, (size_t)ctx->sm_count * 4);
    if (vec) return run<T, xent_twice_kernel<T, N>>(ctx, "xent_twice_kernel", p, grid, 512, 0);
    return run<T, xent_twice_kernel<T, 1>>(ctx, "xent_twice_kernel", p, grid, 512, 0);
}

template <typename T>
int pick(Ctx *ctx, const T *logits, size_t rows, size_t classes, int64_t pitch, const int64_t *targets, int mean, T *loss, T *map) {
    constexpr size_t N = Vec<T>::N;
    std::lock_guard<std::mutex> lock(ctx->ws_mu);
    XentArgs<T> p{};
    p.logits = logits, p.rows = rows, p.classes = classes, p.pitch = pitch, p.targets = targets, p.mean = mean, p.loss = loss, p.map = map;
    p.cluster = 1;
    const bool vec = classes % N == 0 && pitch % (int64_t)N == 0 && (((uintptr_t)logits | (uintptr_t)map) & 15u) == 0;
    return pick_size<T>(ctx, p, vec);
}

}  // namespace
}  // namespace rtb

using namespace rtb;

RTB_API int rtb_cross_entropy(rtb_ctx *c, int dtype, const void *logits, size_t rows, size_t classes, ptrdiff_t pitch, const int64_t *targets,
                              int reduction, void *loss, void *grad_map) {
    if (!c || !loss) return fail(RTB_ERR_INVALID, "null argument");
    if (dtype != RTB_F32 && dtype != RTB_F64) return fail(RTB_ERR_DTYPE, "cross-entropy is defined for f32 and f64 only");
    if (reduction != 0 && reduction != 1) return fail(RTB_ERR_INVALID, "reduction must be 0 (mean) or 1 (sum)");
    if (rows && !targets) return fail(RTB_ERR_INVALID, "null targets");
    if (rows && classes && !logits) return fail(RTB_ERR_INVALID, "null logits");
    Ctx *ctx = reinterpret_cast<Ctx *>(c);
    if (int rc = use_device(ctx)) return rc;
    if (dtype == RTB_F32)
        return pick<float>(ctx, (const float *)logits, rows, classes, (int64_t)pitch, targets, reduction == 0, (float *)loss, (float *)grad_map);
    return pick<double>(ctx, (const double *)logits, rows, classes, (int64_t)pitch, targets, reduction == 0, (double *)loss, (double *)grad_map);
}
