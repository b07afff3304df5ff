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
//   up to 1 MB a row      a CTA of up to 1024 threads, 128 bytes of the row in each; beyond 128 KB a cluster of up to 8 CTAs that exchange
//                         their pairs through shared memory
//   beyond                a CTA reads the row twice (the second time mostly from L2)
// A CTA copies the rows ahead into shared memory, vector by vector as it takes a row's vectors from there into registers.
// f32 with the map: 8192 x 32000 340 us (6.2 TB/s), 16384 x 8192 202 us (5.3), 2048 x 131072 400 us (5.4, clusters of four),
// 65536 x 1024 97 us (5.5), 262144 x 64 35 us (3.8), 1000000 x 10 46 us (1.7: single 4-byte loads, two barriers a tile); 4096 x 10
// 6 us, a chain of latencies; read twice, 2048 x 300000 1842 us.  The loss alone: 8192 x 32000 227 us (4.6 TB/s): half
// the bytes, two thirds of the time.
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

// Sums of exponentials are kept relative to a shift c that depends on a maximum m of the logits alone.  f64: c = m, s = sum of
// exp(x - m).  f32, |m| <= kNear: powers of two, 2c = rint(m log2 e) and s = sum of 2^(x log2 e - 2c): one fused multiply-add rounds each
// exponent once, and bringing sums to a common shift is exact.  That needs m log2 e below 2^23: its own rounding, which stays in every
// exponent, is then a quarter at most (from 2^31 on it would be 128 and more, an overflow).  f32 beyond kNear, masks of
// -1e9 and the like: c = m and s = sum of exp(x - m), as in f64.  The near shifts are halved so that |c| <= 0.73 kNear: a shift tells of
// which kind it is, shifts have the order of their maxima, and those of different far maxima differ.
// c = -inf: no logit above -inf yet.  A NaN is skipped by the maximum and kept by the sum.
constexpr float kLog2e = 1.4426950408889634f, kNear = 4194304.0f;   // 2^22
template <typename T> struct alignas(2 * sizeof(T)) Lse {
    T c, s;
};
__device__ __forceinline__ bool is_far(float c) { return fabsf(c) > kNear; }   // of a maximum or of its shift
__device__ __forceinline__ bool is_far(double) { return false; }
__device__ __forceinline__ float shift_of(float m) { return is_far(m) ? m : 0.5f * rintf(m * kLog2e); }
__device__ __forceinline__ double shift_of(double m) { return m; }
__device__ __forceinline__ float exp2_(float x) {   // zero below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// what a sum of shift c is multiplied by to have the shift `top` >= c
__device__ __forceinline__ float rescale(float c, float top) {
    if (fmaxf(fabsf(c), fabsf(top)) > kNear) {   // log2 of e^c / e^top, whichever way either is written
        const bool fc = is_far(c), ft = is_far(top);
        const float d = fmaf(fc ? (ft ? c - top : c) : -top, kLog2e, fc ? (ft ? 0.0f : -2.0f * top) : 2.0f * c);
        return c == -INFINITY ? 1.0f : exp2_(d);
    }
    const float d = 2.0f * (c - top);   // a whole number
    return d >= -126.0f ? __int_as_float(((int)d + 127) << 23) : 0.0f;
}
__device__ __forceinline__ double rescale(double c, double top) { return c == -(double)INFINITY ? 1.0 : exp(c - top); }
// exponential of x relative to a near shift, given as 2c, or to the maximum itself
__device__ __forceinline__ float exp_near(float x, float c2) { return exp2_(fmaf(x, kLog2e, -c2)); }
__device__ __forceinline__ float exp_far(float x, float m) { return exp2_((x - m) * kLog2e); }
__device__ __forceinline__ double exp_near(double x, double m) { return exp(x - m); }
__device__ __forceinline__ double exp_far(double x, double m) { return exp(x - m); }
__device__ __forceinline__ float near_base(float shift) { return 2.0f * shift; }
__device__ __forceinline__ double near_base(double shift) { return shift; }
// x becomes the exponentials of N values
template <typename T, int N> __device__ __forceinline__ Lse<T> lse_of(T (&x)[N]) {
    T m[4] = {lowest<T>(), lowest<T>(), lowest<T>(), lowest<T>()}, s[4] = {};
#pragma unroll
    for (int k = 0; k < N; ++k) m[k % 4] = max_(m[k % 4], x[k]);
    const T top = max_(max_(m[0], m[1]), max_(m[2], m[3]));
    const T shift = shift_of(top);
    if (is_far(top) && top != lowest<T>()) {
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = exp_far(x[k], top);
    } else {
        const T base = top == lowest<T>() ? (T)0 : near_base(shift);
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = exp_near(x[k], base);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) s[k % 4] += x[k];
    return Lse<T>{shift, (s[0] + s[1]) + (s[2] + s[3])};
}
// log(sum of exponentials) - target, without cancellation where the target is near the maximum.  Far from zero in 64 bits: in f32 the
// distance of a masked target times log2 e, or the sum of such losses, would overflow though the loss or the mean fits.
__device__ __forceinline__ double minus_log(const Lse<float> &l, float target) {
    if (is_far(l.c)) return (double)logf(l.s) + ((double)l.c - (double)target);
    if (is_far(target)) return 0.6931471805599453 * ((double)log2f(l.s) + (2.0 * (double)l.c - (double)target * (double)kLog2e));
    return 0.6931471805599453f * (log2f(l.s) - fmaf(target, kLog2e, -2.0f * l.c));
}
__device__ __forceinline__ double minus_log(const Lse<double> &l, double target) { return log(l.s) - (target - l.c); }

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

// ---- rows of up to TPR * NV packs of N: TPR threads of a warp hold a row ---------------------------------------
template <typename T, int TPR, int NV, int N>
__global__ void __launch_bounds__(256) xent_warp_kernel(const __grid_constant__ XentArgs<T> p) {
    constexpr int G = 256 / TPR;
    __shared__ unsigned long long sn[8];
    const int in_row = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    grid_dep_sync();
    const T inv_n = map_factor<T, 256>(p, sn);
    // one thread a row: its map goes through shared memory, so that a warp writes consecutive addresses
    __shared__ alignas(16) T tile[TPR == 1 ? 256 * NV * N : 1];
    XentPartial mine{0.0, 0};
    const size_t step = (size_t)gridDim.x * G;
    int64_t t_next = (size_t)blockIdx.x * G + slot < p.rows ? p.targets[(size_t)blockIdx.x * G + slot] : -1;
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < p.rows; r0 += step) {
        const size_t r = r0 + slot;
        const int64_t t = t_next;
        t_next = r + step < p.rows ? p.targets[r + step] : -1;   // ahead: whether a row is read depends on it
        const bool counted = t >= 0, bad = (uint64_t)t >= p.classes;
        const int tt = bad ? -1 : (int)t;
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
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) e[k * N + i] = lowest<T>();
            }
        }
#pragma unroll
        for (int k = 0; k < NV * N; ++k)
            if ((k / N * TPR + in_row) * N + k % N == tt) xt = e[k], mine_t = counted;
        const Lse<T> own = lse_of(e);
        // the row's shift first: one rescaling, then a plain sum
        T top = own.c;
#pragma unroll
        for (int d = TPR / 2; d; d >>= 1) top = max_(top, __shfl_xor_sync(0xffffffffu, top, d));
        const T f = rescale(own.c, top);
        T sum = own.s * f;
#pragma unroll
        for (int d = TPR / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (counted) {
            if (mine_t) mine.loss += minus_log(Lse<T>{top, sum}, xt);
            if (bad && in_row == 0) mine.loss = NAN;
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
                    q.e[i] = counted ? (e[k * N + i] * to_p - ((int)j + i == tt ? (T)1 : (T)0)) * inv_n : (T)0;
                if constexpr (TPR == 1) tile[slot * p.classes + j] = q.e[0];
                else if constexpr (N > 1) *reinterpret_cast<Vec<T> *>(g + j) = q;
                else g[j] = q.e[0];
            }
        }
        if constexpr (TPR == 1) {
            if (p.map) {
                const size_t n = min((size_t)G, p.rows - r0) * p.classes;
                __syncthreads();
                for (size_t i = threadIdx.x; i < n; i += 256) p.map[r0 * p.classes + i] = tile[i];
                __syncthreads();
            }
        }
    }
    finish_loss<T, 256>(p, mine);
}

// ---- a CTA, or each CTA of a cluster, holds THREADS * NV vectors of 16 bytes of a row ----------------------------
// Vectors lie at 16-byte boundaries of the logits; where a row starts in the middle of one (an odd number of classes), its first
// and last vectors are partly the row's.
// AHEAD rows are in shared memory or on their way.  A row's vectors are taken, and replaced by a later row's, one by one, so that
// copies never all wait for the last of a row.
// ALIGNED: every row is whole vectors.
template <typename T, int THREADS, int NV, int AHEAD, bool ALIGNED>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) xent_cta_kernel(const __grid_constant__ XentArgs<T> p) {
    constexpr int kWarps = THREADS / 32, N = Vec<T>::N;
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
    auto phase_of = [&](const T *x) { return ALIGNED ? 0 : (int)(((uintptr_t)x & 15u) / sizeof(T)); };
    // the class of the thread's first vector's first element; that of vector k is k * kStep further, below zero or its vector
    // beyond `classes` at the row's ends
    constexpr int kStep = THREADS * N;
    const int class0 = (int)(rank * NV * THREADS + threadIdx.x) * N;
    struct Row {
        const T *x;      // the thread's first class, possibly in front of the row
        int first, left; // its number; classes from it to the end (0: nothing to copy)
    };
    auto row_of = [&](size_t r, int64_t t) {
        const T *x = row_at(t < 0 ? 0 : r);
        const int first = class0 - phase_of(x);
        return Row{x + first, first, t < 0 ? 0 : classes - first};
    };
    auto copy_vector = [&](const Row &row, int ahead, int k) {
        if (k * kStep < row.left) {
            if (ALIGNED) {
                copy_async<16>(slot(ahead, k), row.x + k * kStep);
            } else if (k > 0 || row.first >= 0) {
                copy_async_16(slot(ahead, k), row.x + k * kStep, k * kStep + N <= row.left ? 16 : (unsigned)(row.left - k * kStep) * (unsigned)sizeof(T));
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (row.first + i >= 0 && i < row.left) copy_async<sizeof(T)>(&slot(ahead, k)->e[i], row.x + i);
            }
        }
        copy_commit();
    };
    int64_t t_of[AHEAD + 1];   // targets of this row and of those ahead
#pragma unroll
    for (int d = 0; d <= AHEAD; ++d) t_of[d] = target_of(row0 + d * stride);
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
        const Row row = row_of(row0 + d * stride, t_of[d]);
#pragma unroll
        for (int k = 0; k < NV; ++k)
            copy_vector(row, d, k);
    }
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
        const Row row = row_of(r, t), later = row_of(r + AHEAD * stride, t_of[AHEAD]);
        T e[NV * N];
        T xt = (T)0;          // the target's logit, in the thread that holds it: the map may take the logits' place
        const bool bad = t >= (int64_t)classes, leader = rank == 0 && threadIdx.x == 0;
        const int tt = (int)t - row.first;   // the target seen from the thread's first class
        const bool mine_t = t >= 0 && !bad && tt >= 0 && tt < NV * kStep && tt % kStep < N;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            copy_wait<AHEAD * NV - 1>();
            if (k * kStep < row.left) {
                const P q = *slot(ahead, k);
#pragma unroll
                for (int i = 0; i < N; ++i) e[k * N + i] = q.e[i];
                if (!ALIGNED && ((k == 0 && row.first < 0) || k * kStep + N > row.left)) {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (row.first + k * kStep + i < 0 || k * kStep + i >= row.left) e[k * N + i] = lowest<T>();
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) e[k * N + i] = lowest<T>();
            }
            copy_vector(later, ahead, k);
        }
        if (mine_t) {
#pragma unroll
            for (int k = 0; k < NV * N; ++k)
                if (k / N * kStep + k % N == tt) xt = e[k];
        }
        if (t < 0) {
            if (p.map) {
                T *g = p.map + r * p.classes;
                for (int j = (int)(rank * NV * THREADS * N + threadIdx.x), k = 0; k < NV * N; ++k, j += THREADS)
                    if (j < classes) g[j] = (T)0;
            }
        } else {
            const Lse<T> own = lse_of(e);
            Lse<T> l{warp_max(own.c), (T)0};
            l.s = own.s * rescale(own.c, l.c);
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
            T c = lowest<T>();
            for (unsigned k = lane; k < nc * kWarps; k += 32) c = max_(c, pairs[buf][k].c);
            c = warp_max(c);
            T sum = (T)0;
            for (unsigned k = lane; k < nc * kWarps; k += 32) sum += pairs[buf][k].s * rescale(pairs[buf][k].c, c);
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lost) sum = nan_<T>();
            const T inv_s = bad ? nan_<T>() : (T)1 / sum;
            const T to_p = rescale(own.c, c) * inv_s, to_map = to_p * inv_n;
            if (leader) mine.rows += 1;
            if (leader && bad) mine.loss = NAN;
            T et = (T)0;
            if (mine_t) {
#pragma unroll
                for (int k = 0; k < NV * N; ++k)
                    if (k / N * kStep + k % N == tt) et = e[k];
                mine.loss += minus_log(Lse<T>{c, sum}, xt);
            }
            if (p.map) {
                T *g = p.map + r * p.classes;
                g += row.first;
                const bool whole = ALIGNED || ((uintptr_t)g & 15u) == 0;   // the map's vectors lie as the logits' do
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    if (k * kStep >= row.left) continue;
                    P q;
#pragma unroll
                    for (int i = 0; i < N; ++i) q.e[i] = e[k * N + i] * to_map;
                    if (ALIGNED || (whole && (k > 0 || row.first >= 0) && k * kStep + N <= row.left)) {
                        st<T, N>(g + k * kStep, q);
                    } else {
#pragma unroll
                        for (int i = 0; i < N; ++i)
                            if (row.first + k * kStep + i >= 0 && k * kStep + i < row.left) g[k * kStep + i] = q.e[i];
                    }
                }
                if (mine_t) g[tt] = (et * to_p - (T)1) * inv_n;   // over what the thread has just written there
            }
        }
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) t_of[d] = t_of[d + 1];
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
        T m = lowest<T>(), sum = (T)0;   // the sum relative to this thread's maximum so far
        for (size_t k = threadIdx.x; k < packs; k += THREADS) {
            const P q = ld<T, N>(x + k * N);
            T top = m;
#pragma unroll
            for (int j = 0; j < N; ++j) top = max_(top, q.e[j]);
            if (top > m) {
                sum = m == lowest<T>() ? sum : sum * exp_(m - top);
                m = top;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) sum += q.e[j] == lowest<T>() ? (T)0 : exp_(q.e[j] - m);
        }
        const T warp_top = warp_max(m);
        sum = m == lowest<T>() ? sum : sum * exp_(m - warp_top);
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) pairs[warp] = Lse<T>{warp_top, sum};
        __syncthreads();
        m = pairs[0].c;
        for (int w = 1; w < kWarps; ++w) m = max_(m, pairs[w].c);
        sum = (T)0;
        for (int w = 0; w < kWarps; ++w) sum += pairs[w].c == lowest<T>() ? pairs[w].s : pairs[w].s * exp_(pairs[w].c - m);
        const bool bad = (uint64_t)t >= p.classes;
        if (threadIdx.x == 0) {
            mine.loss += bad ? (double)NAN : (double)log_(sum) - ((double)x[t] - (double)m);
            mine.rows += 1;
        }
        __syncthreads();   // the pairs are written again for the next row, x[t] may be overwritten below
        if (g) {
            const T inv_s = bad ? nan_<T>() : (T)1 / sum;
            for (size_t k = threadIdx.x; k < packs; k += THREADS) {
                P q = ld<T, N>(x + k * N);
#pragma unroll
                for (int j = 0; j < N; ++j) q.e[j] = (exp_(q.e[j] - m) * inv_s - (k * N + j == (size_t)t ? (T)1 : (T)0)) * inv_n;
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

template <typename T, int THREADS, int NV, int AHEAD, bool ALIGNED> int run_rows(Ctx *ctx, XentArgs<T> &p) {
    constexpr auto kernel = xent_cta_kernel<T, THREADS, NV, AHEAD, ALIGNED>;
    constexpr size_t smem = (size_t)AHEAD * THREADS * NV * 16;
    // as many clusters as run at once (a CTA of 1024 threads fills an SM, eight of 128 do), the rows dealt out among them
    unsigned fit = 0;
    if (int rc = clusters_at_once<XentArgs<T>, kernel>(ctx, THREADS, p.cluster, smem, &fit)) return rc;
    const size_t clusters = std::max<size_t>(1, std::min<size_t>(p.rows, fit));
    return run<T, kernel>(ctx, "xent_cta_kernel", p, clusters * p.cluster, THREADS, smem);
}
// Rows that need six vectors of a thread at most leave room to copy two rows ahead.
template <typename T, int THREADS> int run_cta(Ctx *ctx, XentArgs<T> &p, unsigned cluster, bool vec, size_t room) {
    p.cluster = cluster;
    if (room <= (size_t)cluster * THREADS * 6 * 16)
        return vec ? run_rows<T, THREADS, 6, 2, true>(ctx, p) : run_rows<T, THREADS, 6, 2, false>(ctx, p);
    return vec ? run_rows<T, THREADS, 8, 1, true>(ctx, p) : run_rows<T, THREADS, 8, 1, false>(ctx, p);
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
    const size_t room = bytes + (vec ? 0 : 16);   // a row that starts inside a vector takes one more
    if (room <= 64 * 128) return run_cta<T, 64>(ctx, p, 1, vec, room);
    if (room <= 128 * 128) return run_cta<T, 128>(ctx, p, 1, vec, room);
    if (room <= 256 * 128) return run_cta<T, 256>(ctx, p, 1, vec, room);
    if (room <= 512 * 128) return run_cta<T, 512>(ctx, p, 1, vec, room);
    for (unsigned cluster = 1; cluster <= kMaxCluster; ++cluster)
        if (room <= (size_t)cluster * 1024 * 128) return run_cta<T, 1024>(ctx, p, cluster, vec, room);
    const size_t grid = std::max<size_t>(1, std::min<size_t>(p.rows, (size_t)ctx->sm_count * 4));
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
    return guarded([&]() -> int {
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
    });
}
