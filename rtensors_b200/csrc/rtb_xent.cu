// Softmax cross-entropy of (rows, classes) logits against one class per row, with its gradient map:
//
//   loss = sum_r [ log sum_j exp(x_rj - m_r) - (x_rt - m_r) ]  [ / count ],   m_r = max_j x_rj
//   map_rj = (exp(x_rj - m_r) / sum_r - [j = t_r])  [ / count ]
//
// One pass over a row keeps the running maximum and the sum rescaled to it; a second pass writes the map.  The second read
// of a row comes from the caches.  HBM-bound: 4 bytes read and 4 written per element in f32.
//
// A row with t < 0 does not count (padding): its map is zero.  t >= classes gives NaN for the row and the loss.
// Rows are dealt to CTAs statically and every sum has a fixed order: results are deterministic.
#include <algorithm>

#include "rtb_internal.h"

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

// The running (maximum, sum of exp(x - maximum)).  Entries of -inf add nothing and keep a maximum of -inf harmless; a NaN
// is skipped by the maximum and kept by the sum.
template <typename T> struct Lse {
    T m, s;
    __device__ __forceinline__ void merge(T m2, T s2) {
        const T top = max_(m, m2);
        const T a = m == lowest<T>() ? (T)1 : exp_(m - top), b = m2 == lowest<T>() ? (T)1 : exp_(m2 - top);
        s = s * a + s2 * b;
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

// TPR threads share a row (32: a warp, else the whole CTA)
template <typename T, int THREADS, int TPR, bool VEC>
__global__ void __launch_bounds__(THREADS) xent_kernel(const T *logits, size_t rows, size_t classes, int64_t pitch, const int64_t *targets,
                                                       int mean, const unsigned long long *counts, T *loss, T *map, XentPartial *partials,
                                                       unsigned *done_counter) {
    constexpr int N = VEC ? Vec<T>::N : 1;
    constexpr int G = THREADS / TPR;   // rows at a time
    __shared__ T sm[32], ss[32];
    __shared__ XentPartial sp[32];
    __shared__ T s_inv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int in_row = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    grid_dep_sync();
    if (map && mean) {
        if (warp == 0) {
            unsigned long long n = counts[lane] + counts[lane + 32];
#pragma unroll
            for (int d = 16; d; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
            if (lane == 0) s_inv = (T)1 / (T)n;
        }
        __syncthreads();
    }
    const T inv_n = map && mean ? s_inv : (T)1;
    XentPartial mine{0.0, 0};
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < rows; r0 += (size_t)gridDim.x * G) {
        const size_t r = r0 + slot;
        const bool have = r < rows;   // the same in all threads of a row
        const int64_t t = have ? targets[r] : -1;
        const T *x = logits + (have ? (int64_t)r * pitch : 0);
        T *g = map ? map + (have ? r * classes : 0) : nullptr;
        if (t < 0) {
            if (have && g)
                for (size_t j = in_row; j < classes; j += TPR) g[j] = (T)0;
            if (TPR == 32) continue;
            continue;   // TPR == THREADS: the whole CTA skips the row together
        }
        const size_t packs = classes / N;
        Lse<T> l{lowest<T>(), (T)0};
        for (size_t k = in_row; k < packs; k += TPR) {
            if constexpr (VEC) {
                const Vec<T> q = reinterpret_cast<const Vec<T> *>(x)[k];
                l.template add<N>(q.e);
            } else {
                l.template add<1>(x + k);
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            const T m2 = __shfl_xor_sync(0xffffffffu, l.m, d), s2 = __shfl_xor_sync(0xffffffffu, l.s, d);
            l.merge(m2, s2);
        }
        if (TPR > 32) {
            if (lane == 0) sm[warp] = l.m, ss[warp] = l.s;
            __syncthreads();
            l.m = sm[0], l.s = ss[0];
            for (int w = 1; w < TPR / 32; ++w) l.merge(sm[w], ss[w]);
        }
        const bool bad = (uint64_t)t >= classes;
        if (in_row == 0) {
            mine.loss += bad ? (double)NAN : (double)(log_(l.s) - (x[t] - l.m));
            mine.rows += 1;
        }
        if (g) {
            const T inv_s = bad ? nan_<T>() : (T)1 / l.s;
            for (size_t k = in_row; k < packs; k += TPR) {
                if constexpr (VEC) {
                    Vec<T> q = reinterpret_cast<const Vec<T> *>(x)[k];
#pragma unroll
                    for (int j = 0; j < N; ++j) q.e[j] = (exp_(q.e[j] - l.m) * inv_s - (k * N + j == (size_t)t ? (T)1 : (T)0)) * inv_n;
                    reinterpret_cast<Vec<T> *>(g)[k] = q;
                } else {
                    g[k] = (exp_(x[k] - l.m) * inv_s - (k == (size_t)t ? (T)1 : (T)0)) * inv_n;
                }
            }
        }
        if (TPR > 32) __syncthreads();   // sm / ss are written again for the next row
    }
    // one partial per CTA; the last CTA adds them in order
    if (in_row == 0) sp[slot] = mine;
    __syncthreads();
    __shared__ bool last;
    if (threadIdx.x == 0) {
        for (int k = 1; k < G; ++k) mine.loss += sp[k].loss, mine.rows += sp[k].rows;
        partials[blockIdx.x] = mine;
        __threadfence();
        last = atomicAdd(done_counter, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    XentPartial all{0.0, 0};
    for (unsigned k = threadIdx.x; k < gridDim.x; k += THREADS) {
        all.loss += __ldcg(&partials[k].loss);
        all.rows += __ldcg(&partials[k].rows);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        all.loss += __shfl_down_sync(0xffffffffu, all.loss, d);
        all.rows += __shfl_down_sync(0xffffffffu, all.rows, d);
    }
    if (lane == 0) sp[warp] = all;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < THREADS / 32; ++w) all.loss += sp[w].loss, all.rows += sp[w].rows;
        *loss = (T)(mean ? all.loss / (double)all.rows : all.loss);
        *done_counter = 0;   // ready for the next launch on this stream
    }
}

template <typename T, int THREADS, int TPR, bool VEC>
int run(Ctx *ctx, const T *logits, size_t rows, size_t classes, int64_t pitch, const int64_t *targets, int mean, T *loss, T *map) {
    constexpr size_t G = THREADS / TPR;
    const size_t want = std::max<size_t>(1, (rows + G - 1) / G);
    const unsigned grid = (unsigned)std::min<size_t>(want, (size_t)ctx->sm_count * (2048 / THREADS));
    void *ws = nullptr;
    if (int rc = workspace(ctx, 1024 + grid * sizeof(XentPartial), &ws)) return rc;
    unsigned long long *counts = (unsigned long long *)((char *)ws + kWsHeader);
    XentPartial *partials = (XentPartial *)((char *)ws + kWsHeader + 1024);
    if (map && mean) {
        launch_dep(ctx, kCountCtas, 256, xent_count_kernel, targets, rows, counts);
        if (int rc = check_launch(ctx, "xent_count_kernel")) return rc;
    }
    launch_dep(ctx, grid, THREADS, xent_kernel<T, THREADS, TPR, VEC>, logits, rows, classes, pitch, targets, mean,
               (const unsigned long long *)counts, loss, map, partials, (unsigned *)ws);
    return check_launch(ctx, "xent_kernel");
}

template <typename T>
int pick(Ctx *ctx, const T *logits, size_t rows, size_t classes, int64_t pitch, const int64_t *targets, int mean, T *loss, T *map) {
    constexpr int N = Vec<T>::N;
    std::lock_guard<std::mutex> lock(ctx->ws_mu);
    const bool vec = classes % N == 0 && pitch % N == 0 && (((uintptr_t)logits | (uintptr_t)map) & 15u) == 0;
    if (classes <= 1024)
        return vec ? run<T, 256, 32, true>(ctx, logits, rows, classes, pitch, targets, mean, loss, map)
                   : run<T, 256, 32, false>(ctx, logits, rows, classes, pitch, targets, mean, loss, map);
    return vec ? run<T, 512, 512, true>(ctx, logits, rows, classes, pitch, targets, mean, loss, map)
               : run<T, 512, 512, false>(ctx, logits, rows, classes, pitch, targets, mean, loss, map);
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
