// 8-bit activation checkpoints (format: rtb_ckpt8.cuh): store, restore, and the backward maps of the tape's nodes
// fed from codes, so that the restored tensor never exists in memory.  All HBM-bound: f32 moves 5 bytes per
// element to store or restore, 9 to apply a map.  A warp holds a block (four elements a lane), several blocks at a time so that
// their loads are in flight together; a block's magnitude is one warp-wide maximum of bit patterns.  67M f32: store 53 us
// (6.4 TB/s), restore 52 us (6.4), a map 90 us (6.7); 34M f64: 48, 48 and 86 us.
#include "rtb_internal.h"
#include "rtb_ckpt8.cuh"

namespace rtb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;   // blocks of a warp, loads of all in flight at once

// The store's chain from load over maximum and reciprocal to code is long, so warps in flight count for more than registers:
// blocks of a warp, CTAs of an SM.  67M f32: 54 us at 7 or 8 CTAs, 58 at 6, 64 as the compiler chooses; 34M f64: 49 at 8, 51 at 6.
// At 7 CTAs ptxas takes 32 registers and spills some 100 bytes a thread.
template <typename T> struct StoreShape;
template <> struct StoreShape<float> { static constexpr int unroll = 4, ctas = 7; };
template <> struct StoreShape<double> { static constexpr int unroll = 2, ctas = 8; };

// max |x| of a block.  A NaN wins (max.NaN), and as bits NaN > inf > every finite magnitude, so one comparison tells.
template <typename T> struct Bits;
template <> struct Bits<float> {
    using U = uint32_t;
    static constexpr U inf = 0x7f800000u;
    static __device__ __forceinline__ float top(float a, float b) {
        float m;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)));
        return m;
    }
    static __device__ __forceinline__ U bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
    static __device__ __forceinline__ float value(U u) { return __uint_as_float(u); }
    static __device__ __forceinline__ U warp_max(U u) { return __reduce_max_sync(0xffffffffu, u); }
};
template <> struct Bits<double> {
    using U = unsigned long long;
    static constexpr U inf = 0x7ff0000000000000ull;
    static __device__ __forceinline__ double top(double a, double b) {
        const U u = max(bits(a), bits(b));
        return __longlong_as_double((long long)u);
    }
    static __device__ __forceinline__ U bits(double x) { return (U)__double_as_longlong(x) & 0x7fffffffffffffffull; }
    static __device__ __forceinline__ double value(U u) { return __longlong_as_double((long long)u); }
    static __device__ __forceinline__ U warp_max(U u) {   // the high words' maximum, then the low words' among the lanes that hold it
        const uint32_t hi = (uint32_t)(u >> 32), top_hi = __reduce_max_sync(0xffffffffu, hi);
        const uint32_t top_lo = __reduce_max_sync(0xffffffffu, hi == top_hi ? (uint32_t)u : 0u);
        return ((U)top_hi << 32) | top_lo;
    }
};

// round(127 x / m), ties to even, exactly.  f32: the quotient in 64 bits decides every case (127 x is exact there, and
// a quotient that is no tie is at least 2^-33 of itself away from one).  x times an approximate 127 / m is off by less
// than 1e-4 and decides all but the values that near to a tie; adding 1.5 2^23 rounds it and leaves the code in the low byte.
struct Quantise32 {
    float m, inv;
    bool wide;
    __device__ __forceinline__ explicit Quantise32(float mag) : m(mag), wide(!(mag > 1e-30f && mag < 1e37f)) {
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(mag));
        inv *= 127.0f;
    }
    // four codes, packed
    __device__ __forceinline__ uint32_t codes(const float x[4]) const {
        const float magic = 12582912.0f;
        uint32_t c[4];
        float off = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float t = fmaf(x[k], inv, magic);
            c[k] = __float_as_uint(t);
            off = fmaxf(off, fabsf(fmaf(x[k], inv, magic - t)));
        }
        if (wide || off > 0.4998f) {
#pragma unroll
            for (int k = 0; k < 4; ++k) c[k] = m > 0.0f ? (uint32_t)(int)rint(127.0 * (double)x[k] / (double)m) : 0u;
        }
        return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    }
};
// f64: the product with a reciprocal decides all but the values within 1e-8 of a tie.  An approximate reciprocal within 2^-18, refined
// once by Newton's step, is within 2^-36, and 127 times that is below 2e-9.  What is left is decided by the sign of
// 254 |x| - (2 n + 1) m for the whole number n below the quotient: both products as exact sums of two numbers, compared part by part.
// Such a decision is made for all four values of a lane, and its warp waits: 34M values of 0, 1/2 and 1, a third of
// them ties, 240 us instead of 48 (the f32 division: 67M 429 us instead of 53).
struct Quantise64 {
    double m, inv, scale;
    bool wide;
    __device__ __forceinline__ explicit Quantise64(double mag) : m(mag), scale(1.0), wide(!(mag > 1e-280 && mag < 1e300)) {
        double r;
        asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(r) : "d"(mag));
        inv = 127.0 * fma(r, fma(-mag, r, 1.0), r);
        if (wide) scale = mag > 1.0 ? 0x1p-20 : 0x1p512, m = mag * scale;   // the products stay finite, their lower parts normal
    }
    __device__ __forceinline__ uint32_t exact(double x) const {
        const double s = fabs(x) * scale, n = floor(127.0 * s / m), odd = 2.0 * n + 1.0;
        const double left = 254.0 * s, right = odd * m;
        const double d = (left - right) + (fma(254.0, s, -left) - fma(odd, m, -right));
        const int c = (int)n + (d > 0.0 || (d == 0.0 && ((int)n & 1)) ? 1 : 0);
        return (uint32_t)(x < 0.0 ? -c : c);
    }
    __device__ __forceinline__ uint32_t codes(const double x[4]) const {
        const double magic = 6755399441055744.0;   // 1.5 2^52
        uint32_t c[4];
        double off = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double t = fma(x[k], inv, magic);
            c[k] = (uint32_t)__double2loint(t);
            off = fmax(off, fabs(fma(x[k], inv, magic - t)));
        }
        if (wide || off > 0.49999999) {
#pragma unroll
            for (int k = 0; k < 4; ++k) c[k] = m > 0.0 ? exact(x[k]) : 0u;
        }
        return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    }
};
template <typename T> struct QuantiseOf;
template <> struct QuantiseOf<float> { using type = Quantise32; };
template <> struct QuantiseOf<double> { using type = Quantise64; };

// Lane l holds elements 4 l .. 4 l + 3 of its block: one access of 16 bytes, in f64 of 32 (two of 16 would each touch every line of
// the block's kilobyte).
__device__ __forceinline__ void vector4(const float *p, float v[4]) {
    const float4 q = *reinterpret_cast<const float4 *>(p);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
}
__device__ __forceinline__ void vector4(const double *p, double v[4]) {
    asm volatile("ld.global.v4.f64 {%0, %1, %2, %3}, [%4];" : "=d"(v[0]), "=d"(v[1]), "=d"(v[2]), "=d"(v[3]) : "l"(p) : "memory");
}
__device__ __forceinline__ void put_vector4(float *p, const float v[4]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void put_vector4(double *p, const double v[4]) {
    asm volatile("st.global.v4.f64 [%0], {%1, %2, %3, %4};" ::"l"(p), "d"(v[0]), "d"(v[1]), "d"(v[2]), "d"(v[3]) : "memory");
}
template <typename T, bool VEC> __device__ __forceinline__ void load4(const T *p, size_t i, size_t n, T v[4]) {
    if (VEC && i + 4 <= n) {
        vector4(p + i, v);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = i + k < n ? p[i + k] : (T)0;
    }
}
template <typename T, bool VEC> __device__ __forceinline__ void store4(T *p, size_t i, size_t n, const T v[4]) {
    if (VEC && i + 4 <= n) {
        put_vector4(p + i, v);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) p[i + k] = v[k];
    }
}

__device__ __forceinline__ uint32_t load_codes(const int8_t *p, size_t i, size_t n) {
    if (i + 4 <= n) return *reinterpret_cast<const uint32_t *>(p + i);
    uint32_t c = 0;
    for (int k = 0; k < 3; ++k)
        if (i + k < n) c |= (uint32_t)(uint8_t)p[i + k] << (8 * k);
    return c;
}
__device__ __forceinline__ void store_codes(int8_t *p, size_t i, size_t n, uint32_t c) {
    if (i + 4 <= n) {
        *reinterpret_cast<uint32_t *>(p + i) = c;
        return;
    }
    for (int k = 0; k < 3; ++k)
        if (i + k < n) p[i + k] = (int8_t)(c >> (8 * k));
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, StoreShape<T>::ctas) ckpt8_store_kernel(const T *src, size_t n, int8_t *codes, T *mags) {
    constexpr int U = StoreShape<T>::unroll;
    const int lane = threadIdx.x & 31;
    const size_t block0 = ((size_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * U;
    grid_dep_sync();
    T v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) load4<T, VEC>(src, (block0 + u) * kCkpt8Block + lane * 4, n, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        using B = Bits<T>;
        const size_t i = (block0 + u) * kCkpt8Block + lane * 4;
        const typename B::U top = B::warp_max(B::bits(B::top(B::top(v[u][0], v[u][1]), B::top(v[u][2], v[u][3]))));
        if ((block0 + u) * kCkpt8Block >= n) continue;   // the same in the whole warp
        uint32_t c = 0;
        T m = B::value(top);
        if (top >= B::inf) {
            m = B::value(B::inf | 1u);   // some NaN
        } else {
            c = typename QuantiseOf<T>::type(m).codes(v[u]);
        }
        store_codes(codes, i, n, c);
        if (lane == 0) mags[block0 + u] = m;
    }
}

// KIND < 0: restore only
template <typename T, int KIND> __device__ __forceinline__ T map(T r, T up) {
    if constexpr (KIND == RTB_CKPT8_MUL) return r * up;
    if constexpr (KIND == RTB_CKPT8_SIGMOID) return r * ((T)1 - r) * up;
    if constexpr (KIND == RTB_CKPT8_TANH) return ((T)1 - r * r) * up;
    if constexpr (KIND == RTB_CKPT8_SQUARE) return (T)2 * r * up;
    return r;
}

template <typename T, int KIND, bool VEC>
__global__ void __launch_bounds__(kThreads) ckpt8_read_kernel(const int8_t *codes, const T *mags, const T *up, size_t n, T *dst) {
    const int lane = threadIdx.x & 31;
    const size_t block0 = ((size_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * kUnroll;
    grid_dep_sync();
    uint32_t c[kUnroll];
    T w[kUnroll][4], m[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const size_t i = (block0 + u) * kCkpt8Block + lane * 4;
        c[u] = load_codes(codes, i, n);
        if (KIND >= 0) load4<T, VEC>(up, i, n, w[u]);
        m[u] = (block0 + u) * kCkpt8Block < n ? mags[block0 + u] : (T)0;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const size_t i = (block0 + u) * kCkpt8Block + lane * 4;
        const Ckpt8Scale<T> scale(m[u]);
        T out[4];
        scale.template restore<4>(c[u], out);
#pragma unroll
        for (int k = 0; k < 4; ++k) out[k] = map<T, KIND>(out[k], KIND >= 0 ? w[u][k] : (T)0);
        store4<T, VEC>(dst, i, n, out);
    }
}

int tiles(size_t n, int unroll, unsigned *grid) {
    const size_t blocks = (n + kCkpt8Block - 1) / kCkpt8Block, tile = (size_t)kWarps * unroll, g = (blocks + tile - 1) / tile;
    if (g > 0x7fffffffu) return fail(RTB_ERR_TOO_LARGE, "checkpoint of %zu elements is beyond one launch", n);
    *grid = (unsigned)g;
    return RTB_OK;
}

template <typename T> bool aligned4(const T *p) { return ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0; }

template <typename T> int store_typed(Ctx *ctx, const T *src, size_t n, int8_t *codes, T *mags) {
    unsigned grid = 0;
    if (int rc = tiles(n, StoreShape<T>::unroll, &grid)) return rc;
    if (aligned4(src)) launch_dep(ctx, grid, kThreads, ckpt8_store_kernel<T, true>, src, n, codes, mags);
    else launch_dep(ctx, grid, kThreads, ckpt8_store_kernel<T, false>, src, n, codes, mags);
    return check_launch(ctx, "ckpt8_store_kernel");
}

template <typename T, int KIND> int read_typed(Ctx *ctx, const int8_t *codes, const T *mags, const T *up, size_t n, T *dst) {
    unsigned grid = 0;
    if (int rc = tiles(n, kUnroll, &grid)) return rc;
    if (aligned4(up) && aligned4(dst)) launch_dep(ctx, grid, kThreads, ckpt8_read_kernel<T, KIND, true>, codes, mags, up, n, dst);
    else launch_dep(ctx, grid, kThreads, ckpt8_read_kernel<T, KIND, false>, codes, mags, up, n, dst);
    return check_launch(ctx, "ckpt8_read_kernel");
}

template <typename T> int read_kind(Ctx *ctx, int kind, const int8_t *codes, const T *mags, const T *up, size_t n, T *dst) {
    switch (kind) {
        case -1: return read_typed<T, -1>(ctx, codes, mags, up, n, dst);
        case RTB_CKPT8_MUL: return read_typed<T, RTB_CKPT8_MUL>(ctx, codes, mags, up, n, dst);
        case RTB_CKPT8_SIGMOID: return read_typed<T, RTB_CKPT8_SIGMOID>(ctx, codes, mags, up, n, dst);
        case RTB_CKPT8_TANH: return read_typed<T, RTB_CKPT8_TANH>(ctx, codes, mags, up, n, dst);
        case RTB_CKPT8_SQUARE: return read_typed<T, RTB_CKPT8_SQUARE>(ctx, codes, mags, up, n, dst);
    }
    return fail(RTB_ERR_INVALID, "unknown checkpoint map %d", kind);
}

int check_ckpt(rtb_ctx *c, int dtype) {
    if (!c) return fail(RTB_ERR_INVALID, "null ctx");
    if (dtype != RTB_F32 && dtype != RTB_F64) return fail(RTB_ERR_DTYPE, "checkpoints are defined for f32 and f64 only");
    return RTB_OK;
}

int read_any(rtb_ctx *c, int dtype, int kind, const int8_t *codes, const void *mags, const void *up, size_t n, void *dst) {
    if (n == 0) return RTB_OK;
    if (!codes || !mags || !dst || (kind >= 0 && !up)) return fail(RTB_ERR_INVALID, "null argument");
    if ((uintptr_t)codes & 3u) return fail(RTB_ERR_INVALID, "the codes must be 4-byte aligned");
    Ctx *ctx = reinterpret_cast<Ctx *>(c);
    if (int rc = use_device(ctx)) return rc;
    return dtype == RTB_F32 ? read_kind<float>(ctx, kind, codes, (const float *)mags, (const float *)up, n, (float *)dst)
                            : read_kind<double>(ctx, kind, codes, (const double *)mags, (const double *)up, n, (double *)dst);
}

}  // namespace
}  // namespace rtb

using namespace rtb;

RTB_API int rtb_ckpt8_store(rtb_ctx *c, int dtype, const void *src, size_t n, int8_t *codes, void *mags) {
    return guarded([&]() -> int {
        if (int rc = check_ckpt(c, dtype)) return rc;
        if (n == 0) return RTB_OK;
        if (!src || !codes || !mags) return fail(RTB_ERR_INVALID, "null argument");
        if ((uintptr_t)codes & 3u) return fail(RTB_ERR_INVALID, "the codes must be 4-byte aligned");
        Ctx *ctx = reinterpret_cast<Ctx *>(c);
        if (int rc = use_device(ctx)) return rc;
        return dtype == RTB_F32 ? store_typed<float>(ctx, (const float *)src, n, codes, (float *)mags)
                                : store_typed<double>(ctx, (const double *)src, n, codes, (double *)mags);
    });
}

RTB_API int rtb_ckpt8_restore(rtb_ctx *c, int dtype, const int8_t *codes, const void *mags, size_t n, void *dst) {
    return guarded([&]() -> int {
        if (int rc = check_ckpt(c, dtype)) return rc;
        return read_any(c, dtype, -1, codes, mags, nullptr, n, dst);
    });
}

RTB_API int rtb_ckpt8_grad(rtb_ctx *c, int dtype, int kind, const int8_t *codes, const void *mags, const void *up, size_t n, void *dst) {
    return guarded([&]() -> int {
        if (int rc = check_ckpt(c, dtype)) return rc;
        if (kind < RTB_CKPT8_MUL || kind > RTB_CKPT8_SQUARE) return fail(RTB_ERR_INVALID, "unknown checkpoint map %d", kind);
        return read_any(c, dtype, kind, codes, mags, up, n, dst);
    });
}
