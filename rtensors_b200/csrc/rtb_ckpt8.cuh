// 8-bit activation checkpoints: the format, shared by the kernels that write and read it.
//
// kCkpt8Block consecutive elements share one magnitude m = max |x| (in the tensor's own type); an element is
// the code c = round(127 x / m), the quotient rounded to nearest in real arithmetic, ties to even.  It stands for
// c m / 127, half a step (m / 254) from x at most; +-m, 0 and therefore a mask of zeros and ones are exact.
// A block that holds an infinity or a NaN has magnitude NaN and stands for NaN as a whole.
#pragma once
#include <cstdint>

namespace rtb {

constexpr int kCkpt8Shift = 7;
constexpr int kCkpt8Block = 1 << kCkpt8Shift;   // one warp, four elements per lane

#ifdef __CUDACC__
__device__ __forceinline__ float ckpt8_fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double ckpt8_fma(double a, double b, double c) { return fma(a, b, c); }

// m / 127 as an unevaluated sum hi + lo: c hi + c lo rounds to c m / 127 to within half an ulp and a little (a
// single rounded m / 127 would put up to 127 / 2 ulp on m itself).  Tiny magnitudes are scaled up and
// the result scaled back, so that hi and lo are no subnormals.
template <typename T> struct Ckpt8Scale {
    T hi, lo;
    bool small;
    __device__ __forceinline__ explicit Ckpt8Scale(T m) {
        const T up = sizeof(T) == 4 ? (T)18446744073709551616.0 : (T)1.3407807929942597e154;      // 2^64, 2^512
        small = m < (sizeof(T) == 4 ? (T)1e-30f : (T)1e-280);
        if (small) m = m * up;
        const T r127 = (T)(1.0 / 127.0);
        hi = m * r127;
        lo = ckpt8_fma((T)-127, hi, m) * r127;   // the residual itself is exact
    }
    __device__ __forceinline__ T restore(int8_t code) const { return down(times((T)code)); }
    // the first N of four packed codes.  A byte becomes the lowest mantissa byte of 2^23 (2^52): two instructions where a
    // conversion from 8 bits runs at an eighth of the rate.
    template <int N> __device__ __forceinline__ void restore(uint32_t four, T *out) const {
        four ^= 0x80808080u;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if constexpr (sizeof(T) == 4) out[k] = times(__uint_as_float(__byte_perm(four, 0x4b000000u, 0x7540u + k)) - 8388736.0f);
            else out[k] = times(__hiloint2double(0x43300000, (int)__byte_perm(four, 0u, 0x4440u + k)) - 4503599627370624.0);
        }
        if (small) {
#pragma unroll
            for (int k = 0; k < N; ++k) out[k] = down(out[k]);
        }
    }

  private:
    __device__ __forceinline__ T times(T c) const { return ckpt8_fma(c, hi, c * lo); }
    __device__ __forceinline__ T down(T v) const {
        return small ? v * (sizeof(T) == 4 ? (T)5.421010862427522e-20 : (T)7.458340731200207e-155) : v;   // 2^-64, 2^-512
    }
};
#endif

}  // namespace rtb
