// Rows in 8 bits: with a = max |x[r, :]| and u = (1 / a) * 127 the entries are q = rint(x u), whole numbers from -127 to 127 (ties
// to even), and an entry stands for q * scale with scale = a * (1 / 127).  Each quotient and product is rounded to FP32 once, so
// that q and scale are the same wherever they are computed.
//
// A row of zeros, or one so small that u is infinite (a < 3.8e-37), gets zeros and the scale 0; a row with a value that
// is not finite gets zeros and the scale NaN, so that every product with it is NaN.
#pragma once
#include "common.cuh"

namespace {

// |x| as an unsigned number: ascends with |x|, and what is not finite lies at 0x7f800000 and above.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// N neighbouring values at p as they are stored; N > 1: 16 bytes at once.
template <typename T, int N>
struct Piece {
    T v[N];
    __device__ __forceinline__ void take(const uint4& bytes) {
        static_assert(N * sizeof(T) == 16, "16 bytes");
        *(uint4*)v = bytes;
    }
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (N * sizeof(T) == 16) *(uint4*)v = *(const uint4*)p;
        else v[0] = *p;
    }
    __device__ __forceinline__ unsigned most() const {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) m = max(m, abs_bits(to_f32(v[i])));
        return m;
    }
    __device__ __forceinline__ void store(int8_t* q, float u) const {          // u = 0: zeros, whatever the values are
        union { int8_t b[N]; unsigned w[(N + 3) / 4]; } o;
#pragma unroll
        for (int i = 0; i < N; ++i) o.b[i] = u == 0.0f ? (int8_t)0 : (int8_t)__float2int_rn(to_f32(v[i]) * u);
        if constexpr (N == 1) *q = o.b[0];
        else if constexpr (N == 4) *(unsigned*)q = o.w[0];
        else *(uint2*)q = make_uint2(o.w[0], o.w[1]);
    }
};

// What a row's entries are multiplied with (0: they are zeros, whatever the values are) and the row's scale, from the largest abs_bits of its values.
struct RowScale {
    float up, scale;
};
__device__ __forceinline__ RowScale row_scale(unsigned most) {
    const bool finite = most < 0x7f800000u;
    const float a = __uint_as_float(most), up = 1.0f / a * 127.0f;
    const bool zero = !finite || abs_bits(up) >= 0x7f800000u;
    return {zero ? 0.0f : up, !finite ? __uint_as_float(0x7fffffffu) : zero ? 0.0f : a * (1.0f / 127.0f)};
}

}  // namespace
