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
    alignas(N * sizeof(T)) T v[N];
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
        if constexpr (sizeof(T) == 2 && N > 1) {                               // two values to an instruction: their upper halves are all there is
            const unsigned* w = (const unsigned*)v;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
            return max(m & 0xffff0000u, m << 16);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) m = max(m, abs_bits(to_f32(v[i])));
            return m;
        }
    }
    // up = 0: zeros, whatever the values are.  A product below 2^22 plus 1.5 x 2^23 is rounded to a whole number, ties to even, whose lowest byte is the
    // entry: an addition for each value and three byte selections for four, where conversions run at a quarter of the rate (8,192 rows of 8,192: 37 us
    // with them, 31 without).
    __device__ __forceinline__ void store(int8_t* q, float up) const {
        unsigned w[(N + 3) / 4] = {};
        if (up != 0.0f) {
            unsigned b[N];
#pragma unroll
            for (int i = 0; i < N; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(to_f32(v[i]), up), 12582912.0f));
            if constexpr (N == 1) w[0] = b[0];
            else {
#pragma unroll
                for (int i = 0; i < N; i += 4) w[i / 4] = __byte_perm(__byte_perm(b[i], b[i + 1], 0x0040), __byte_perm(b[i + 2], b[i + 3], 0x0040), 0x5410);
            }
        }
        if constexpr (N == 1) *q = (int8_t)w[0];
        else if constexpr (N == 4) *(unsigned*)q = w[0];
        else *(uint2*)q = make_uint2(w[0], w[1]);
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
