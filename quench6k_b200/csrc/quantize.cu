// Rows in 8 bits: with a = max |x[r, :]| and u = (1 / a) * 127 the entries are q = rint(x u), whole numbers from -127 to 127 (ties
// to even), and an entry stands for q * scale with scale = a * (1 / 127).  Each quotient and product is rounded to FP32 once, so
// that q and scale are the same wherever they are computed.
//
// A row of zeros, or one so small that u is infinite (a < 3.8e-37), gets zeros and the scale 0; a row with a value that
// is not finite gets zeros and the scale NaN, so that every product with it is NaN.
#include "common.cuh"

namespace {

// |x| as an unsigned number: ascends with |x|, and what is not finite lies at 0x7f800000 and above.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* x, long long ldx, int K, int8_t* q, float* scale) {
    pdl_enter();
    __shared__ unsigned most_of_warp[8];
    const T* row = x + (long long)blockIdx.x * ldx;
    int8_t* out = q + (long long)blockIdx.x * K;
    unsigned most = 0;
    for (int k = threadIdx.x; k < K; k += 256) most = max(most, abs_bits(to_f32(row[k])));
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0) most_of_warp[threadIdx.x >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) most = max(most, most_of_warp[w]);
    const float a = __uint_as_float(most);
    const bool finite = most < 0x7f800000u;
    const float u = 1.0f / a * 127.0f;
    const bool zero = !finite || abs_bits(u) >= 0x7f800000u;
    if (threadIdx.x == 0) scale[blockIdx.x] = !finite ? __uint_as_float(0x7fffffffu) : zero ? 0.0f : a * (1.0f / 127.0f);
    for (int k = threadIdx.x; k < K; k += 256) out[k] = zero ? (int8_t)0 : (int8_t)__float2int_rn(to_f32(row[k]) * u);
}

}  // namespace

// x: [R, K] of dtype code (FP32 or bfloat16), row pitch ldx elements; q: int8 [R, K]; scale: FP32 [R].
Q6K_API int q6k_quantize_rows(const void* x, long long ldx, int R, int K, int dtype, void* q, float* scale, cudaStream_t st) {
    if (R == 0) return 0;
    Q6K_REQUIRE(R > 0 && K > 0 && ldx >= K, "quantize_rows: %d rows of %d with a pitch of %lld", R, K, ldx);
    Q6K_DISPATCH(dtype, { q6k_launch(quantize_rows_kernel<T>, R, 256, 0, st, (const T*)x, ldx, K, (int8_t*)q, scale); });
    return q6k_check_launch("quantize_rows");
}
