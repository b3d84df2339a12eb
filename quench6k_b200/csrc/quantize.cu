// Rows in 8 bits: with a = max |x[r, :]| and u = (1 / a) * 127 the entries are q = rint(x u), whole numbers from -127 to 127 (ties
// to even), and an entry stands for q * scale with scale = a * (1 / 127).  Each quotient and product is rounded to FP32 once, so
// that q and scale are the same wherever they are computed.
//
// A row of zeros, or one so small that u is infinite (a < 3.8e-37), gets zeros and the scale 0; a row with a value that
// is not finite gets zeros and the scale NaN, so that every product with it is NaN.
#include "common.cuh"

namespace {

// One pass over the rows: a row stays in registers between its largest value and its entries.

// |x| as an unsigned number: ascends with |x|, and what is not finite lies at 0x7f800000 and above.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// N neighbouring values at p as they are stored; N > 1: 16 bytes at once.
template <typename T, int N>
struct Piece {
    T v[N];
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

// TPR threads of a block of 256 share a row and hold NP pieces of N values each; longer rows are read a second time.
template <typename T, int N, int TPR, int NP>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* x, long long ldx, int R, int K, int8_t* q, float* scale) {
    pdl_enter();
    __shared__ unsigned most_of_warp[8];
    const int r = blockIdx.x * (256 / TPR) + threadIdx.x / TPR, at = threadIdx.x % TPR * N;
    const bool live = r < R;
    const T* row = x + (long long)(live ? r : 0) * ldx;
    Piece<T, N> held[NP];
    unsigned most = 0;
    for (int k0 = 0; k0 < K; k0 += TPR * N * NP) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (k0 + i * TPR * N + at < K) held[i].load(row + k0 + i * TPR * N + at);
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (k0 + i * TPR * N + at < K) most = max(most, held[i].most());
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (TPR > 32) {
        if ((threadIdx.x & 31) == 0) most_of_warp[threadIdx.x >> 5] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) most = max(most, most_of_warp[w]);
    }
    if (!live) return;
    const bool finite = most < 0x7f800000u;
    const float a = __uint_as_float(most), up = 1.0f / a * 127.0f;
    const bool zero = !finite || abs_bits(up) >= 0x7f800000u;
    const float u = zero ? 0.0f : up;
    if (at == 0) scale[r] = !finite ? __uint_as_float(0x7fffffffu) : zero ? 0.0f : a * (1.0f / 127.0f);
    int8_t* out = q + (long long)r * K;
    const bool again = K > TPR * N * NP;
    for (int k0 = 0; k0 < K; k0 += TPR * N * NP) {
        if (again) {
#pragma unroll
            for (int i = 0; i < NP; ++i)
                if (k0 + i * TPR * N + at < K) held[i].load(row + k0 + i * TPR * N + at);
        }
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (k0 + i * TPR * N + at < K) held[i].store(out + k0 + i * TPR * N + at, u);
    }
}

// Short rows: a warp each; others: a block each, which holds rows of up to 16 KB (in single values, where they do not start on 16 bytes, of 8,192 values).
template <typename T, int N>
void launch(const T* x, long long ldx, int R, int K, int8_t* q, float* scale, cudaStream_t st) {
    constexpr int SHORT = N == 1 ? 16 : 4, MID = N == 1 ? 8 : 2, LONG = N == 1 ? 32 : 4;
    if (K <= 32 * N * SHORT) q6k_launch(quantize_rows_kernel<T, N, 32, SHORT>, (R + 7) / 8, 256, 0, st, x, ldx, R, K, q, scale);
    else if (K <= 256 * N * MID) q6k_launch(quantize_rows_kernel<T, N, 256, MID>, R, 256, 0, st, x, ldx, R, K, q, scale);
    else q6k_launch(quantize_rows_kernel<T, N, 256, LONG>, R, 256, 0, st, x, ldx, R, K, q, scale);
}

}  // namespace

// x: [R, K] of dtype code (FP32 or bfloat16), row pitch ldx elements; q: int8 [R, K]; scale: FP32 [R].
Q6K_API int q6k_quantize_rows(const void* x, long long ldx, int R, int K, int dtype, void* q, float* scale, cudaStream_t st) {
    if (R == 0) return 0;
    Q6K_REQUIRE(R > 0 && K > 0 && ldx >= K, "quantize_rows: %d rows of %d with a pitch of %lld", R, K, ldx);
    Q6K_DISPATCH(dtype, {
        constexpr int N = 16 / sizeof(T);
        if (K % N == 0 && ldx % N == 0 && (((uintptr_t)x | (uintptr_t)q) & 15) == 0) launch<T, N>((const T*)x, ldx, R, K, (int8_t*)q, scale, st);
        else launch<T, 1>((const T*)x, ldx, R, K, (int8_t*)q, scale, st);
    });
    return q6k_check_launch("quantize_rows");
}
