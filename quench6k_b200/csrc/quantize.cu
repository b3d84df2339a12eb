// Rows in 8 bits (quantize.cuh says how).  One pass over the rows: a row stays in registers between its largest value and its
// entries.
#include "quantize.cuh"

namespace {

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
    const RowScale s = row_scale(most);
    if (at == 0) scale[r] = s.scale;
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
            if (k0 + i * TPR * N + at < K) held[i].store(out + k0 + i * TPR * N + at, s.up);
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
int q6k_quantize_rows_launch(const void* x, long long ldx, int R, int K, int dtype, void* q, float* scale, cudaStream_t st) {
    if (R == 0) return 0;
    Q6K_REQUIRE(R > 0 && K > 0 && ldx >= K, "quantize_rows: %d rows of %d with a pitch of %lld", R, K, ldx);
    Q6K_DISPATCH(dtype, {
        constexpr int N = 16 / sizeof(T);
        if (K % N == 0 && ldx % N == 0 && (((uintptr_t)x | (uintptr_t)q) & 15) == 0) launch<T, N>((const T*)x, ldx, R, K, (int8_t*)q, scale, st);
        else launch<T, 1>((const T*)x, ldx, R, K, (int8_t*)q, scale, st);
    });
    return q6k_check_launch("quantize_rows");
}

Q6K_API int q6k_quantize_rows(const void* x, long long ldx, int R, int K, int dtype, void* q, float* scale, cudaStream_t st) {
    return q6k_quantize_rows_launch(x, ldx, R, K, dtype, q, scale, st);
}
