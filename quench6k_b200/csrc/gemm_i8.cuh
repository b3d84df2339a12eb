// What the 8-bit product kernels share: their operands, the checks of them, and how a result leaves.
#pragma once
#include "common.cuh"

enum { I8_STORE = 0, I8_ADD = 1, I8_GATED = 2, I8_ACT = 4 };     // FP32 stored or added; bfloat16 act(v) * u, bfloat16 act(v)

struct I8Args {
    const int8_t *a, *w, *w2;
    const float *a_scale, *w_scale, *w2_scale;
    const int* a_rows;             // row r of the product is row a_rows[r] of a (null: r)
    const int* offsets;            // grouped: rows offsets[g] .. offsets[g + 1] - 1 go against matrix g
    const int* pair_expert;        // pairs: row r is row r / pair_div of a against matrix pair_expert[r]
    void* out;
    long long lda, ldo;
    int rows, N, K, groups, pair_div;
    int early;                     // the kernel before this one on the stream made a and a_scale and nothing else that is read here
    int epilogue, act;
    float act_param;
    const __nv_bfloat16* x;        // not null: the one row of a and its scale are still to be made from this
    int a_total;                   // with a_rows: the rows of a; a number outside them gives a row of NaN
};

namespace {

#define I8_OPERANDS                                                                                                                   \
    const void *a, long long lda, const float *a_scale, int rows, const void *w, const float *w_scale, const void *w2, const float *w2_scale, int N, int K, \
        const int *a_rows, const int *offsets, int groups, const int *pair_expert, int pair_div, void *out, long long ldo, int epilogue, float act_param, int early
#define I8_NAMES a, lda, a_scale, rows, w, w_scale, w2, w2_scale, N, K, a_rows, offsets, groups, pair_expert, pair_div, out, ldo, epilogue, act_param, early

inline int i8_args(I8Args* p, const char* who, I8_OPERANDS) {
    const int act = epilogue >> 8, epi = epilogue & 255;         // the activation's code (q6k_activation) rides above bit 8
    Q6K_REQUIRE(rows >= 0 && N > 0 && K > 0 && K % 16 == 0 && K < 131072, "%s: %d rows, N=%d, K=%d (a multiple of 16 below 131072)", who, rows, N, K);
    Q6K_REQUIRE(lda % 16 == 0 && lda >= K && (((uintptr_t)a | (uintptr_t)w | (uintptr_t)w2) & 15) == 0, "%s: rows must start on 16 bytes", who);
    Q6K_REQUIRE((epi == I8_GATED) == (w2 != nullptr) && (epi == I8_STORE || epi == I8_ADD || epi == I8_GATED || epi == I8_ACT), "%s: epilogue %d", who, epi);
    Q6K_REQUIRE(act >= 0 && act <= (epi == I8_GATED ? Q6K_ACT_CLAMPED : 2), "%s: unknown activation %d", who, act);
    Q6K_REQUIRE(!(offsets && pair_expert) && groups >= 1 && pair_div >= 1, "%s: groups %d, pair_div %d", who, groups, pair_div);
    *p = I8Args{(const int8_t*)a, (const int8_t*)w, (const int8_t*)w2, a_scale, w_scale, w2_scale, a_rows, offsets, pair_expert, out, lda, ldo,
                rows, N, K, groups, pair_div, early, epi, act, act_param, nullptr, 0};
    return 0;
}

// Whether the launch may start while the kernel before it still runs (it then fetches weights before its wait).  Where the caller cannot say what that
// kernel writes, it may be these very weights, just taken to 8 bits.
inline bool i8_overlaps(const I8Args& p) { return p.early != 0 && q6k_pdl_mode() != 0; }

// silu(g) u by a fast exponential and quotient: the exponential is off by up to 2 + 1.2 |g| units of 2^-23, which is the result's error where it outweighs the 1
// (2^-17 at g = -40), the quotient by two; the result is then rounded to bfloat16 (2^-8).  Where e^-g is beyond 2^126 the value is below 1e-36 |u| and
// comes out as zero.
__device__ __forceinline__ float i8_silu_times(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }
__device__ __forceinline__ float i8_gated(float g, float u, int act, float param) { return act == 0 ? i8_silu_times(g, u) : q6k_gated(g, u, act, param); }

// v (and u, the second matrix's) is the scaled product that belongs at out[at].
template <bool DUAL>
__device__ __forceinline__ void i8_store(const I8Args& p, long long at, float v, float u) {
    if (DUAL) ((__nv_bfloat16*)p.out)[at] = __float2bfloat16_rn(i8_gated(v, u, p.act, p.act_param));
    else if (p.epilogue == I8_ACT) ((__nv_bfloat16*)p.out)[at] = __float2bfloat16_rn(q6k_activation(v, p.act));
    else if (p.epilogue == I8_ADD) ((float*)p.out)[at] += v;
    else ((float*)p.out)[at] = v;
}

}  // namespace
