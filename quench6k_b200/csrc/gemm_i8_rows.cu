// Products in 8-bit integers for few rows:
//   y[r, n] = x_scale[r] * w_scale[n] * sum_k x[r, k] w[n, k]
// with x and w in int8 and the sum in 32-bit integers (exact: K < 131,072), on mma.sync with the weights as the M side (16 output
// columns per instruction) and the rows as the N side (8 per instruction).
//
// Like its bfloat16 counterpart (gemm_skinny.cu) it is a stream of weights with as little around it as possible.  The sum over k
// may be taken in any order as long as both operands agree, so a lane fetches 16 contiguous bytes of a weight row and of an
// activation row and hands them to two instructions as if they were the layout's pieces; the four lanes that share a row cover
// 64 contiguous bytes.  A block's eight warps split K in turns, a warp has all its loads of a turn in flight at once, and the
// warps' sums meet in shared memory.
#include "common.cuh"
#include "gemm_i8.cuh"

namespace {

constexpr int R8_WARPS = 8, R8_ROWS = 16;

__device__ __forceinline__ void r8_mma(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// grid: (blocks of 16 RB columns, 1 or pairs).  NB: blocks of 8 rows; RB: blocks of 16 columns; LOADS: 16-byte loads per lane and weight row in flight at once.
template <bool DUAL, int NB, int RB, int LOADS>
__global__ void __launch_bounds__(R8_WARPS * 32) gemm_i8_rows_kernel(const I8Args p) {
    pdl_launch();
    constexpr int MATS = DUAL ? 2 : 1, TURN = 64 * LOADS;
    __shared__ int meet[R8_WARPS][MATS * RB * NB * 4 * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, pair = lane & 3;
    const int n0 = blockIdx.x * RB * 16, row0 = blockIdx.y, rows = p.pair_expert ? 1 : p.rows;
    if (!p.early) pdl_wait();
    int g = 0;
    if (p.pair_expert) {
        g = p.pair_expert[row0];
        if ((unsigned)g >= (unsigned)p.groups) return;
    }
    const uint64_t once = l2_evict_first_policy();
    const long long first = (long long)g * p.N;
    const int8_t* wrow[MATS][RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long r = first + min(n0 + rb * 16 + quad + 8 * h, p.N - 1);      // a ragged last block reads a valid row and drops the sums
            wrow[0][rb][h] = p.w + r * p.K + pair * 16;
            if (DUAL) wrow[1][rb][h] = p.w2 + r * p.K + pair * 16;
        }
    auto source = [&](int r) -> long long { return p.pair_expert ? r / p.pair_div : p.a_rows ? p.a_rows[r] : r; };
    const int8_t* xrow[NB];
    bool live[NB], waited = false;
    int acc[MATS][RB][NB][4] = {};
    for (int k0 = warp * TURN; k0 < p.K; k0 += R8_WARPS * TURN) {
        uint4 w[MATS][RB][2][LOADS], x[NB][LOADS];
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int k = k0 + j * 64;
            const bool in = k + pair * 16 < p.K;          // K is a multiple of 16: a lane's 16 bytes are inside or outside as a whole
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int h = 0; h < 2; ++h) w[m][rb][h][j] = in ? ld_once(wrow[m][rb][h] + k, once) : make_uint4(0, 0, 0, 0);
        }
        if (!waited) {
            if (p.early) pdl_wait();
            waited = true;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                live[nb] = nb * 8 + quad < rows;
                xrow[nb] = p.a + source(live[nb] ? row0 + nb * 8 + quad : row0) * p.lda + pair * 16;
            }
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int k = k0 + j * 64;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) x[nb][j] = k + pair * 16 < p.K && live[nb] ? ld_after_wait(xrow[nb] + k) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const uint4 lo = w[m][rb][0][j], hi = w[m][rb][1][j], t = x[nb][j];
                        r8_mma(acc[m][rb][nb], lo.x, hi.x, lo.y, hi.y, t.x, t.y);
                        r8_mma(acc[m][rb][nb], lo.z, hi.z, lo.w, hi.w, t.z, t.w);
                    }
    }
    if (!waited && p.early) pdl_wait();                   // a warp without a turn of its own
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 4; ++i) meet[warp][(((m * RB + rb) * NB + nb) * 4 + i) * 32 + lane] = acc[m][rb][nb][i];
    __syncthreads();
    for (int idx = threadIdx.x; idx < RB * NB * 4 * 32; idx += R8_WARPS * 32) {
        const int ln = idx & 31, i = (idx >> 5) & 3, nb = (idx >> 7) % NB, rb = (idx >> 7) / NB;
        const int n = n0 + rb * 16 + (ln >> 2) + 8 * (i >> 1), r = nb * 8 + 2 * (ln & 3) + (i & 1);
        if (n >= p.N || r >= rows) continue;
        int s = 0, s2 = 0;
#pragma unroll
        for (int q = 0; q < R8_WARPS; ++q) {
            s += meet[q][idx];
            if (DUAL) s2 += meet[q][RB * NB * 4 * 32 + idx];
        }
        const float xs = p.a_scale[source(row0 + r)];
        const float v = (float)s * (xs * p.w_scale[first + n]);
        const float u = DUAL ? (float)s2 * (xs * p.w2_scale[first + n]) : 0.0f;
        i8_store<DUAL>(p, (long long)(row0 + r) * p.ldo + n, v, u);
    }
}

template <bool DUAL, int NB, int RB, int LOADS>
void launch(const I8Args& p, int pairs, cudaStream_t st) {
    q6k_launch_as(p.early != 0, gemm_i8_rows_kernel<DUAL, NB, RB, LOADS>, dim3((p.N + RB * 16 - 1) / (RB * 16), pairs), R8_WARPS * 32, 0, st, p);
}

}  // namespace

// See ops.gemm_i8 and ops.linear_i8 for the operands: up to 16 rows, or any number of pairs.
Q6K_API int q6k_gemm_i8_rows(I8_OPERANDS, cudaStream_t st) {
    I8Args p;
    if (int rc = i8_args(&p, "gemm_i8_rows", I8_NAMES)) return rc;
    if (p.rows == 0) return 0;
    Q6K_REQUIRE(!offsets && rows <= (pair_expert ? 65535 : R8_ROWS), "gemm_i8_rows: %d rows", rows);
    const int pairs = pair_expert ? rows : 1, row_blocks = pair_expert || rows <= 8 ? 1 : 2;
    // 32 columns a block where that leaves every SM two of them; long rows of few blocks: eight loads a row at once
    const bool wide = (long long)N * pairs >= 148 * 2 * 32, deep = K >= 8192 && !wide;
    if (w2) {
        if (row_blocks == 1) launch<true, 1, 1, 4>(p, pairs, st);
        else launch<true, 2, 1, 4>(p, pairs, st);
    } else if (row_blocks == 1) {
        if (wide) launch<false, 1, 2, 4>(p, pairs, st);
        else if (deep) launch<false, 1, 1, 8>(p, pairs, st);
        else launch<false, 1, 1, 4>(p, pairs, st);
    } else {
        if (deep) launch<false, 2, 1, 8>(p, pairs, st);
        else launch<false, 2, 1, 4>(p, pairs, st);
    }
    return q6k_check_launch("gemm_i8_rows");
}
