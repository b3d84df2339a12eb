// Products in 8-bit integers for few rows:
//   y[r, n] = x_scale[r] * w_scale[n] * sum_k x[r, k] w[n, k]
// with x and w in int8 and the sum in 32-bit integers (exact: K < 131,072), on mma.sync with the weights as the M side (16 output
// columns per instruction) and the rows as the N side (8 per instruction).
//
// Like its bfloat16 counterpart (gemm_skinny.cu) it is a stream of weights with as little around it as possible.  The sum over k
// may be taken in any order as long as both operands agree, so a lane fetches 16 contiguous bytes of a weight row and of an
// activation row and hands them to two instructions as if they were the layout's pieces; the four lanes that share a row cover
// 64 contiguous bytes.  A block's eight warps split K, and their sums meet in shared memory.
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

// grid: (blocks of 16 columns, tiles of 16 rows or pairs)
template <bool DUAL>
__global__ void __launch_bounds__(R8_WARPS * 32) gemm_i8_rows_kernel(const I8Args p) {
    pdl_enter();
    constexpr int MATS = DUAL ? 2 : 1, NB = R8_ROWS / 8;
    __shared__ int meet[R8_WARPS][MATS * NB * 4 * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, pair = lane & 3;
    const int n0 = blockIdx.x * 16;
    int g = 0, row0, rows;
    if (p.pair_expert) {
        g = p.pair_expert[blockIdx.y];
        if ((unsigned)g >= (unsigned)p.groups) return;
        row0 = blockIdx.y, rows = 1;
    } else if (p.offsets) {
        int tiles = 0, end = 0;
        for (g = 0; g < p.groups; ++g) {
            end = min(p.offsets[g + 1], p.rows);
            const int mine = (end - p.offsets[g] + R8_ROWS - 1) / R8_ROWS;
            if (mine > 0 && tiles + mine > (int)blockIdx.y) break;
            tiles += max(mine, 0);
        }
        if (g == p.groups) return;
        row0 = p.offsets[g] + ((int)blockIdx.y - tiles) * R8_ROWS;
        rows = min(R8_ROWS, end - row0);
    } else {
        row0 = blockIdx.y * R8_ROWS, rows = min(R8_ROWS, p.rows - row0);
    }
    auto source = [&](int r) -> long long { return p.pair_expert ? r / p.pair_div : p.a_rows ? p.a_rows[r] : r; };

    const long long first = (long long)g * p.N;
    const int8_t* wrow[MATS][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long long r = first + min(n0 + quad + 8 * h, p.N - 1);      // a ragged last block reads a valid row and drops the sums
        wrow[0][h] = p.w + r * p.K + pair * 16;
        if (DUAL) wrow[1][h] = p.w2 + r * p.K + pair * 16;
    }
    const int8_t* xrow[NB];
    bool live[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        live[nb] = nb * 8 + quad < rows;
        xrow[nb] = p.a + source(live[nb] ? row0 + nb * 8 + quad : row0) * p.lda + pair * 16;
    }
    int acc[MATS][NB][4] = {};
    for (int k = warp * 64; k < p.K; k += R8_WARPS * 64) {
        const bool in = k + pair * 16 < p.K;              // K is a multiple of 16: a lane's 16 bytes are inside or outside as a whole
        uint4 b[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) b[nb] = in && live[nb] ? *(const uint4*)(xrow[nb] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            const uint4 lo = in ? *(const uint4*)(wrow[m][0] + k) : make_uint4(0, 0, 0, 0), hi = in ? *(const uint4*)(wrow[m][1] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                r8_mma(acc[m][nb], lo.x, hi.x, lo.y, hi.y, b[nb].x, b[nb].y);
                r8_mma(acc[m][nb], lo.z, hi.z, lo.w, hi.w, b[nb].z, b[nb].w);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 4; ++i) meet[warp][((m * NB + nb) * 4 + i) * 32 + lane] = acc[m][nb][i];
    __syncthreads();
    for (int idx = threadIdx.x; idx < NB * 4 * 32; idx += R8_WARPS * 32) {
        const int ln = idx & 31, i = (idx >> 5) & 3, nb = idx >> 7;
        const int n = n0 + (ln >> 2) + 8 * (i >> 1), r = nb * 8 + 2 * (ln & 3) + (i & 1);
        if (n >= p.N || r >= rows) continue;
        int s = 0, s2 = 0;
#pragma unroll
        for (int q = 0; q < R8_WARPS; ++q) {
            s += meet[q][idx];
            if (DUAL) s2 += meet[q][NB * 4 * 32 + idx];
        }
        const float xs = p.a_scale[source(row0 + r)];
        const float v = (float)s * (xs * p.w_scale[first + n]);
        const float u = DUAL ? (float)s2 * (xs * p.w2_scale[first + n]) : 0.0f;
        i8_store<DUAL>(p, (long long)(row0 + r) * p.ldo + n, v, u);
    }
}

}  // namespace

// See ops.gemm_i8 for the operands.  row_tiles: how many tiles of 16 rows there are at most.
Q6K_API int q6k_gemm_i8_rows(I8_OPERANDS, cudaStream_t st) {
    I8Args p;
    if (int rc = i8_args(&p, "gemm_i8_rows", I8_NAMES)) return rc;
    if (p.rows == 0) return 0;
    const long long tiles = pair_expert ? rows : offsets ? rows / R8_ROWS + (groups < rows ? groups : rows) : (rows + R8_ROWS - 1) / R8_ROWS;
    Q6K_REQUIRE(tiles <= 65535, "gemm_i8_rows: %lld tiles of rows", tiles);
    const dim3 grid((N + 15) / 16, (unsigned)tiles);
    if (w2) q6k_launch(gemm_i8_rows_kernel<true>, grid, R8_WARPS * 32, 0, st, p);
    else q6k_launch(gemm_i8_rows_kernel<false>, grid, R8_WARPS * 32, 0, st, p);
    return q6k_check_launch("gemm_i8_rows");
}
