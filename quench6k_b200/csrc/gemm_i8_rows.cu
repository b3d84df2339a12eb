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
// A single row that comes in bfloat16 is taken to 8 bits by every block for itself (by the rule of quantize.cuh), while its first
// weights are on their way, where all blocks run at a time: 2,048 x 2,048 3.0 us where two launches take 3.8 (2.3 and 3.8 if the weights are
// known to be old; 2,048 x 8,192 7.6 and 6.7, 6.4 and 6.7, and a launch less for the host); with more rows or more blocks the launch in front is
// the shorter way (four rows 5.8 and 3.8, 2 x 8,192 x 2,048 18 and 10).
#include "common.cuh"
#include "gemm_i8.cuh"
#include "quantize.cuh"

namespace {

constexpr int R8_WARPS = 8, R8_ROWS = 16;

__device__ __forceinline__ void r8_mma(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// grid: (blocks of 16 RB columns, 1 or pairs).  NB: blocks of 8 rows; RB: blocks of 16 columns; LOADS: 16-byte loads per lane and weight row in flight at once;
// HERE: the one row is x in bfloat16, taken to 8 bits here.
template <bool DUAL, int NB, int RB, int LOADS, bool HERE>
__global__ void __launch_bounds__(R8_WARPS * 32) gemm_i8_rows_kernel(const I8Args p) {
    pdl_launch();
    constexpr int MATS = DUAL ? 2 : 1, TURN = 64 * LOADS;
    __shared__ int meet[R8_WARPS][MATS * RB * NB * 4 * 32];
    __shared__ unsigned most[R8_WARPS];
    extern __shared__ __align__(16) int8_t row8[];        // HERE: [K]
    float scale = 0.0f;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, pair = lane & 3;
    const int n0 = blockIdx.x * RB * 16, row0 = blockIdx.y, rows = p.pair_expert ? 1 : p.rows;
    if (!p.early) pdl_wait();
    int g = 0;
    if (p.pair_expert) {
        g = p.pair_expert[row0];
        if ((unsigned)g >= (unsigned)p.groups) {
            if (p.early) pdl_wait();                      // a block that ends has waited too: who waits for this kernel counts on it
            return;
        }
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
    auto is_row = [&](long long r) { return !p.a_rows || (unsigned long long)r < (unsigned long long)p.a_total; };
    // every thread of the block once: the row in 8 bits to shared memory
    auto take_row = [&] {
        if constexpr (HERE) {
            unsigned m = 0;
            for (int k = threadIdx.x * 8; k < p.K; k += R8_WARPS * 256) {
                Piece<__nv_bfloat16, 8> v;
                v.take(ld_after_wait(p.x + k));
                m = max(m, v.most());
            }
            m = __reduce_max_sync(0xffffffffu, m);
            if (lane == 0) most[warp] = m;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < R8_WARPS; ++q) m = max(m, most[q]);
            const RowScale s = row_scale(m);
            scale = s.scale;
            for (int k = threadIdx.x * 8; k < p.K; k += R8_WARPS * 256) {
                Piece<__nv_bfloat16, 8> v;
                v.take(ld_after_wait(p.x + k));
                v.store(row8 + k, s.up);
            }
            __syncthreads();
        }
    };
    // thread -> (column block, row block, element of the fragment, lane of the fragment): columns quad (+8), rows 2 pair (+1).  The scales of a thread's
    // results are asked for with the first weights and rows, so that they are there when the sums are.
    constexpr int OUTS = RB * NB * 4 * 32, ITERS = (OUTS + R8_WARPS * 32 - 1) / (R8_WARPS * 32);
    auto result = [&](int it, int& idx, int& n, int& r) {
        idx = it * R8_WARPS * 32 + threadIdx.x;
        const int ln = idx & 31, i = (idx >> 5) & 3, nb = (idx >> 7) % NB, rb = (idx >> 7) / NB;
        n = n0 + rb * 16 + (ln >> 2) + 8 * (i >> 1), r = nb * 8 + 2 * (ln & 3) + (i & 1);
        return idx < OUTS && n < p.N && r < rows;
    };
    float ws[ITERS], ws2[ITERS], xs[ITERS];
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        int idx, n, r;
        const bool mine = result(it, idx, n, r);
        ws[it] = mine ? p.w_scale[first + n] : 0.0f, ws2[it] = DUAL && mine ? p.w2_scale[first + n] : 0.0f;
    }
    const int8_t* xrow[NB];
    bool live[NB], first_turn = true;
    int acc[MATS][RB][NB][4] = {};
    int k0 = warp * TURN;
    do {                                                  // (a warp without a turn of its own loads nothing in its first one)
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
        if (first_turn) {
            first_turn = false;
            if (p.early) pdl_wait();
            if constexpr (HERE) take_row();
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                live[nb] = nb * 8 + quad < rows;
                if (HERE) xrow[nb] = row8 + pair * 16;
                else {
                    const long long from = source(live[nb] ? row0 + nb * 8 + quad : row0);
                    live[nb] = live[nb] && is_row(from);
                    xrow[nb] = p.a + (live[nb] ? from : 0) * p.lda + pair * 16;
                }
            }
#pragma unroll
            for (int it = 0; it < ITERS; ++it) {
                int idx, n, r;
                if (HERE) xs[it] = scale;
                else if (result(it, idx, n, r)) {
                    const long long from = source(row0 + r);
                    xs[it] = is_row(from) ? p.a_scale[from] : __uint_as_float(0x7fffffffu);
                } else xs[it] = 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int k = k0 + j * 64;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) x[nb][j] = k + pair * 16 >= p.K || !live[nb] ? make_uint4(0, 0, 0, 0) : HERE ? *(const uint4*)(xrow[nb] + k) : ld_after_wait(xrow[nb] + k);
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
        k0 += R8_WARPS * TURN;
    } while (k0 < p.K);
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 4; ++i) meet[warp][(((m * RB + rb) * NB + nb) * 4 + i) * 32 + lane] = acc[m][rb][nb][i];
    __syncthreads();
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        int idx, n, r;
        if (!result(it, idx, n, r)) continue;
        int s = 0, s2 = 0;
#pragma unroll
        for (int q = 0; q < R8_WARPS; ++q) {
            s += meet[q][idx];
            if (DUAL) s2 += meet[q][OUTS + idx];
        }
        i8_store<DUAL>(p, (long long)(row0 + r) * p.ldo + n, (float)s * (xs[it] * ws[it]), DUAL ? (float)s2 * (xs[it] * ws2[it]) : 0.0f);
    }
}

// Pairs against short rows: a warp takes 16 columns over all of K, so that nothing waits for another warp.  grid (blocks of 16 PAIR_WARPS columns, pairs).
// The rows are taken to 8 bits by the launch in front, which has waited for all that is older: weights and pair list are fetched before the wait.
constexpr int PAIR_WARPS = 4;
template <bool DUAL, int LOADS>
__global__ void __launch_bounds__(PAIR_WARPS * 32) gemm_i8_pairs_kernel(const I8Args p) {
    pdl_launch();
    constexpr int MATS = DUAL ? 2 : 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, pair = lane & 3;
    const int n0 = (blockIdx.x * PAIR_WARPS + warp) * 16, row = blockIdx.y;
    const int g = p.pair_expert[row];
    if ((unsigned)g >= (unsigned)p.groups || n0 >= p.N) {
        pdl_wait();                                       // a warp that ends has waited too: who waits for this kernel counts on it
        return;
    }
    const uint64_t once = l2_evict_first_policy();
    const long long first = (long long)g * p.N;
    const int8_t* wrow[MATS][2];
    float ws[MATS][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long long r = first + min(n0 + quad + 8 * h, p.N - 1);      // a ragged last block reads a valid row and drops the sums
        wrow[0][h] = p.w + r * p.K + pair * 16, ws[0][h] = p.w_scale[r];
        if (DUAL) wrow[MATS - 1][h] = p.w2 + r * p.K + pair * 16, ws[MATS - 1][h] = p.w2_scale[r];
    }
    const long long from = row / p.pair_div;
    const int8_t* xrow = p.a + from * p.lda + pair * 16;
    float xs = 0.0f;
    int acc[MATS][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += 64 * LOADS) {
        uint4 w[MATS][2][LOADS], x[LOADS];
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) w[m][h][j] = k0 + j * 64 + pair * 16 < p.K ? ld_once(wrow[m][h] + k0 + j * 64, once) : make_uint4(0, 0, 0, 0);
        if (k0 == 0) {
            pdl_wait();
            xs = p.a_scale[from];
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j) x[j] = quad == 0 && k0 + j * 64 + pair * 16 < p.K ? ld_after_wait(xrow + k0 + j * 64) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                r8_mma(acc[m], w[m][0][j].x, w[m][1][j].x, w[m][0][j].y, w[m][1][j].y, x[j].x, x[j].y);
                r8_mma(acc[m], w[m][0][j].z, w[m][1][j].z, w[m][0][j].w, w[m][1][j].w, x[j].z, x[j].w);
            }
    }
    if (pair == 0) {                                      // the lanes with the one row's sums
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (n0 + quad + 8 * h < p.N)
                i8_store<DUAL>(p, (long long)row * p.ldo + n0 + quad + 8 * h, (float)acc[0][2 * h] * (xs * ws[0][h]), (float)acc[MATS - 1][2 * h] * (xs * ws[MATS - 1][h]));
    }
}

template <bool DUAL, int NB, int RB, int LOADS>
void launch(const I8Args& p, int pairs, cudaStream_t st) {
    q6k_launch_as(p.early != 0, gemm_i8_rows_kernel<DUAL, NB, RB, LOADS, false>, dim3((p.N + RB * 16 - 1) / (RB * 16), pairs), R8_WARPS * 32, 0, st, p);
}

// Whether rows (not pairs) come here rather than to the tensor-memory kernel: up to eight, or sixteen against a matrix of less than 32 MB (16 rows: 2,048 x
// 2,048 4.0 us here and 7.0 there, 5,120 x 2,048 7.1 and 9.0; 32,768 x 2,048 20 and 15, 151,936 x 2,048 64 and 52).
bool few_rows(int rows, int N, int K, bool dual) { return rows <= 8 || (rows <= R8_ROWS && (long long)N * K * (dual ? 2 : 1) < (32LL << 20)); }

// Columns and loads of a block.  Measured in a graph, weights from HBM (columns x loads a row; the first is taken):
//   one matrix: 4 loads of 16 columns (8 rows, 32,768 x 2,048: 15.6 us, 2 x 32 columns 17.3; 151,936 x 2,048: 54, 61), 8 where rows are long and blocks few (2,048 x
//   8,192: 6.6, with four 8.2);
//   a gated pair of matrices: 2 loads of 32 columns where blocks are many (2 x 8,192 x 2,048: 9.6, 4 of 16 10.2).
// Pairs (with the rows' way to 8 bits), warps for themselves or blocks that split K:
//   one matrix: warps (64 pairs, 2,048 x 512: 14.5 us and 21.4; four pairs 4.3 and 5.7; 16 pairs, 5,120 x 2,048 31.2 and 33.2), 4 loads where K ends there (256 pairs,
//   2,048 x 256: 22.8, with eight 31.5);
//   a gated pair: warps where rows are short or warps many (64 pairs, 2 x 1,024 x 512: 14.1 and 20.7; 2 x 512 x 2,048: 23.5 and 24.8), blocks otherwise (8 pairs, 2 x 512 x
//   2,048: 7.7, warps 11.8; 16 pairs, 2 x 2,048 x 5,120: 54.5, 55.9).
int launch_rows(const I8Args& p, cudaStream_t st) {
    if (p.rows == 0) return 0;
    Q6K_REQUIRE(!p.offsets && p.rows <= (p.pair_expert ? 65535 : R8_ROWS), "gemm_i8_rows: %d rows", p.rows);
    const int pairs = p.pair_expert ? p.rows : 1, two = p.pair_expert || p.rows <= 8 ? 1 : 2;      // blocks of eight rows
    const long long blocks = (long long)((p.N + 15) / 16) * pairs;                               // of 16 columns
    const bool deep = p.K >= 8192 && blocks < 4 * 148;
    if (p.pair_expert && (!p.w2 || p.K <= 256 || (p.K <= 2048 && blocks >= (p.K <= 1024 ? 5 : 8) * 148))) {
        const dim3 grid((p.N + PAIR_WARPS * 16 - 1) / (PAIR_WARPS * 16), pairs);
        if (p.w2) q6k_launch_as(true, gemm_i8_pairs_kernel<true, 4>, grid, PAIR_WARPS * 32, 0, st, p);
        else if (p.K <= 256) q6k_launch_as(true, gemm_i8_pairs_kernel<false, 4>, grid, PAIR_WARPS * 32, 0, st, p);
        else q6k_launch_as(true, gemm_i8_pairs_kernel<false, 8>, grid, PAIR_WARPS * 32, 0, st, p);
    } else if (p.w2) {
        if (two == 2) launch<true, 2, 1, 4>(p, pairs, st);
        else if (p.pair_expert || blocks >= 4 * 148) launch<true, 1, 2, 2>(p, pairs, st);
        else launch<true, 1, 1, 4>(p, pairs, st);
    } else if (two == 2) {
        if (deep) launch<false, 2, 1, 8>(p, pairs, st);
        else launch<false, 2, 1, 4>(p, pairs, st);
    } else if (deep) launch<false, 1, 1, 8>(p, pairs, st);
    else launch<false, 1, 1, 4>(p, pairs, st);
    return q6k_check_launch("gemm_i8_rows");
}

}  // namespace

int q6k_quantize_rows_launch(const void* x, long long ldx, int R, int K, int dtype, void* q, float* scale, cudaStream_t st);
int q6k_gemm_i8_tc_launch(const I8Args& p, int a_total, void* gathered, cudaStream_t st);

// Bytes of scratch that q6k_gemm_i8 takes for rows that are picked (a_rows), with groups or without; 0: the product reads them where they are.
Q6K_API long long q6k_gemm_i8_scratch(int rows, int N, int K, int dual, int grouped) {
    return !grouped && few_rows(rows, N, K, dual != 0) ? 0 : (long long)rows * (K + 4LL);
}

// See ops.gemm_i8 for the operands.  a has `a_total` rows.  gathered: scratch for rows that are picked, 16-byte aligned (q6k_gemm_i8_scratch).
Q6K_API int q6k_gemm_i8(I8_OPERANDS, int a_total, void* gathered, cudaStream_t st) {
    I8Args p;
    if (int rc = i8_args(&p, "gemm_i8", I8_NAMES)) return rc;
    Q6K_REQUIRE(!pair_expert, "gemm_i8: pairs come with rows that are not in 8 bits");
    p.a_total = a_total;
    if (!offsets && few_rows(rows, N, K, w2 != nullptr)) return launch_rows(p, st);
    return q6k_gemm_i8_tc_launch(p, a_total, gathered, st);
}

// Bytes of scratch that q6k_linear_i8 takes for T rows of dtype code that lie on 16 bytes or do not, with a pair list or without; 0: the row is taken to 8
// bits by the product's blocks, all of which run at a time.
Q6K_API long long q6k_linear_i8_scratch(int T, int N, int K, int dtype, int aligned, int pairs) {
    return T == 1 && !pairs && dtype == Q6K_BF16 && aligned && K <= 8192 && (N + 15) / 16 <= 2 * 148 ? 0 : (long long)T * K + 4LL * T;
}

// See ops.linear_i8: x of dtype code, T rows of pitch ldx; a, lda and a_scale of the operands are not looked at, and `early` says that the weights are
// older than the kernel before this call, where the row is taken to 8 bits by the product (a launch of its own in front has waited for all that
// is older).  scratch: 16-byte aligned.
Q6K_API int q6k_linear_i8(const void* x, long long ldx, int T, int dtype, void* scratch, I8_OPERANDS, cudaStream_t st) {
    I8Args p;
    if (int rc = i8_args(&p, "linear_i8", scratch, K, (const float*)((char*)scratch + (long long)T * K), rows, w, w_scale, w2, w2_scale, N, K, a_rows, offsets, groups, pair_expert,
                         pair_div, out, ldo, epilogue, act_param, 1))
        return rc;
    Q6K_REQUIRE(!offsets && !a_rows && (pair_expert ? (rows + pair_div - 1) / pair_div <= T : rows == T), "linear_i8: %d rows of %d", rows, T);
    if (rows == 0) return 0;
    const bool few = pair_expert || few_rows(rows, N, K, w2 != nullptr);
    if (q6k_linear_i8_scratch(T, N, K, dtype, ((uintptr_t)x & 15) == 0, pair_expert != nullptr) == 0) {
        p.x = (const __nv_bfloat16*)x, p.early = early;
        const int blocks = (N + 15) / 16;
        if (w2) q6k_launch_as(early != 0, gemm_i8_rows_kernel<true, 1, 1, 4, true>, blocks, R8_WARPS * 32, K, st, p);
        else if (K > 4096) q6k_launch_as(early != 0, gemm_i8_rows_kernel<false, 1, 1, 8, true>, blocks, R8_WARPS * 32, K, st, p);
        else q6k_launch_as(early != 0, gemm_i8_rows_kernel<false, 1, 1, 4, true>, blocks, R8_WARPS * 32, K, st, p);
        return q6k_check_launch("linear_i8");
    }
    Q6K_REQUIRE(scratch && ((uintptr_t)scratch & 15) == 0, "linear_i8: no scratch");
    if (int rc = q6k_quantize_rows_launch(x, ldx, T, K, dtype, scratch, (float*)p.a_scale, st)) return rc;
    return few ? launch_rows(p, st) : q6k_gemm_i8_tc_launch(p, T, nullptr, st);
}
