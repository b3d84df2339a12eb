// Products in 8-bit integers on the 5th-generation tensor cores (tcgen05.mma kind::i8, 32-bit integer accumulators in tensor
// memory), operands brought into shared memory by TMA.  sm_100a only.
//
//   y[r, n] = a_scale[r] * w_scale[g, n] * sum_k a[r, k] w[g, n, k]          int8 operands, K contiguous
//
// As in the bfloat16 products (gemm_tc.cu) the weights are the M side of the MMA and the rows the N side: a tile of 128 weight
// rows per CTA against BT rows of a.  A persistent unit (one CTA, or a pair of CTAs that work on one tile of 256 weight rows
// with cta_group::2) walks the tiles:
//   warp 0     producer: TMA loads of [128 weights x 128 bytes of k] and [rows x 128 bytes] into a ring of stages
//   warp 1     tensor memory (two accumulators) and the MMAs, four of K = 32 per stage
//   others     epilogue: accumulators to registers, the two scales, the store
// A gated product's tile holds 64 rows of the gate's matrix (lanes 0-63) and the same 64 of the other one (lanes 64-127); the
// two warps that hold a column's two products exchange half of theirs through shared memory.
// A product with fewer tiles than SMs and long rows cuts K over a cluster's CTAs (SPLIT): each leaves its 32-bit sums in its shared memory, and after a
// barrier of the cluster every CTA adds up and finishes its share of the tile's rows.  The sums are integers, so the result is the same however K is cut.
// Grouped products find their tiles from the groups' offsets in the kernel: no tile list is made.
// Every wait on an mbarrier is bounded; a wait that runs out records a code that q6k_gemm_i8_status() returns, and the roles fall
// through to the common exit.
#include <atomic>

#include "common.cuh"
#include "gemm_i8.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace {

constexpr int BK = 128;                // int8 per k-block: one 128-byte swizzle row
constexpr int WM = 128;                // weight rows of a CTA
constexpr int MAX_STAGES = 10, MAX_GROUPS = 4096;
constexpr int SWAP_BYTES = 2 * 16 * 32 * 4;      // a gated epilogue warp's 16 rows for its partner, two buffers
constexpr int SCALE_BYTES = 128 * 4;             // an epilogue warp's rows' scales

__device__ int g_i8_status = 0;

struct TcArgs {
    I8Args p;
    int stages, n_x, n_y;              // tiles along N, and along the rows (dense)
    int w_once;                        // every weight tile is fetched once, or by few units side by side
    int split;                         // SPLIT: CTAs of a cluster, which share a tile's K
    int whole, cut;                    // dense: tiles that are taken whole, and into how many pieces along the rows each of the others is cut
};

// D: 32-bit integers, A and B signed 8-bit integers, both K-major, M rows, N = n.
__device__ __forceinline__ uint32_t idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int CTAS>
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CTAS == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
            : "memory");
}
constexpr uint32_t PEER_MASK = 0xFEFFFFFFu;    // a shared-memory address of either CTA of a pair -> the same offset in the even one

template <int CTAS>
__device__ __forceinline__ void commit(uint32_t bar) {          // with a pair: at this offset in both CTAs
    if constexpr (CTAS == 1) umma_commit(bar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
                     : "memory");
}
template <int CTAS>
__device__ __forceinline__ void load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, bool once, uint64_t policy) {
    if constexpr (CTAS == 1) {
        if (once) tma_load_2d_once(dst, map, x, y, bar, policy);
        else tma_load_2d(dst, map, x, y, bar);
    } else {
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
                     "r"(x), "r"(y), "r"(bar & PEER_MASK)
                     : "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void arrive_leader(uint32_t bar) {
    if constexpr (CTAS == 1) mbar_arrive(bar);
    else asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar & PEER_MASK) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Which weights, which rows; n: the rows that are loaded and multiplied, the tile's rows rounded up.  (With whole tiles throughout, 16,384 rows of 256 experts,
// 2 x 512 columns, K 2,048, took 106 us; the L2 cache delivered 12 TB/s, a good third of it for rows of other experts.)
struct Tile {
    int g, n0, row0, row_end, n;
};

// Tile t: tiles along N fastest (units side by side share the rows).  Grouped: starts[g], in shared memory, is how many row tiles come before group g, and
// behind the groups + 1 of them lie the groups' first rows.
template <int BT, int CTAS>
__device__ __forceinline__ Tile tile_of(const TcArgs& a, int t, int cols, const int* starts) {
    Tile o;
    int rows = BT, skip = 0;                             // of the tile: which rows of it are meant
    if (!a.p.offsets && t >= a.whole) {                  // the last round of a dense product
        const int u = t - a.whole;
        rows = BT / a.cut, skip = u % a.cut * rows, t = a.whole + u / a.cut;
    }
    const int y = t / a.n_x;
    o.n0 = t % a.n_x * cols;
    if (a.p.offsets) {
        int lo = 0, hi = a.p.groups - 1;                 // the last group with starts[g] <= y (empty groups share their start with the next)
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (starts[mid] <= y) lo = mid;
            else hi = mid - 1;
        }
        o.g = lo;
        const int* offsets = starts + a.p.groups + 1;
        o.row0 = offsets[lo] + (y - starts[lo]) * BT, o.row_end = offsets[lo + 1];
    } else {
        o.g = 0, o.row0 = y * BT + skip, o.row_end = min(a.p.rows, o.row0 + rows);
    }
    o.n = max(32 * CTAS, min(BT, (o.row_end - o.row0 + 32 * CTAS - 1) / (32 * CTAS) * (32 * CTAS)));      // (a piece behind the last row is multiplied with zeros)
    return o;
}

__host__ __device__ constexpr int epilogue_warps(int bt) { return bt >= 64 ? 8 : 4; }

template <int BT, int CTAS, bool DUAL, bool SPLIT>
__global__ void __launch_bounds__(64 + 32 * epilogue_warps(BT), 1) gemm_i8_tc_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_w2,
                                                                                    const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_a32,
                                                                                    const TcArgs a) {
    if (a.p.offsets && !a.p.early) pdl_wait();
    constexpr int EW = epilogue_warps(BT), SPAN = BT / (EW / 4);       // rows that an epilogue warp takes of a whole tile
    constexpr uint32_t W_BYTES = WM * BK, A_BYTES = BT / CTAS * BK, STAGE_BYTES = W_BYTES + A_BYTES;
    constexpr int COLS = DUAL ? WM / 2 : WM;                           // output columns of a CTA's tile
    constexpr uint32_t TMEM_COLS = 2 * BT <= 32 ? 32 : 2 * BT <= 64 ? 64 : 2 * BT <= 128 ? 128 : 2 * BT <= 256 ? 256 : 512;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t bars[2 * MAX_STAGES + 4];
    __shared__ uint32_t tmem_slot;
    const I8Args& p = a.p;
    const int stages = a.stages, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = smem_u32(smem), swap0 = ring + stages * STAGE_BYTES;
    const uint32_t scales0 = swap0 + (DUAL ? EW * SWAP_BYTES : 0);
    int* starts = (int*)(smem + (size_t)stages * STAGE_BYTES + (DUAL ? EW * SWAP_BYTES : 0) + EW * SCALE_BYTES);
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[MAX_STAGES]);
    const uint32_t acc_full0 = smem_u32(&bars[2 * MAX_STAGES]), acc_empty0 = smem_u32(&bars[2 * MAX_STAGES + 2]);
    const int rank = CTAS == 2 ? (int)cluster_rank() : 0;
    const int per_unit = SPLIT ? a.split : CTAS, unit = blockIdx.x / per_unit, units = gridDim.x / per_unit;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1);
        for (int b = 0; b < 2; ++b) mbar_init(acc_full0 + 8 * b, 1), mbar_init(acc_empty0 + 8 * b, EW * CTAS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_a) : "memory");
    }
    if (warp == 1) {
        if constexpr (CTAS == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    if (p.offsets) {                                     // row tiles before each group (everyone fetches, so that one latency passes and not one for each 32 groups)
        int* offsets = starts + p.groups + 1;
        for (int g = threadIdx.x; g <= p.groups; g += blockDim.x) offsets[g] = min(max(p.offsets[g], 0), p.rows);
        __syncthreads();
        if (warp == 2) {
            int before = 0;
            for (int g0 = 0; g0 <= p.groups; g0 += 32) {
                const int g = g0 + lane;
                const int rows = g < p.groups ? offsets[g + 1] - offsets[g] : 0;
                const int mine = rows > 0 ? (rows + BT - 1) / BT : 0;
                int upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                if (g <= p.groups) starts[g] = before + upto - mine;
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CTAS == 2) cluster_sync();             // both CTAs' barriers exist before either signals the other
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch();                                        // this block holds its tensor memory: a successor may come
    const int total = p.offsets ? a.n_x * starts[p.groups] : a.whole + (a.n_x * a.n_y - a.whole) * a.cut, kb_all = (p.K + BK - 1) / BK;
    // the k-blocks of this CTA: kb0 .. kb0 + kbs - 1 (SPLIT: one tile for each cluster, and every slice has some)
    const int slice = SPLIT ? (int)cluster_rank() : 0, slice_kbs = SPLIT ? (kb_all + a.split - 1) / a.split : kb_all;
    const int kb0 = slice * slice_kbs, kbs = min(slice_kbs, kb_all - kb0);

    if (warp == 0) {
        if (elect_one()) {
            const uint64_t once = l2_evict_first_policy();
            auto load_w = [&](uint32_t st, uint32_t fb, int i, int wy, int n) {
                if (rank == 0) mbar_expect_tx(fb, CTAS * W_BYTES + n * BK);
                load<CTAS>(st, &tm_w, (kb0 + i) * BK, wy, fb, a.w_once, once);
                if (DUAL) load<CTAS>(st + W_BYTES / 2, &tm_w2, (kb0 + i) * BK, wy, fb, a.w_once, once);
            };
            int pre = 0;                                 // k-blocks whose weights went out before the wait (with nothing to wait for, the first rows would queue behind them)
            for (int t = unit; p.early && t < total && pre < stages; t += units) {
                const Tile tl = tile_of<BT, CTAS>(a, t, CTAS * COLS, starts);
                for (int i = 0; i < kbs && pre < stages; ++i, ++pre) load_w(ring + pre * STAGE_BYTES, full0 + 8 * pre, i, tl.g * p.N + tl.n0 + rank * COLS, tl.n);
            }
            pdl_wait();
            int s = 0;
            uint32_t st = ring, phase = 0;
            bool ok = true;
            for (int t = unit; t < total && ok; t += units) {
                const Tile tl = tile_of<BT, CTAS>(a, t, CTAS * COLS, starts);
                const int wy = tl.g * p.N + tl.n0 + rank * COLS, ay = tl.row0 + rank * (tl.n / CTAS);
                for (int i = 0; i < kbs; ++i) {
                    const uint32_t fb = full0 + 8 * s;
                    if (pre > 0) {                       // a fresh stage, its weights on the way
                        --pre;
                    } else {
                        if (!mbar_wait(empty0 + 8 * s, phase ^ 1)) {
                            atomicExch(&g_i8_status, 21);
                            ok = false;
                            break;
                        }
                        load_w(st, fb, i, wy, tl.n);
                    }
                    if (tl.n == BT) load<CTAS>(st + W_BYTES, &tm_a, (kb0 + i) * BK, ay, fb, false, once);
                    else
                        for (int c = 0; c < tl.n / CTAS; c += 32) load<CTAS>(st + W_BYTES + c * BK, &tm_a32, (kb0 + i) * BK, ay + c, fb, false, once);
                    if (++s == stages) s = 0, st = ring, phase ^= 1;
                    else st += STAGE_BYTES;
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            int s = 0, nt = 0;
            uint32_t st = ring, phase = 0;
            bool ok = true;
            for (int t = unit; t < total && ok; t += units, ++nt) {
                const int buf = nt & 1;
                if (!mbar_wait(acc_empty0 + 8 * buf, ((nt >> 1) & 1) ^ 1)) {
                    atomicExch(&g_i8_status, 24);
                    break;
                }
                tc_fence_after();
                const uint32_t idesc = idesc_i8(CTAS * WM, tile_of<BT, CTAS>(a, t, CTAS * COLS, starts).n);
                for (int i = 0; i < kbs; ++i) {
                    if (!mbar_wait(full0 + 8 * s, phase)) {
                        atomicExch(&g_i8_status, 22);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t dw = umma_desc_k(st), da = umma_desc_k(st + W_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / 32; ++k) umma_i8<CTAS>(tmem + buf * BT, dw + 2 * k, da + 2 * k, idesc, (i | k) != 0);      // + 32 bytes of k per step
                    commit<CTAS>(empty0 + 8 * s);
                    if (++s == stages) s = 0, st = ring, phase ^= 1;
                    else st += STAGE_BYTES;
                }
                if (ok) commit<CTAS>(acc_full0 + 8 * buf);
            }
        }
    } else {
        const int quarter = warp & 3, part = (warp - 2) >> 2;           // lanes 32 quarter .. of the accumulator, rows part * SPAN .. of the tile
        const bool gate = quarter < 2;
        const uint32_t mine = swap0 + (warp - 2) * SWAP_BYTES, theirs = swap0 + ((part << 2 | ((quarter ^ 2) + 2 & 3)) * SWAP_BYTES);
        int nt = 0, turn = 0;
        bool ok = true;
        pdl_wait();                                      // the rows' scales come from the kernel before, and the output may still be in use by it
        for (int t = unit; t < total; t += units, ++nt) {
            const Tile tl = tile_of<BT, CTAS>(a, t, CTAS * COLS, starts);
            const int buf = nt & 1, n = tl.n0 + rank * COLS + (DUAL ? quarter & 1 : quarter) * 32 + lane;
            const long long at_n = (long long)tl.g * p.N + n;
            const float ws = n < p.N ? p.w_scale[at_n] : 0.0f, ws2 = DUAL && n < p.N ? p.w2_scale[at_n] : 0.0f;
            const int span = tl.n == BT ? SPAN : (tl.n / (EW / 4) + 31) / 32 * 32, row0 = tl.row0 + part * span;      // this warp's rows of the tile
            const int end = min(span, tl.row_end - row0);
            // the rows' scales go to shared memory while the accumulator fills (read from global memory where they are needed, every 16 rows waited for them:
            // 2,048 x 2,048 x 2,048 16.0 us, 15.4 that way)
            const uint32_t scales = scales0 + (warp - 2) * SCALE_BYTES;
            __syncwarp();
#pragma unroll
            for (int c = 0; c < SPAN; c += 32) {             // (span is at most SPAN)
                const int r = row0 + c + lane;
                const float xs = r < tl.row_end ? p.a_scale[r] : 0.0f;
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(scales + (c + lane) * 4), "f"(xs) : "memory");
            }
            __syncwarp();
            auto scales_of = [&](int c0, float* xs) {    // of 16 rows
#pragma unroll
                for (int j = 0; j < 16; j += 4)
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(xs[j]), "=f"(xs[j + 1]), "=f"(xs[j + 2]), "=f"(xs[j + 3]) : "r"(scales + (c0 + j) * 4) : "memory");
            };
            if (ok && !mbar_wait(acc_full0 + 8 * buf, (nt >> 1) & 1)) {
                if (lane == 0) atomicExch(&g_i8_status, 23);
                ok = false;                              // on to the barriers that a partner may be waiting at, with no further wait
            }
            tc_fence_after();
            const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + buf * BT + part * span;
            auto release = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_leader<CTAS>(acc_empty0 + 8 * buf);
            };
            if (end <= 0) release();
            if constexpr (SPLIT) {                       // the sums of this slice, row by row, where the ring was (every MMA has read it)
#pragma unroll 1
                for (int c0 = 0; ok && c0 < end; c0 += 16) {
                    float v[16];
                    tmem_ld16_issue(from + c0, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + ((part * span + c0 + j) * WM + quarter * 32 + lane) * 4), "f"(v[j]) : "memory");
                }
            } else if constexpr (DUAL) {
#pragma unroll 1
                for (int c0 = 0; c0 < end; c0 += 32, ++turn) {
                    float v[16], u[16];                  // 32-bit integers until they are scaled
                    tmem_ld16_issue(from + c0 + (gate ? 0 : 16), v);
                    tmem_ld16_issue(from + c0 + (gate ? 16 : 0), u);
                    tmem_ld_wait();
                    if (c0 + 32 >= end) release();
                    const uint32_t at = (turn & 1) * (SWAP_BYTES / 2) + lane * 4;
#pragma unroll
                    for (int j = 0; j < 16; ++j) asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + at + j * 128), "f"(u[j]) : "memory");
                    // both have written; and the buffers of the turn before have been read
                    asm volatile("bar.sync %0, 64;" ::"r"(1 + part * 2 + (quarter & 1)) : "memory");
#pragma unroll
                    for (int j = 0; j < 16; ++j) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(u[j]) : "r"(theirs + at + j * 128) : "memory");
                    const int first = c0 + (gate ? 0 : 16), rows = n < p.N ? end - first : 0;
                    float xs[16];
                    scales_of(first, xs);
                    __nv_bfloat16* o = (__nv_bfloat16*)p.out + (long long)(row0 + first) * p.ldo + n;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float g = (float)__float_as_int(gate ? v[j] : u[j]) * (xs[j] * ws), up = (float)__float_as_int(gate ? u[j] : v[j]) * (xs[j] * ws2);
                        v[j] = g, u[j] = up;
                    }
                    if (p.act == 0) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] = i8_silu_times(v[j], u[j]);
                    } else {
#pragma unroll 1
                        for (int i = 0; i < 4; ++i) {       // a loop over quarters: sixteen copies of the other gates' code do not fit the instruction cache
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float y = q6k_gated(v[j], u[j], p.act, p.act_param);
                                v[j] = v[j + 4], v[j + 4] = v[j + 8], v[j + 8] = v[j + 12], v[j + 12] = y;
                                u[j] = u[j + 4], u[j + 4] = u[j + 8], u[j + 8] = u[j + 12];
                            }
                        }
                    }
                    if (rows >= 16) {
#pragma unroll
                        for (int j = 0; j < 16; ++j, o += p.ldo) *o = __float2bfloat16_rn(v[j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j, o += p.ldo)
                            if (j < rows) *o = __float2bfloat16_rn(v[j]);
                    }
                }
            } else {
#pragma unroll 1
                for (int c0 = 0; c0 < end; c0 += 16) {
                    float v[16];                         // 32-bit integers until they are scaled
                    tmem_ld16_issue(from + c0, v);
                    tmem_ld_wait();
                    if (c0 + 16 >= end) release();
                    float xs[16];
                    scales_of(c0, xs);
                    const int rows = n < p.N ? end - c0 : 0;
                    const long long at = (long long)(row0 + c0) * p.ldo + n;
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = (float)__float_as_int(v[j]) * (xs[j] * ws);
                    if (p.epilogue == I8_ACT) {
                        __nv_bfloat16* o = (__nv_bfloat16*)p.out + at;
#pragma unroll 1
                        for (int i = 0; i < 16; ++i, o += p.ldo) {
                            if (i < rows) *o = __float2bfloat16_rn(q6k_activation(v[0], p.act));
#pragma unroll
                            for (int j = 0; j < 15; ++j) v[j] = v[j + 1];
                        }
                    } else if (p.epilogue == I8_ADD) {   // nobody else adds here: one addition each, without waiting for what is there
                        float* o = (float*)p.out + at;
#pragma unroll
                        for (int j = 0; j < 16; ++j, o += p.ldo)
                            if (j < rows) atomicAdd(o, v[j]);      // (a sum below 1.2e-38 may become 0)
                    } else if (rows >= 16) {
                        float* o = (float*)p.out + at;
#pragma unroll
                        for (int j = 0; j < 16; ++j, o += p.ldo) *o = v[j];
                    } else {
                        float* o = (float*)p.out + at;
#pragma unroll
                        for (int j = 0; j < 16; ++j, o += p.ldo)
                            if (j < rows) *o = v[j];
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (SPLIT) {
        cluster_sync();                                  // every slice's sums are there
        const Tile tl = tile_of<BT, CTAS>(a, unit, COLS, starts);
        const int rows = min(tl.row_end - tl.row0, BT), share = (rows + a.split - 1) / a.split, r0 = slice * share, r1 = min(rows, r0 + share);
        for (int i = r0 * (COLS / 4) + threadIdx.x; i < r1 * (COLS / 4); i += blockDim.x) {
            const int r = i / (COLS / 4), c = i % (COLS / 4) * 4;
            int s[4] = {}, s2[4] = {};
            for (int q = 0; q < a.split; ++q) {
                int v[4];
                uint32_t at;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(ring + (r * WM + c) * 4), "r"(q));
                asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += v[j];
                if (DUAL) {
                    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at + COLS * 4) : "memory");
#pragma unroll
                    for (int j = 0; j < 4; ++j) s2[j] += v[j];
                }
            }
            const float xs = p.a_scale[tl.row0 + r];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = tl.n0 + c + j;
                if (n < p.N)
                    i8_store<DUAL>(p, (long long)(tl.row0 + r) * p.ldo + n, (float)s[j] * (xs * p.w_scale[n]), DUAL ? (float)s2[j] * (xs * p.w2_scale[n]) : 0.0f);
            }
        }
        cluster_sync();                                  // nobody leaves while others read its sums
    }
    if constexpr (CTAS == 2) cluster_sync();             // the peer has no MMA, copy or arrival of ours in flight
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// Rows picked from a with their scales, a warp each, so that the tiles' loads find them side by side (a number outside a: zeros and the scale NaN).
// (Loads that gather four rows each, in the product itself, are too slow for it: 2,048 tokens against 256 experts took 266 us that way and 115 this way, this kernel
// included; 24 tokens 76 and 52.)
__global__ void __launch_bounds__(256) gather_i8_kernel(const int8_t* a, long long lda, const float* a_scale, const int* a_rows, int a_total, int rows, int K, int8_t* out, float* scale) {
    pdl_enter();
    const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= rows) return;
    const int from = a_rows[r];
    const bool is_row = (unsigned)from < (unsigned)a_total;
    const int8_t* src = a + from * lda;
    int8_t* dst = out + (long long)r * K;
    if (lane == 0) scale[r] = is_row ? a_scale[from] : __uint_as_float(0x7fffffffu);
    for (int k0 = lane * 16; k0 < K; k0 += 4 * 512) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (k0 + i * 512 < K) v[i] = is_row ? *(const uint4*)(src + k0 + i * 512) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (k0 + i * 512 < K) *(uint4*)(dst + k0 + i * 512) = v[i];
    }
}

// ---------------------------------------------------------------------------------------- host
// An int8 matrix [rows, cols] in boxes of [box_rows, 128] with the 128-byte swizzle; reads outside give zeros.
int make_i8_map(CUtensorMap* map, const void* base, long long rows, int cols, long long pitch, int box_rows, bool weights) {
    EncodeTiled fn = encode_fn();
    if (!fn) return q6k_fail("gemm_i8: the driver does not offer cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, weights ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return q6k_fail("gemm_i8: cuTensorMapEncodeTiled failed with code %d (%lld rows of %d, pitch %lld, box %d)", (int)r, rows, cols, pitch, box_rows);
    return 0;
}

int sm_count() {
    static int n = 0;
    if (!n) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    }
    return n;
}

template <int BT, int CTAS, bool DUAL, bool SPLIT = false>
int launch(const TcArgs& args, int a_total, cudaStream_t st) {
    TcArgs t = args;
    const I8Args& p = t.p;
    constexpr int EW = epilogue_warps(BT), COLS = CTAS * (DUAL ? WM / 2 : WM);
    constexpr int stage = WM * BK + BT / CTAS * BK;
    CUtensorMap tw, tw2, ta, ta32;
    const int w_box = DUAL ? WM / 2 : WM;
    if (int rc = make_i8_map(&tw, p.w, (long long)p.groups * p.N, p.K, p.K, w_box, true)) return rc;
    tw2 = tw;
    if (DUAL)
        if (int rc = make_i8_map(&tw2, p.w2, (long long)p.groups * p.N, p.K, p.K, w_box, true)) return rc;
    if (int rc = make_i8_map(&ta, p.a, a_total, p.K, p.lda, BT / CTAS, false)) return rc;
    if (int rc = make_i8_map(&ta32, p.a, a_total, p.K, p.lda, 32, false)) return rc;
    const int extra = (DUAL ? EW * SWAP_BYTES : 0) + EW * SCALE_BYTES + (p.offsets ? 2 * (p.groups + 1) * 4 : 0);
    t.stages = (222 * 1024 - extra) / stage;
    if (t.stages > MAX_STAGES) t.stages = MAX_STAGES;
    t.n_x = (p.N + COLS - 1) / COLS, t.n_y = (p.rows + BT - 1) / BT;
    const long long row_tiles = p.offsets ? p.rows / BT + (p.groups < p.rows ? p.groups : p.rows) : t.n_y, total = t.n_x * row_tiles;
    const int units = sm_count() / CTAS;
    Q6K_REQUIRE(total < (1LL << 31) - 2 * 148, "gemm_i8: %lld tiles", total);
    t.whole = t.cut > 1 ? (int)(total - total % units) : (int)total;
    t.w_once = p.offsets ? p.rows <= 2LL * p.groups * BT : t.n_y == 1;
    const size_t smem = (size_t)t.stages * stage + extra + 1024;
    static std::atomic<unsigned long long> configured{0};              // a bit for each device
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= 64) return q6k_fail("gemm_i8: device %d", device);
    if (!(configured.load() >> device & 1)) {
        if (cudaFuncSetAttribute(gemm_i8_tc_kernel<BT, CTAS, DUAL, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024) != cudaSuccess)
            return q6k_check_launch("gemm_i8: shared memory attribute");
        configured.fetch_or(1ull << device);
    }
    const int cluster = SPLIT ? t.split : CTAS;
    Q6K_REQUIRE(!SPLIT || total * cluster <= 0x7fffffff, "gemm_i8: %lld tiles of %d slices", total, cluster);
    const long long pieces = p.offsets ? total : t.whole + (total - t.whole) * t.cut;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster * (unsigned)(SPLIT || pieces < units ? pieces : units)), cfg.blockDim = dim3(64 + 32 * EW), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[2];
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster, attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    if (i8_overlaps(p)) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    cfg.attrs = attr;
    cudaLaunchKernelEx(&cfg, gemm_i8_tc_kernel<BT, CTAS, DUAL, SPLIT>, tw, tw2, ta, ta32, t);
    return q6k_check_launch("gemm_i8");
}

// Rows of a tile (negative: a pair of CTAs).  A unit's time for one tile of K = 2,048, in tenths of a microsecond, measured over many tiles (8,192 x 2
// columns): a wide tile re-reads less and feeds the tensor cores better, a narrow one leaves fewer units idle in the last round.  With the least
// rounds x time, 1,522 rows x (2 x 8,192), K 2,048 take 40.8 us on pairs of 256 (42.6 of 192; 60.3 with single CTAs of 128), 256 rows x 2,048 take
// 6.6 us on tiles of 32 (7.2 of 128, 11.1 on pairs), 64 rows x (2 x 8,192) 9.7 on 64 (12.8 on 32), all in a graph with weights from HBM.
// Grouped rows: the experts' shares are known on the device only, so half as much again as an even share.
// split: CTAs that share a tile's K, where that takes less time: a slice's share of it and two microseconds for the sums to meet (2,048 columns, K 8,192,
// 32 rows: 16.8 us in 16 CTAs, 10.3 in four slices; K 2,048: 7.0 and 7.0, in two 8.4).
// cut: the pieces along the rows of each tile of the last round, where its tiles fill less than half of the units (1,522 rows x (2 x 8,192): 14 tiles over 74
// pairs as 56 pieces of 64 rows, 42.0 -> 40.6 us; 2,048 rows x 8,192 33.8 -> 32.3).  A piece takes longer than a narrow tile of a product of narrow tiles: with their
// times 1,300 x 4,096, K 4,096 was cut, too, and took 25.5 us instead of 23.6.
int choose_tile(const I8Args& p, bool dual, int* split, int* cut) {
    *split = *cut = 1;
    if (p.offsets) {
        const int share = p.rows / p.groups + p.rows / p.groups / 2;
        return share <= 32 ? 32 : share <= 64 ? 64 : 128;
    }
    static const int tiles[][2] = {{32, 35}, {64, 38}, {128, 47}, {256, 76}, {-192, 56}, {-256, 64}};
    long long best = -1;
    int pick = 0;
    for (auto& t : tiles) {
        const int bt = t[0] < 0 ? -t[0] : t[0], ctas = t[0] < 0 ? 2 : 1, cols = ctas * (dual ? WM / 2 : WM);
        const long long units = sm_count() / ctas, count = (long long)((p.N + cols - 1) / cols) * ((p.rows + bt - 1) / bt);
        const int kbs = (p.K + BK - 1) / BK;
        const long long cost = (count + units - 1) / units * t[1] * kbs;                  // in units of a sixteenth of a tenth of a microsecond
        if (best < 0 || cost < best) best = cost, pick = t[0], *split = *cut = 1;
        for (int c = 2; count > units && bt / c >= 32 * ctas && count % units * c <= units; ++c) {
            if (count % units == 0 || bt % c || bt / c % (32 * ctas)) continue;
            const int piece = bt / c / ctas;                                             // rows that each CTA loads for one
            const long long with = (count / units * t[1] + (piece <= 32 ? 48 : piece <= 64 ? 52 : 56)) * kbs;
            if (with < best) best = with, pick = t[0], *split = 1, *cut = c;
        }
        // clusters whose CTAs all run at a time: 96 in eights, 128 in fours and twos (of 148 SMs; 16 clusters of eight took two rounds)
        for (int s = 2; ctas == 1 && bt <= 128 && s <= 8 && count * s <= (s == 8 ? 96 : 128) && (s - 1) * ((kbs + s - 1) / s) < kbs; s *= 2) {
            const long long sliced = (long long)t[1] * ((kbs + s - 1) / s) + 16 * 20;
            if (sliced < best) best = sliced, pick = t[0], *split = s, *cut = 1;
        }
    }
    return pick;
}

}  // namespace

Q6K_API int q6k_gemm_i8_status() {
    int v = -1;
    if (cudaMemcpyFromSymbol(&v, g_i8_status, sizeof v) != cudaSuccess) return -1;
    return v;
}

// More than a few rows, or groups.  gathered (with a_rows): rows * (K + 4) bytes of scratch, for the rows that are picked and their scales.
int q6k_gemm_i8_tc_launch(const I8Args& p, int a_total, void* gathered, cudaStream_t st) {
    TcArgs t{p};
    if (p.rows == 0) return 0;
    Q6K_REQUIRE(p.groups <= MAX_GROUPS && (long long)p.groups * p.N < (1LL << 31) - 256, "gemm_i8: %d groups (at most %d) of %d columns", p.groups, MAX_GROUPS, p.N);
    if (p.a_rows) {
        Q6K_REQUIRE(gathered && ((uintptr_t)gathered & 15) == 0, "gemm_i8: no scratch for the rows that are picked");
        float* gathered_scale = (float*)((char*)gathered + (long long)p.rows * p.K);
        q6k_launch(gather_i8_kernel, (p.rows + 7) / 8, 256, 0, st, p.a, p.lda, p.a_scale, p.a_rows, a_total, p.rows, p.K, (int8_t*)gathered, gathered_scale);
        if (int rc = q6k_check_launch("gemm_i8: gather")) return rc;
        t.p.a = (const int8_t*)gathered, t.p.a_scale = gathered_scale, t.p.a_rows = nullptr, t.p.lda = p.K, t.p.early = 1;
        a_total = p.rows;
    }
    Q6K_REQUIRE(a_total >= p.rows, "gemm_i8: %d rows of %d", p.rows, a_total);
    const bool dual = p.w2 != nullptr;
    const int tile = choose_tile(t.p, dual, &t.split, &t.cut);
    if (t.split > 1) {
        if (tile == 32) return dual ? launch<32, 1, true, true>(t, a_total, st) : launch<32, 1, false, true>(t, a_total, st);
        if (tile == 64) return dual ? launch<64, 1, true, true>(t, a_total, st) : launch<64, 1, false, true>(t, a_total, st);
        if (tile == 128) return dual ? launch<128, 1, true, true>(t, a_total, st) : launch<128, 1, false, true>(t, a_total, st);
        return q6k_fail("gemm_i8: tiles of %d rows in slices", tile);
    }
#define GO(T_, BT_, CTAS_) \
    case T_: return dual ? launch<BT_, CTAS_, true>(t, a_total, st) : launch<BT_, CTAS_, false>(t, a_total, st)
    switch (tile) {
        GO(32, 32, 1);
        GO(64, 64, 1);
        GO(128, 128, 1);
        GO(256, 256, 1);
        GO(-192, 192, 2);
        GO(-256, 256, 2);
    }
#undef GO
    return q6k_fail("gemm_i8: tiles of %d rows", tile);
}
