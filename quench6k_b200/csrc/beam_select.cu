// Beam search's choice: for each request the `count` best continuations of its `width` beams,
//   t[b, v] = score[b] + x[b, v] - log sum_v' exp x[b, v']
// over all beams b and tokens v, in descending order, the lowest place b V + v first among equals.  A continuation whose beam's
// score, logit or sum is not finite counts as -infinity: it comes after every other one, in order of place.
//
// Logits are read once.  A block takes a part of one row and leaves the part's maximum, its sum of exponentials over that
// maximum, and its `count` best logits (within a row the order of the logits is the order of t).  A block per request then
// makes the rows' sums and finds the best of what the parts left.  t is compared in 64 bits, where scores of different beams are not made equal by
// a rounding to 32, nor those of logits of one row that differ by more than some 2^-52 of the score (closer ones, next to zero, are cut by the logit and
// listed by place).
#include <cfloat>

#include "umma.cuh"

namespace {

constexpr int SEL_THREADS = 256, SEL_MAX_COUNT = 128, SEL_MAX_WIDTH = 32;
constexpr int SEL_EACH = 32, SEL_TILE = SEL_THREADS * SEL_EACH;
constexpr int MERGE_THREADS = 512, MERGE_WARPS = MERGE_THREADS / 32, MERGE_HELD = 4;
constexpr int SEL_WARPS = SEL_THREADS / 32, SEL_POOL = 1024, SEL_TILES = 8, SEL_AGAIN = 4;       // keys that a pool holds; the most tiles of a part; pieces that a warp reads again at once
constexpr int SEL_PARTS = 4;       // parts to an SM that a long batch is cut into (8: 29 us where 4 take 25, 128 rows of 151,936 logits: more parts leave more to merge)
constexpr float LOG2E = 1.4426950408889634f;

// An order-preserving number of a finite logit, above 0; 0 for what is not finite.
__device__ __forceinline__ unsigned finite_key(float v) {
    const unsigned u = __float_as_uint(v == 0.0f ? 0.0f : v);
    if ((u & 0x7fffffffu) >= 0x7f800000u) return 0u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k); }
// The same for a score in 64 bits (finite by construction).
__device__ __forceinline__ unsigned long long score_key(double v) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(v == 0.0 ? 0.0 : v);
    return (u >> 63) ? ~u : (u | (1ull << 63));
}

template <int WARPS>
__device__ __forceinline__ int block_count(int v, int* red) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) t += red[w];
    return t;
}

// The best `count` of many keys without sorting them: a number that at least `count` of them reach and few others do.  Every thread brings the largest
// of the keys that it holds.  Few wanted: the first warp's lanes take the largest of THREADS / 32 of those each, and the count-th largest of the 32 is taken out
// by one maximum after the other.  Otherwise the count-th largest of all threads' keys is found from its highest bit down, a barrier for each bit, and no further
// than until few more reach it than are wanted (eight wanted of 512 keys: 1.1 us that way, 0.5 the other; with sixteen wanted more keys are let through than the barriers cost).
// 0: fewer than `count` of those hold any key.  slot: THREADS words of shared memory.
template <int THREADS>
__device__ __forceinline__ unsigned block_threshold(unsigned mine, int count, unsigned* slot) {
    unsigned t = 0;
    if (count <= 12) {
        slot[threadIdx.x] = mine;
        __syncthreads();
        if (threadIdx.x < 32) {
            unsigned k = 0;
#pragma unroll
            for (int i = 0; i < THREADS / 32; ++i) k = max(k, slot[i * 32 + threadIdx.x]);
            for (int i = 0; i < count; ++i) {
                t = __reduce_max_sync(0xffffffffu, k);
                if ((int)threadIdx.x == __ffs(__ballot_sync(0xffffffffu, k == t)) - 1) k = 0;
            }
            if (threadIdx.x == 0) slot[0] = t;
        }
        __syncthreads();
        return slot[0];
    }
    for (int bit = 31; bit >= 0; --bit) {
        const unsigned trial = t | (1u << bit);
        const int c = __syncthreads_count(mine >= trial);
        if (c >= count) t = trial;
        if (c >= count && c <= count + count / 4) break;
    }
    return t;
}

// What a part of a row leaves: its maximum and its sum of exponentials over that maximum.
struct PartHead {
    float most, sum;
};

// grid (parts, rows); a part is `tiles` tiles of 8,192 logits.  best/at: [rows, parts, count] (at -1: none); heads: [rows, parts].  WIDE: rows start
// on 16 bytes.  The pass over the logits keeps each thread's maximum of every tile and its sum, and nothing in it waits for another warp.  The threads'
// maxima give the threshold; the few (thread, tile) pieces that reach it are read again, a warp each.
template <bool WIDE>
__global__ void __launch_bounds__(SEL_THREADS, 4) beam_part_kernel(const float* logits, int V, int tiles, int count, float* best, int* at, PartHead* heads) {
    pdl_enter();
    __shared__ int red[SEL_WARPS];
    __shared__ PartHead of_warp[SEL_WARPS];
    __shared__ unsigned slots[SEL_THREADS];
    __shared__ __align__(16) unsigned long long pool[SEL_POOL];      // a logit's key above the complement of its place: the order of the result in one number
    __shared__ float piece_most[SEL_TILES][SEL_THREADS];
    __shared__ unsigned short pieces[SEL_TILES * SEL_THREADS];
    __shared__ int taken, listed;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* row = logits + (size_t)blockIdx.y * V;
    const int lo = blockIdx.x * tiles * SEL_TILE, hi = (int)min((long long)V, (long long)lo + (long long)tiles * SEL_TILE);
    const size_t slot = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    best += slot * count, at += slot * count;
    auto where = [](int thread, int j) { return WIDE ? (j >> 2) * (SEL_THREADS * 4) + thread * 4 + (j & 3) : j * SEL_THREADS + thread; };
    float most = -INFINITY, sum = 0.0f;                      // of this thread (a NaN is passed over by the maxima and found again in the sum)
    if (threadIdx.x == 0) taken = 0, listed = 0;
    for (int t = 0; t < tiles && lo + t * SEL_TILE < hi; ++t) {
        const int n = hi - lo - t * SEL_TILE;                // (WIDE: a multiple of 4)
        const float* tile = row + lo + t * SEL_TILE;
        float v[SEL_EACH];
        if (WIDE) {
#pragma unroll
            for (int j = 0; j < SEL_EACH; j += 4) {
                const int i = where(threadIdx.x, j);
                const float4 f = i < n ? *(const float4*)(tile + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                v[j] = f.x, v[j + 1] = f.y, v[j + 2] = f.z, v[j + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < SEL_EACH; ++j) v[j] = where(threadIdx.x, j) < n ? tile[where(threadIdx.x, j)] : -INFINITY;
        }
        float high = -INFINITY;
#pragma unroll
        for (int j = 0; j < SEL_EACH; ++j) high = fmaxf(high, v[j]);
        piece_most[t][threadIdx.x] = high;
        const float m = fmaxf(most, high);
        if (m > -INFINITY) {
            // 2^(x L - c) with c = m L rounded: the rounding of c multiplies the whole sum by 2^d, d = m L - c, which is known exactly.  d is up to 2^-24 of c, so
            // that 2^d and 2^-d leave the range of a float where c is beyond 2^31, and m L itself may be infinite: from |m| = 10^6 on (d up to 1/16) the
            // differences x - m, which are exact there for every x whose term counts, are taken instead.
            const float c = m * LOG2E, d = fmaf(m, LOG2E, -c);
            float here = 0.0f;
            if (fabsf(m) < 1e6f) {
#pragma unroll
                for (int j = 0; j < SEL_EACH; ++j) here += ex2_approx(fmaf(v[j], LOG2E, -c));
                here *= ex2_approx(-d);
            } else {
#pragma unroll
                for (int j = 0; j < SEL_EACH; ++j) here += ex2_approx((v[j] - m) * LOG2E);
            }
            sum = sum * ex2_approx((most - m) * LOG2E) + here;
            most = m;
        } else {
#pragma unroll
            for (int j = 0; j < SEL_EACH; ++j)
                if (!(v[j] == -INFINITY)) sum = NAN;         // nothing but NaNs
        }
    }
    const float warp_most = warp_max(most);
    if (most > -INFINITY) sum *= ex2_approx((most - warp_most) * LOG2E);
    sum = warp_sum(sum);
    if (lane == 0) of_warp[warp] = PartHead{warp_most, sum};
    const unsigned low = block_threshold<SEL_THREADS>(finite_key(most), count, slots);
    const float reach = low != 0 ? key_value(low) : -FLT_MAX;
    if (threadIdx.x == 0) {
        PartHead h = of_warp[0];
#pragma unroll
        for (int w = 1; w < SEL_WARPS; ++w) h.most = fmaxf(h.most, of_warp[w].most);
        h.sum = 0.0f;
#pragma unroll
        for (int w = 0; w < SEL_WARPS; ++w)
            if (of_warp[w].sum != 0.0f) h.sum += of_warp[w].sum * ex2_approx((of_warp[w].most - h.most) * LOG2E);
        heads[slot] = h;
    }
    for (int t = 0; t < tiles && lo + t * SEL_TILE < hi; ++t)
        if (piece_most[t][threadIdx.x] >= reach && most < INFINITY) pieces[atomicAdd(&listed, 1)] = (unsigned short)(t * SEL_THREADS + threadIdx.x);
    __syncthreads();
    for (int i0 = warp; i0 < listed; i0 += SEL_WARPS * SEL_AGAIN) {
        float v[SEL_AGAIN];
        int p[SEL_AGAIN], many = 0;
#pragma unroll
        for (int u = 0; u < SEL_AGAIN; ++u) {
            const int i = i0 + u * SEL_WARPS, piece = i < listed ? pieces[i] : 0;
            p[u] = lo + piece / SEL_THREADS * SEL_TILE + where(piece % SEL_THREADS, lane);
            v[u] = i < listed && p[u] < hi ? row[p[u]] : -INFINITY;
        }
        unsigned who[SEL_AGAIN];
#pragma unroll
        for (int u = 0; u < SEL_AGAIN; ++u) who[u] = __ballot_sync(0xffffffffu, v[u] >= reach), many += __popc(who[u]);
        int to = 0;
        if (lane == 0) to = atomicAdd(&taken, many);
        to = __shfl_sync(0xffffffffu, to, 0);
#pragma unroll
        for (int u = 0; u < SEL_AGAIN; ++u) {
            const int at_u = to + __popc(who[u] & ((1u << lane) - 1u));
            if (v[u] >= reach && at_u < SEL_POOL) pool[at_u] = (unsigned long long)finite_key(v[u]) << 32 | (unsigned)~p[u];
            to += __popc(who[u]);
        }
    }
    __syncthreads();
    const int found = taken;
    if (found <= SEL_POOL) {
        for (int i = threadIdx.x; i < found; i += SEL_THREADS) {
            int rank = 0;
            const unsigned long long k = pool[i];
#pragma unroll 8
            for (int j = 0; j < found; ++j) rank += pool[j] > k;
            if (rank < count) best[rank] = key_value((unsigned)(k >> 32)), at[rank] = (int)~(unsigned)k;
        }
        for (int i = found + threadIdx.x; i < count; i += SEL_THREADS) at[i] = -1;
        return;
    }
    // too many equal ones (or an order that hides the best): the count-th largest (logit, lowest place) bit by bit
    __syncthreads();
    if (threadIdx.x == 0) taken = 0;
    auto how_many = [&](auto&& is) {
        int c = 0;
        for (int i = lo + threadIdx.x; i < hi; i += SEL_THREADS) c += is(finite_key(row[i]), i);
        return block_count<SEL_WARPS>(c, red);
    };
    unsigned kth = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const unsigned trial = kth | (1u << bit);
        if (how_many([&](unsigned k, int) { return k >= trial; }) >= count) kth = trial;
    }
    const int above = how_many([&](unsigned k, int) { return k > kth; });
    int last = 0;                                            // of the logits equal to it, those at places below `last` are taken
    for (int step = 1 << 30; step > 0; step >>= 1)
        if (how_many([&](unsigned k, int i) { return k == kth && i < last + step; }) <= count - above) last += step;
    for (int i = lo + threadIdx.x; i < hi; i += SEL_THREADS) {
        const unsigned k = finite_key(row[i]);
        if (k > kth || (k == kth && i < last)) {
            const int to = atomicAdd(&taken, 1);
            if (to < count) best[to] = row[i], at[to] = i;
        }
    }
}

// grid: requests.
__global__ void __launch_bounds__(MERGE_THREADS) beam_merge_kernel(const float* logits, const float* scores, int V, int width, int parts, int count,
                                                                 const float* best, const int* at, const PartHead* heads, float* out_score, int* out_beam,
                                                                 int* out_token) {
    pdl_enter();
    __shared__ double base[SEL_MAX_WIDTH], row_most[SEL_MAX_WIDTH];      // the beam's score less the logarithm of its row's sum over the row's maximum
    __shared__ bool dead[SEL_MAX_WIDTH];
    __shared__ int red[MERGE_WARPS];
    __shared__ unsigned slots[MERGE_THREADS];
    __shared__ unsigned long long key[SEL_POOL];
    __shared__ int place[SEL_POOL];
    __shared__ int taken;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t row0 = (size_t)blockIdx.x * width;
    heads += row0 * parts, best += row0 * parts * count, at += row0 * parts * count, scores += row0;
    const int per_row = parts * count, all = width * per_row;
    // A thread's candidates: one of each 512, at another rank of its list each time (the lists are in order: with the same rank throughout, a few threads would
    // hold all the best, and their maxima would let through more than the pool takes: 128 wanted, 16 requests of 8 beams over 151,936 tokens, 141 us).
    auto candidate = [&](int h) { return h * MERGE_THREADS + ((threadIdx.x + h * 197) & (MERGE_THREADS - 1)); };
    // the first ones are asked for before the rows' sums are made, and kept
    int held_at[MERGE_HELD];
    float held_best[MERGE_HELD];
#pragma unroll
    for (int h = 0; h < MERGE_HELD; ++h) {
        const int i = candidate(h);
        held_at[h] = i < all ? at[i] : -1, held_best[h] = i < all ? best[i] : 0.0f;
    }
    for (int b = warp; b < width; b += MERGE_WARPS) {
        const float score = scores[b];
        float most = -INFINITY;
        double sum = 0.0;                                    // over `most`
        for (int s = lane; s < parts; s += 32) {
            const PartHead h = heads[b * parts + s];
            if (h.sum == 0.0f) continue;                     // nothing finite
            const float m = fmaxf(most, h.most);
            sum = sum * expf(most - m) + (double)h.sum * expf(h.most - m);       // one of the two exponents is 0
            most = m;
        }
        const float all_most = warp_max(most);
        if (sum != 0.0) sum *= expf(most - all_most);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            const double d = (double)score - log(sum);
            base[b] = d, row_most[b] = (double)all_most, dead[b] = !(fabs(d) < INFINITY && fabsf(all_most) < INFINITY);
        }
    }
    if (threadIdx.x == 0) taken = 0;
    __syncthreads();
    const float inverse = 1.0f / (float)per_row;
    auto one = [&](int i, int token, float value, auto&& f) {
        int b = (int)((float)i * inverse);
        b -= b * per_row > i, b += (b + 1) * per_row <= i;
        if (token >= 0 && !dead[b]) f(score_key(base[b] + ((double)value - row_most[b])), b * V + token);
    };
    auto each = [&](auto&& f) {                              // every candidate; the rows are spread over all threads
#pragma unroll
        for (int h = 0; h < MERGE_HELD; ++h) one(candidate(h), held_at[h], held_best[h], f);
#pragma unroll 4
        for (int h = MERGE_HELD; h * MERGE_THREADS < all; ++h) {
            const int i = candidate(h);
            if (i < all) one(i, at[i], best[i], f);
        }
    };
    unsigned long long mine = 0;
    int c = 0;
    each([&](unsigned long long k, int) { mine = k > mine ? k : mine, ++c; });
    const int want = min(count, block_count<MERGE_WARPS>(c, red));
    const unsigned long long reach = (unsigned long long)block_threshold<MERGE_THREADS>((unsigned)(mine >> 32), count, slots) << 32;
    auto take = [&](unsigned long long k, int w) {
        const int to = atomicAdd(&taken, 1);
        if (to < SEL_POOL) key[to] = k, place[to] = w;
    };
    each([&](unsigned long long k, int w) {
        if (k >= reach) take(k, w);
    });
    __syncthreads();
    int found = taken;
    if (found > SEL_POOL) {                                  // as in the parts: the want-th largest (score, lowest place) bit by bit
        auto how_many = [&](auto&& is) {
            c = 0;
            each([&](unsigned long long k, int w) { c += is(k, w); });
            return block_count<MERGE_WARPS>(c, red);
        };
        unsigned long long kth = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long trial = kth | (1ull << bit);
            if (how_many([&](unsigned long long k, int) { return k >= trial; }) >= want) kth = trial;
        }
        const int above = how_many([&](unsigned long long k, int) { return k > kth; });
        int last = 0;
        for (int step = 1 << 30; step > 0; step >>= 1)
            if (how_many([&](unsigned long long k, int w) { return k == kth && w < last + step; }) <= want - above) last += step;
        __syncthreads();
        if (threadIdx.x == 0) taken = 0;
        __syncthreads();
        each([&](unsigned long long k, int w) {
            if (k > kth || (k == kth && w < last)) take(k, w);
        });
        __syncthreads();
        found = min(taken, SEL_POOL);
    }
    out_score += (size_t)blockIdx.x * count, out_beam += (size_t)blockIdx.x * count, out_token += (size_t)blockIdx.x * count;
    for (int i = threadIdx.x; i < found; i += MERGE_THREADS) {
        int rank = 0;
        const unsigned long long u = key[i];
        const int w = place[i];
#pragma unroll 8
        for (int j = 0; j < found; ++j) rank += key[j] > u || (key[j] == u && place[j] < w);
        if (rank >= want) continue;
        out_score[rank] = (float)__longlong_as_double((long long)((u >> 63) ? u & ~(1ull << 63) : ~u));
        out_beam[rank] = w / V, out_token[rank] = w % V;
    }
    // fewer finite continuations than wanted (every one of them is listed): the others in order of place
    if (warp == 0) {
        int filled = want;
        for (int b = 0; b < width && filled < count; ++b)
            for (int v0 = 0; v0 < V && filled < count; v0 += 32) {
                const int v = v0 + lane;
                const bool mine = v < V && (dead[b] || finite_key(logits[(row0 + b) * V + v]) == 0u);
                const unsigned who = __ballot_sync(0xffffffffu, mine);
                const int to = filled + __popc(who & ((1u << lane) - 1u));
                if (mine && to < count) out_score[to] = -INFINITY, out_beam[to] = b, out_token[to] = v;
                filled += __popc(who);
            }
    }
}

// Tiles of a part: as many as leave some four parts to an SM (which run at a time).
int part_tiles(long long rows, int V) {
    const int tiles = (V + SEL_TILE - 1) / SEL_TILE, most = tiles < SEL_TILES ? tiles : SEL_TILES;
    const long long each = (rows * tiles + SEL_PARTS * 148 - 1) / (SEL_PARTS * 148);
    return (int)(each < 1 ? 1 : each < most ? each : most);
}
int row_parts(long long rows, int V) {
    const int tiles = (V + SEL_TILE - 1) / SEL_TILE, each = part_tiles(rows, V);
    return (tiles + each - 1) / each;
}

}  // namespace

// Bytes of scratch that q6k_beam_select takes.
Q6K_API long long q6k_beam_scratch(int rows, int V, int count) {
    return (long long)rows * row_parts(rows, V) * ((long long)count * 8 + (long long)sizeof(PartHead));
}

// logits: FP32 [requests * width, V]; scores: FP32 [requests, width]; out_*: [requests, count].
Q6K_API int q6k_beam_select(const float* logits, const float* scores, int requests, int width, int V, int count, void* scratch, long long scratch_bytes,
                            float* out_score, int* out_beam, int* out_token, cudaStream_t st) {
    if (requests == 0) return 0;
    Q6K_REQUIRE(requests > 0 && requests * (long long)width <= 65535 && width >= 1 && width <= SEL_MAX_WIDTH && V >= 1 && (long long)width * V < (1LL << 31),
                "beam_select: %d requests of %d beams over %d tokens", requests, width, V);
    Q6K_REQUIRE(count >= 1 && count <= SEL_MAX_COUNT && count <= (long long)width * V, "beam_select: %d continuations of %d beams over %d tokens", count, width, V);
    const int rows = requests * width, tiles = part_tiles(rows, V), parts = row_parts(rows, V);
    Q6K_REQUIRE(scratch_bytes >= q6k_beam_scratch(rows, V, count), "beam_select: %lld bytes of scratch, %lld are needed", scratch_bytes, q6k_beam_scratch(rows, V, count));
    float* best = (float*)scratch;
    int* at = (int*)(best + (size_t)rows * parts * count);
    PartHead* heads = (PartHead*)(at + (size_t)rows * parts * count);
    if (V % 4 == 0 && ((uintptr_t)logits & 15) == 0) q6k_launch(beam_part_kernel<true>, dim3(parts, rows), SEL_THREADS, 0, st, logits, V, tiles, count, best, at, heads);
    else q6k_launch(beam_part_kernel<false>, dim3(parts, rows), SEL_THREADS, 0, st, logits, V, tiles, count, best, at, heads);
    q6k_launch_as(true, beam_merge_kernel, requests, MERGE_THREADS, 0, st, logits, scores, V, width, parts, count, best, at, heads, out_score, out_beam, out_token);
    return q6k_check_launch("beam_select");
}
