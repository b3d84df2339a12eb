// Beam search's choice: for each request the `count` best continuations of its `width` beams,
//   t[b, v] = score[b] + x[b, v] - log sum_v' exp x[b, v']
// over all beams b and tokens v, in descending order, the lowest place b V + v first among equals.  A continuation whose beam's
// score, logit or sum is not finite counts as -infinity: it comes after every other one, in order of place.
//
// Logits are read once.  A block takes a slice of one row and leaves the slice's maximum, its sum of exponentials over that
// maximum, and its `count` best logits (within a row the order of the logits is the order of t).  A block per request then
// makes the rows' sums and finds the best of what the slices left.  t is compared in 64 bits: two logits of one row that differ
// give scores that differ, and scores of different beams are not made equal by a rounding.
#include "common.cuh"

namespace {

constexpr int SEL_THREADS = 256, SEL_MAX_COUNT = 256, SEL_MAX_WIDTH = 32;
constexpr int SEL_EACH = 32, SEL_SLICE = SEL_THREADS * SEL_EACH;
constexpr int SEL_WARPS = SEL_THREADS / 32, SEL_POOL = 1024;       // how many keys are ranked by counting

// An order-preserving number of a finite logit, above 0; 0 for what is not finite.
__device__ __forceinline__ unsigned finite_key(float v) {
    const unsigned u = __float_as_uint(v == 0.0f ? 0.0f : v);
    if ((u & 0x7fffffffu) >= 0x7f800000u) return 0u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// The same for a score in 64 bits (finite by construction).
__device__ __forceinline__ unsigned long long score_key(double v) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(v == 0.0 ? 0.0 : v);
    return (u >> 63) ? ~u : (u | (1ull << 63));
}

__device__ __forceinline__ int block_count(int v, int* red) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int w = 0; w < SEL_WARPS; ++w) t += red[w];
    return t;
}

// The best `count` of many keys without sorting them: a key that at least `count` others reach.  Every thread brings the largest of the
// keys that it holds; each warp finds the ceil(count / warps)-th largest of its threads' keys, and the smallest of those is reached by
// as many keys as are wanted (or is 0, where there are fewer).  The keys that reach it are few: they are collected and ranked.
__device__ __forceinline__ unsigned warp_kth(unsigned mine, int k) {
    unsigned m = 0;
    for (; k > 0; --k) {
        m = __reduce_max_sync(0xffffffffu, mine);
        const unsigned who = __ballot_sync(0xffffffffu, mine == m);
        if ((threadIdx.x & 31) == __ffs(who) - 1) mine = 0;
        if (m == 0) break;
    }
    return m;
}
__device__ __forceinline__ unsigned long long warp_kth(unsigned long long mine, int k) {
    unsigned long long m = 0;
    for (; k > 0; --k) {
        const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(mine >> 32));
        const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(mine >> 32) == hi ? (unsigned)mine : 0u);
        m = (unsigned long long)hi << 32 | lo;
        const unsigned who = __ballot_sync(0xffffffffu, mine == m);
        if ((threadIdx.x & 31) == __ffs(who) - 1) mine = 0;
        if (m == 0) break;
    }
    return m;
}
template <typename K>
__device__ __forceinline__ K block_threshold(K mine, int count, K* of_warp) {
    const K m = warp_kth(mine, (count + SEL_WARPS - 1) / SEL_WARPS);
    if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = m;
    __syncthreads();
    K t = of_warp[0];
#pragma unroll
    for (int w = 1; w < SEL_WARPS; ++w) t = of_warp[w] < t ? of_warp[w] : t;
    return t;
}

// grid (slices, rows).  best/at: [rows, slices, count]; head: [rows, slices] of {maximum, sum, how many}.
struct SliceHead {
    float most, sum;
    int found;
};

// WIDE: rows start on 16 bytes.
template <bool WIDE>
__global__ void __launch_bounds__(SEL_THREADS, 4) beam_slice_kernel(const float* logits, int V, int count, float* best, int* at, SliceHead* heads) {
    pdl_enter();
    __shared__ int red[SEL_WARPS];
    __shared__ float redf[32];
    __shared__ unsigned of_warp[SEL_WARPS];
    __shared__ unsigned all[SEL_SLICE];                      // every key of the slice, where the pool is not enough
    unsigned* key = all;
    int* place = (int*)(all + SEL_POOL);
    __shared__ int taken;
    const float* row = logits + (size_t)blockIdx.y * V;
    const int lo = blockIdx.x * SEL_SLICE, n = min(V - lo, SEL_SLICE);
    const size_t slot = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    float v[SEL_EACH];
    auto where = [&](int j) { return WIDE ? (j >> 2) * (SEL_THREADS * 4) + (int)threadIdx.x * 4 + (j & 3) : j * SEL_THREADS + (int)threadIdx.x; };
    if (WIDE) {
#pragma unroll
        for (int j = 0; j < SEL_EACH; j += 4) {
            const float4 f = where(j) < n ? __ldcs((const float4*)(row + lo + where(j))) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);      // n is a multiple of 4
            v[j] = f.x, v[j + 1] = f.y, v[j + 2] = f.z, v[j + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < SEL_EACH; ++j) v[j] = where(j) < n ? __ldcs(row + lo + where(j)) : -INFINITY;
    }
    float most = -INFINITY;
    unsigned mine = 0;
    bool bad = false;                                        // a value that makes the row's sum not finite
#pragma unroll
    for (int j = 0; j < SEL_EACH; ++j) {
        most = fmaxf(most, v[j]);
        bad |= !(v[j] < INFINITY);
    }
    mine = finite_key(most);                                 // rows with another value that is not finite take no part
    if (threadIdx.x == 0) taken = 0;
    const unsigned reach = max(block_threshold(mine, count, of_warp), 1u);
    most = warp_max(most);
    if ((threadIdx.x & 31) == 0) redf[threadIdx.x >> 5] = most;
    const bool any_bad = __syncthreads_or(bad);
#pragma unroll
    for (int w = 0; w < SEL_WARPS; ++w) most = fmaxf(most, redf[w]);
    if (any_bad || most == -INFINITY) {
        if (threadIdx.x == 0) heads[slot] = SliceHead{most, any_bad ? NAN : 0.0f, 0};
        return;
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < SEL_EACH; ++j) {
        sum += __expf(v[j] - most);
        const unsigned k = finite_key(v[j]);
        if (k >= reach) {
            const int to = atomicAdd(&taken, 1);
            if (to < SEL_POOL) key[to] = k, place[to] = where(j);
        }
    }
    sum = block_sum(sum, redf);
    const int found = taken;
    if (threadIdx.x == 0) heads[slot] = SliceHead{most, sum, min(count, found)};
    if (found <= SEL_POOL) {
        for (int i = threadIdx.x; i < found; i += SEL_THREADS) {
            int rank = 0;
            const unsigned k = key[i];
            const int p = place[i];
            for (int j = 0; j < found; ++j) rank += key[j] > k || (key[j] == k && place[j] < p);
            if (rank < count) best[slot * count + rank] = row[lo + p], at[slot * count + rank] = lo + p;
        }
        return;
    }
    // too many equal ones (or an order that hides the best): the count-th largest (logit, lowest place) bit by bit
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SEL_EACH; ++j) all[where(j)] = finite_key(v[j]);
    if (threadIdx.x == 0) taken = 0;
    __syncthreads();
    auto how_many = [&](auto&& is) {
        int c = 0;
        for (int i = threadIdx.x; i < SEL_SLICE; i += SEL_THREADS) c += is(all[i], i);
        return block_count(c, red);
    };
    unsigned kth = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const unsigned trial = kth | (1u << bit);
        if (how_many([&](unsigned k, int) { return k >= trial; }) >= count) kth = trial;
    }
    const int above = how_many([&](unsigned k, int) { return k > kth; });
    int last = 0;                                            // of the logits equal to it, those at places below `last` are taken
    for (int step = SEL_SLICE; step > 0; step >>= 1)
        if (how_many([&](unsigned k, int i) { return k == kth && i < last + step; }) <= count - above) last += step;
    for (int i = threadIdx.x; i < n; i += SEL_THREADS)
        if (all[i] > kth || (all[i] == kth && i < last)) {
            const int to = atomicAdd(&taken, 1);
            if (to < count) best[slot * count + to] = row[lo + i], at[slot * count + to] = lo + i;
        }
}

// grid: requests.
__global__ void __launch_bounds__(SEL_THREADS) beam_merge_kernel(const float* logits, const float* scores, int V, int width, int slices, int count,
                                                                 const float* best, const int* at, const SliceHead* heads, float* out_score, int* out_beam,
                                                                 int* out_token) {
    pdl_enter();
    __shared__ double base[SEL_MAX_WIDTH];                   // the beam's score less the logarithm of its row's sum
    __shared__ bool dead[SEL_MAX_WIDTH];
    __shared__ int red[SEL_THREADS / 32];
    __shared__ unsigned long long of_warp[SEL_WARPS], key[SEL_POOL];
    __shared__ int place[SEL_POOL];
    __shared__ int taken;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t row0 = (size_t)blockIdx.x * width;
    heads += row0 * slices, best += row0 * slices * count, at += row0 * slices * count, scores += row0;
    for (int b = warp; b < width; b += SEL_THREADS / 32) {
        float most = -INFINITY;
        for (int s = lane; s < slices; s += 32) most = fmaxf(most, heads[b * slices + s].most);
        most = warp_max(most);
        double sum = 0.0;
        for (int s = lane; s < slices; s += 32) {
            const SliceHead h = heads[b * slices + s];
            if (!(h.sum == 0.0f)) sum += (double)h.sum * exp((double)h.most - (double)most);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            const double d = (double)scores[b] - ((double)most + log(sum));
            base[b] = d, dead[b] = !(fabs(d) < INFINITY);
        }
    }
    if (threadIdx.x == 0) taken = 0;
    __syncthreads();
    const int per_row = slices * count, all = width * per_row;
    auto candidate = [&](int i, unsigned long long& k, int& where) {
        const int b = i / per_row, s = i / count % slices;
        if (dead[b] || i % count >= heads[b * slices + s].found) return false;
        const int token = at[i];
        k = score_key(base[b] + (double)best[i]), where = b * V + token;
        return true;
    };
    unsigned long long mine = 0;
    int c = 0;
    for (int i = threadIdx.x; i < all; i += SEL_THREADS) {
        unsigned long long k;
        int w;
        if (candidate(i, k, w)) mine = k > mine ? k : mine, ++c;
    }
    const int want = min(count, block_count(c, red));
    const unsigned long long reach = block_threshold(mine, count, of_warp);
    if (want > 0) {
        for (int i = threadIdx.x; i < all; i += SEL_THREADS) {
            unsigned long long k;
            int w;
            if (candidate(i, k, w) && k >= reach) {
                const int to = atomicAdd(&taken, 1);
                if (to < SEL_POOL) key[to] = k, place[to] = w;
            }
        }
    }
    __syncthreads();
    int found = taken;
    if (found > SEL_POOL) {                                  // as in the slices: the want-th largest (score, lowest place) bit by bit
        auto how_many = [&](auto&& is) {
            c = 0;
            for (int i = threadIdx.x; i < all; i += SEL_THREADS) {
                unsigned long long k;
                int w;
                c += candidate(i, k, w) && is(k, w);
            }
            return block_count(c, red);
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
        for (int i = threadIdx.x; i < all; i += SEL_THREADS) {
            unsigned long long k;
            int w;
            if (candidate(i, k, w) && (k > kth || (k == kth && w < last))) {
                const int to = atomicAdd(&taken, 1);
                if (to < SEL_POOL) key[to] = k, place[to] = w;
            }
        }
        __syncthreads();
        found = min(taken, SEL_POOL);
    }
    out_score += (size_t)blockIdx.x * count, out_beam += (size_t)blockIdx.x * count, out_token += (size_t)blockIdx.x * count;
    for (int i = threadIdx.x; i < found; i += SEL_THREADS) {
        int rank = 0;
        const unsigned long long u = key[i];
        const int w = place[i];
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

int sel_slices(int V) { return (V + SEL_SLICE - 1) / SEL_SLICE; }

}  // namespace

Q6K_API int q6k_beam_max_count() { return SEL_MAX_COUNT; }
Q6K_API int q6k_beam_max_width() { return SEL_MAX_WIDTH; }
// Bytes of scratch that q6k_beam_select takes.
Q6K_API long long q6k_beam_scratch(int rows, int V, int count) {
    return (long long)rows * sel_slices(V) * ((long long)count * 8 + (long long)sizeof(SliceHead));
}

// logits: FP32 [requests * width, V]; scores: FP32 [requests, width]; out_*: [requests, count].
Q6K_API int q6k_beam_select(const float* logits, const float* scores, int requests, int width, int V, int count, void* scratch, long long scratch_bytes,
                            float* out_score, int* out_beam, int* out_token, cudaStream_t st) {
    if (requests == 0) return 0;
    Q6K_REQUIRE(requests > 0 && requests * (long long)width <= 65535 && width >= 1 && width <= SEL_MAX_WIDTH && V >= 1 && (long long)width * V < (1LL << 31),
                "beam_select: %d requests of %d beams over %d tokens", requests, width, V);
    Q6K_REQUIRE(count >= 1 && count <= SEL_MAX_COUNT && count <= (long long)width * V, "beam_select: %d continuations of %d beams over %d tokens", count, width, V);
    const int rows = requests * width, slices = sel_slices(V);
    Q6K_REQUIRE(scratch_bytes >= q6k_beam_scratch(rows, V, count), "beam_select: %lld bytes of scratch, %lld are needed", scratch_bytes, q6k_beam_scratch(rows, V, count));
    float* best = (float*)scratch;
    int* at = (int*)(best + (size_t)rows * slices * count);
    SliceHead* heads = (SliceHead*)(at + (size_t)rows * slices * count);
    if (V % 4 == 0 && ((uintptr_t)logits & 15) == 0) q6k_launch(beam_slice_kernel<true>, dim3(slices, rows), SEL_THREADS, 0, st, logits, V, count, best, at, heads);
    else q6k_launch(beam_slice_kernel<false>, dim3(slices, rows), SEL_THREADS, 0, st, logits, V, count, best, at, heads);
    q6k_launch_as(true, beam_merge_kernel, requests, SEL_THREADS, 0, st, logits, scores, V, width, slices, count, best, at, heads, out_score, out_beam, out_token);
    return q6k_check_launch("beam_select");
}
