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
    for (int w = 0; w < SEL_THREADS / 32; ++w) t += red[w];
    return t;
}

// grid (slices, rows).  best/at: [rows, slices, count]; head: [rows, slices] of {maximum, sum, how many}.
struct SliceHead {
    float most, sum;
    int found;
};

__global__ void __launch_bounds__(SEL_THREADS) beam_slice_kernel(const float* logits, int V, int count, float* best, int* at, SliceHead* heads) {
    pdl_enter();
    __shared__ int red[SEL_THREADS / 32];
    __shared__ float redf[32];
    __shared__ int taken;
    const float* row = logits + (size_t)blockIdx.y * V;
    const int lo = blockIdx.x * SEL_SLICE, n = min(V - lo, SEL_SLICE);
    const size_t slot = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    float v[SEL_EACH];
    float most = -INFINITY;
    bool bad = false;                                        // a value that makes the row's sum not finite
#pragma unroll
    for (int j = 0; j < SEL_EACH; ++j) {
        const int i = j * SEL_THREADS + threadIdx.x;
        v[j] = i < n ? row[lo + i] : -INFINITY;
        most = fmaxf(most, v[j]);
        bad |= !(v[j] < INFINITY);
    }
    most = warp_max(most);
    if ((threadIdx.x & 31) == 0) redf[threadIdx.x >> 5] = most;
    if (threadIdx.x == 0) taken = 0;
    const bool any_bad = __syncthreads_or(bad);
#pragma unroll
    for (int w = 0; w < SEL_THREADS / 32; ++w) most = fmaxf(most, redf[w]);
    float sum = 0.0f;
    if (most > -INFINITY && !any_bad) {
#pragma unroll
        for (int j = 0; j < SEL_EACH; ++j) sum += expf(v[j] - most);
    }
    sum = block_sum(sum, redf);
    // the count-th largest (logit, lowest place) of the slice, bit by bit
    int finite = 0;
#pragma unroll
    for (int j = 0; j < SEL_EACH; ++j) finite += finite_key(v[j]) != 0u;
    finite = block_count(finite, red);
    const int want = min(count, finite);
    if (threadIdx.x == 0) heads[slot] = SliceHead{most, any_bad ? NAN : sum, any_bad ? 0 : want};
    if (want == 0 || any_bad) return;
    unsigned kth = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const unsigned trial = kth | (1u << bit);
        int c = 0;
#pragma unroll
        for (int j = 0; j < SEL_EACH; ++j) c += finite_key(v[j]) >= trial;
        if (block_count(c, red) >= want) kth = trial;
    }
    int above = 0;
#pragma unroll
    for (int j = 0; j < SEL_EACH; ++j) above += finite_key(v[j]) > kth;
    above = block_count(above, red);
    int last = 0;                                            // of the logits equal to it, those at places below `last` are taken
    for (int step = SEL_SLICE; step > 0; step >>= 1) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < SEL_EACH; ++j) c += finite_key(v[j]) == kth && j * SEL_THREADS + (int)threadIdx.x < last + step;
        if (block_count(c, red) <= want - above) last += step;
    }
#pragma unroll
    for (int j = 0; j < SEL_EACH; ++j) {
        const unsigned k = finite_key(v[j]);
        const int i = j * SEL_THREADS + threadIdx.x;
        if (k > kth || (k == kth && i < last)) {
            const int to = atomicAdd(&taken, 1);
            if (to < want) best[slot * count + to] = v[j], at[slot * count + to] = lo + i;
        }
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
    __shared__ unsigned long long key[SEL_MAX_COUNT];
    __shared__ int place[SEL_MAX_COUNT];
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
    int c = 0;
    for (int i = threadIdx.x; i < all; i += SEL_THREADS) {
        unsigned long long k;
        int w;
        c += candidate(i, k, w);
    }
    const int want = min(count, block_count(c, red));
    unsigned long long kth = 0;
    int last = 0;
    if (want > 0) {
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long trial = kth | (1ull << bit);
            c = 0;
            for (int i = threadIdx.x; i < all; i += SEL_THREADS) {
                unsigned long long k;
                int w;
                c += candidate(i, k, w) && k >= trial;
            }
            if (block_count(c, red) >= want) kth = trial;
        }
        int above = 0;
        for (int i = threadIdx.x; i < all; i += SEL_THREADS) {
            unsigned long long k;
            int w;
            above += candidate(i, k, w) && k > kth;
        }
        above = block_count(above, red);
        for (int step = 1 << 30; step > 0; step >>= 1) {
            c = 0;
            for (int i = threadIdx.x; i < all; i += SEL_THREADS) {
                unsigned long long k;
                int w;
                c += candidate(i, k, w) && k == kth && w < last + step;
            }
            if (block_count(c, red) <= want - above) last += step;
        }
        for (int i = threadIdx.x; i < all; i += SEL_THREADS) {
            unsigned long long k;
            int w;
            if (candidate(i, k, w) && (k > kth || (k == kth && w < last))) {
                const int to = atomicAdd(&taken, 1);
                if (to < want) key[to] = k, place[to] = w;
            }
        }
    }
    __syncthreads();
    out_score += (size_t)blockIdx.x * count, out_beam += (size_t)blockIdx.x * count, out_token += (size_t)blockIdx.x * count;
    for (int i = threadIdx.x; i < want; i += SEL_THREADS) {
        int rank = 0;
        for (int j = 0; j < want; ++j) rank += key[j] > key[i] || (key[j] == key[i] && place[j] < place[i]);
        const unsigned long long u = key[i];
        out_score[rank] = (float)__longlong_as_double((long long)((u >> 63) ? u & ~(1ull << 63) : ~u));
        out_beam[rank] = place[i] / V, out_token[rank] = place[i] % V;
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
    q6k_launch(beam_slice_kernel, dim3(slices, rows), SEL_THREADS, 0, st, logits, V, count, best, at, heads);
    q6k_launch(beam_merge_kernel, requests, SEL_THREADS, 0, st, logits, scores, V, width, slices, count, best, at, heads, out_score, out_beam, out_token);
    return q6k_check_launch("beam_select");
}
