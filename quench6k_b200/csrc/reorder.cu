// Beams that go on from one another: row r of a group of `width` rows takes over what row parent[r] of its group holds, all rows
// at once (a row may be the parent of others and have another parent itself).  Two forms of what a row holds: positions of paged
// tensors, reached through a block table, and slots of fixed-size states.
//
// A thread owns one place (16 bytes of a position's row, or of a state) in all rows of a group: it reads the parents' values
// for every row that moves, and writes them after the last read.  So no second copy is needed whatever the parents are,
// and nothing is synchronised.  All tensors of a call are handled by one launch.
#include "common.cuh"

namespace {

constexpr int RE_TENSORS = 128, RE_MAX_WIDTH = 32, RE_THREADS = 256, RE_PIECE = 4096;

struct PageTensors {                       // [heads, pages, page_size, a row of row_bytes]
    char* base[RE_TENSORS];
    int heads[RE_TENSORS], pages[RE_TENSORS], row_bytes[RE_TENSORS];
};
struct SlotTensors {                       // [slots, slot_bytes]
    char* base[RE_TENSORS];
    long long bytes[RE_TENSORS];
    int slots[RE_TENSORS];
};

// The group's parents; a parent outside the group counts as the row itself, which stays.
__device__ __forceinline__ int parent_of(const int* parents, int group, int width, int b) {
    const int p = parents[group * width + b];
    return (unsigned)p < (unsigned)width ? p : b;
}

// A warp works on a piece of up to RE_PIECE bytes of one head's part of one page, in all rows of a group: there the positions lie one after the other,
// so that which bytes a row takes over are two numbers.  grid (blocks along the pieces, tensors, groups); V: what a lane moves at a time; W: the most rows
// of a group; U: places that a lane has under way at once.
// (A thread for each place, which found its page and row by divisions of its own, held 150 registers: 163 us for 262 MB where this takes 60.)
// What a row's pointers, bounds and values take in registers shows in wide groups: with 16 bytes at a time, 8 rows spill 156 bytes under the 80 registers
// that let three blocks run, 16 take 248 registers and one block an SM, 32 spill 860 bytes.  1,024 positions in 48 tensors, half of the rows moving,
// 805 MB (123 us at the copy's rate): groups of four 133 us, of eight 153, of sixteen 163; of 32 (512 positions) 182.  Three rows of five, 1,007 MB, 351 (154 at
// the copy's rate): few loads under way in the form for eight.
template <typename V, int W, int U>
__global__ void __launch_bounds__(RE_THREADS, W <= 8 ? 3 : 1) reorder_pages_kernel(const __grid_constant__ PageTensors t, const int* table, int blocks, int page_size, const int* parents,
                                                                   const int* first, const int* lengths, int width) {
    pdl_enter();
    __shared__ int par[RE_MAX_WIDTH], from[RE_MAX_WIDTH], to[RE_MAX_WIDTH];
    const int group = blockIdx.z, row0 = group * width, lane = threadIdx.x & 31;
    if (threadIdx.x < width) {
        const int b = threadIdx.x, p = parent_of(parents, group, width, b);
        par[b] = p, from[b] = max(first[row0 + b], 0), to[b] = p == b ? 0 : (int)min((long long)lengths[row0 + p], (long long)blocks * page_size);
    }
    __syncthreads();
    int lo = 0x7fffffff, hi = 0;
    for (int b = 0; b < width; ++b)
        if (from[b] < to[b]) lo = min(lo, from[b]), hi = max(hi, to[b]);
    if (lo >= hi) return;
    char* base = t.base[blockIdx.y];
    const unsigned heads = t.heads[blockIdx.y], pages = t.pages[blockIdx.y], row_bytes = t.row_bytes[blockIdx.y];
    const long long page_bytes = (long long)page_size * row_bytes;
    const unsigned per_page = (unsigned)((page_bytes + RE_PIECE - 1) / RE_PIECE);
    const int block0 = lo / page_size, block1 = (hi - 1) / page_size + 1;
    const long long pieces = (long long)(block1 - block0) * heads * per_page;
    for (long long piece = (long long)blockIdx.x * (RE_THREADS / 32) + (threadIdx.x >> 5); piece < pieces; piece += (long long)gridDim.x * (RE_THREADS / 32)) {
        const unsigned head = (unsigned)(piece / per_page % heads);
        const int block = block0 + (int)(piece / per_page / heads);
        const long long begin = piece % per_page * RE_PIECE, end = min(begin + RE_PIECE, page_bytes);
        // lane b: row b's pages here (its parent's and its own), and which bytes of the piece it takes over
        int src = -1, dst = -1, f = 0, e = 0;
        if (lane < width && from[lane] < to[lane]) {
            src = table[(size_t)(row0 + par[lane]) * blocks + block], dst = table[(size_t)(row0 + lane) * blocks + block];
            const long long at = (long long)block * page_size;
            f = (int)(min(max((from[lane] - at) * row_bytes, begin), end) - begin), e = (int)(min(max((to[lane] - at) * row_bytes, begin), end) - begin);
        }
        unsigned moving = __ballot_sync(0xffffffffu, (unsigned)src < pages && (unsigned)dst < pages && f < e);
        if (moving == 0) continue;
        const V* from_page[W];
        V* to_page[W];
        int f_of[W], e_of[W];
        const int n = __popc(moving);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const int b = moving ? __ffs(moving) - 1 : 0;
            moving &= moving - 1;
            char* at = base + head * (pages * page_bytes) + begin;
            from_page[k] = (const V*)(at + __shfl_sync(0xffffffffu, src, b) * page_bytes), to_page[k] = (V*)(at + __shfl_sync(0xffffffffu, dst, b) * page_bytes);
            f_of[k] = __shfl_sync(0xffffffffu, f, b), e_of[k] = k < n ? __shfl_sync(0xffffffffu, e, b) : 0;
        }
        const int vecs = (int)((end - begin) / (int)sizeof(V));
        for (int i0 = lane; i0 < vecs; i0 += 32 * U) {
            V held[U][W];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    const int i = i0 + 32 * u, at = i * (int)sizeof(V);
                    if (k < n && at >= f_of[k] && at < e_of[k]) held[u][k] = from_page[k][i];
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    const int i = i0 + 32 * u, at = i * (int)sizeof(V);
                    if (k < n && at >= f_of[k] && at < e_of[k]) to_page[k][i] = held[u][k];
                }
        }
    }
}

template <typename V, int W>
__global__ void __launch_bounds__(RE_THREADS) reorder_slots_kernel(const __grid_constant__ SlotTensors t, const int* slots, const int* parents, int width) {
    pdl_enter();
    __shared__ int par[RE_MAX_WIDTH], slot[RE_MAX_WIDTH];
    const int group = blockIdx.z;
    if (threadIdx.x < width) {
        const int b = threadIdx.x, s = slots[group * width + b];
        par[b] = parent_of(parents, group, width, b), slot[b] = (unsigned)s < (unsigned)t.slots[blockIdx.y] ? s : -1;
    }
    __syncthreads();
    char* base = t.base[blockIdx.y];
    const long long bytes = t.bytes[blockIdx.y], places = bytes / (long long)sizeof(V);
    for (long long i = (long long)blockIdx.x * RE_THREADS + threadIdx.x; i < places; i += (long long)gridDim.x * RE_THREADS) {
        V held[W];
        bool moves[W];
#pragma unroll
        for (int b = 0; b < W; ++b) {
            moves[b] = b < width && par[b] != b && slot[b] >= 0 && slot[par[b]] >= 0;
            if (moves[b]) held[b] = *(const V*)(base + slot[par[b]] * bytes + i * (long long)sizeof(V));
        }
#pragma unroll
        for (int b = 0; b < W; ++b)
            if (moves[b]) *(V*)(base + slot[b] * bytes + i * (long long)sizeof(V)) = held[b];
    }
}

// The widest of 16, 4 and 1 bytes that divides every address and size or'ed into `all`.
int vector_bytes(unsigned long long all) { return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1; }

template <typename V>
void launch_pages(const PageTensors& t, int n, int groups, int width, int blocks_x, const int* table, int blocks, int page_size, const int* parents, const int* first,
                  const int* lengths, cudaStream_t st) {
    const dim3 grid(blocks_x, n, groups);
#define GO(W_, U_) q6k_launch(reorder_pages_kernel<V, W_, U_>, grid, RE_THREADS, 0, st, t, table, blocks, page_size, parents, first, lengths, width)
    if (width <= 4) GO(4, 2);
    else if (width <= 8) GO(8, 1);
    else if (width <= 16) GO(16, 1);
    else GO(RE_MAX_WIDTH, 1);
#undef GO
}

template <typename V>
void launch_slots(const SlotTensors& t, int n, int groups, int width, int blocks_x, const int* slots, const int* parents, cudaStream_t st) {
    const dim3 grid(blocks_x, n, groups);
    if (width <= 4) q6k_launch(reorder_slots_kernel<V, 4>, grid, RE_THREADS, 0, st, t, slots, parents, width);
    else if (width <= 8) q6k_launch(reorder_slots_kernel<V, 8>, grid, RE_THREADS, 0, st, t, slots, parents, width);
    else if (width <= 16) q6k_launch(reorder_slots_kernel<V, 16>, grid, RE_THREADS, 0, st, t, slots, parents, width);
    else q6k_launch(reorder_slots_kernel<V, RE_MAX_WIDTH>, grid, RE_THREADS, 0, st, t, slots, parents, width);
}

}  // namespace

// bases, heads, pages, row_bytes: n tensors [heads, pages, page_size, row_bytes] on the host's side; table: int32 [groups * width, blocks];
// parents: int32 [groups, width]; first, lengths: int32 [groups * width].  Row r takes over positions first[r] .. lengths[parent] - 1.
Q6K_API int q6k_reorder_pages(int n, const long long* bases, const int* heads, const int* pages, const int* row_bytes, const int* table, int groups, int width,
                              int blocks, int page_size, const int* parents, const int* first, const int* lengths, cudaStream_t st) {
    if (n == 0 || groups == 0 || blocks == 0) return 0;
    Q6K_REQUIRE(n > 0 && n <= RE_TENSORS && groups > 0 && groups <= 65535 && width >= 1 && width <= RE_MAX_WIDTH && blocks > 0 && page_size > 0,
                "reorder_pages: %d tensors (at most %d), %d groups of %d rows (at most %d), %d blocks of %d", n, RE_TENSORS, groups, width, RE_MAX_WIDTH, blocks, page_size);
    PageTensors t;
    unsigned long long all = 0;
    long long most = 0;
    for (int i = 0; i < n; ++i) {
        Q6K_REQUIRE(heads[i] > 0 && pages[i] > 0 && row_bytes[i] > 0, "reorder_pages: tensor %d has %d heads, %d pages, rows of %d bytes", i, heads[i], pages[i], row_bytes[i]);
        t.base[i] = (char*)bases[i], t.heads[i] = heads[i], t.pages[i] = pages[i], t.row_bytes[i] = row_bytes[i];
        all |= (unsigned long long)bases[i] | (unsigned long long)row_bytes[i];
        const long long pieces = (long long)blocks * heads[i] * (((long long)page_size * row_bytes[i] + RE_PIECE - 1) / RE_PIECE);
        if (pieces > most) most = pieces;
    }
    const int vb = vector_bytes(all);
    // Enough blocks for every piece of the table, and no more than some eight to an SM in all (three run at a time): first and lengths lie in device memory and
    // the call says nothing else of how many positions move, and a block without any costs its start (48 tensors, eight requests of four beams, 21
    // positions of 1,789: 12.7 us with sixteen, 9.7 with eight, 7.8 with four; but all of 4,096 positions of two requests: 197, 199 and 214 us).
    const long long want = (most + RE_THREADS / 32 - 1) / (RE_THREADS / 32), cap = (148 * 8 + (long long)n * groups - 1) / ((long long)n * groups);
    const int bx = (int)(want < cap ? want : cap);
    if (vb == 16) launch_pages<uint4>(t, n, groups, width, bx, table, blocks, page_size, parents, first, lengths, st);
    else if (vb == 4) launch_pages<uint32_t>(t, n, groups, width, bx, table, blocks, page_size, parents, first, lengths, st);
    else launch_pages<uint8_t>(t, n, groups, width, bx, table, blocks, page_size, parents, first, lengths, st);
    return q6k_check_launch("reorder_pages");
}

// bases, slots, bytes: n tensors [slots, bytes]; slot_ids: int32 [groups * width]; parents: int32 [groups, width].
Q6K_API int q6k_reorder_slots(int n, const long long* bases, const int* slots, const long long* bytes, const int* slot_ids, int groups, int width, const int* parents,
                              cudaStream_t st) {
    if (n == 0 || groups == 0) return 0;
    Q6K_REQUIRE(n > 0 && n <= RE_TENSORS && groups > 0 && groups <= 65535 && width >= 1 && width <= RE_MAX_WIDTH,
                "reorder_slots: %d tensors (at most %d), %d groups of %d rows (at most %d)", n, RE_TENSORS, groups, width, RE_MAX_WIDTH);
    SlotTensors t;
    unsigned long long all = 0;
    long long most = 0;
    for (int i = 0; i < n; ++i) {
        Q6K_REQUIRE(slots[i] > 0 && bytes[i] > 0, "reorder_slots: tensor %d has %d slots of %lld bytes", i, slots[i], bytes[i]);
        t.base[i] = (char*)bases[i], t.slots[i] = slots[i], t.bytes[i] = bytes[i];
        all |= (unsigned long long)bases[i] | (unsigned long long)bytes[i];
        if (bytes[i] > most) most = bytes[i];
    }
    const int vb = vector_bytes(all);
    const long long want = (most / vb + RE_THREADS - 1) / RE_THREADS, cap = (148 * 8 * 8 + (long long)n * groups - 1) / ((long long)n * groups);
    const int bx = (int)(want < cap ? want : cap);
    if (vb == 16) launch_slots<uint4>(t, n, groups, width, bx, slot_ids, parents, st);
    else if (vb == 4) launch_slots<uint32_t>(t, n, groups, width, bx, slot_ids, parents, st);
    else launch_slots<uint8_t>(t, n, groups, width, bx, slot_ids, parents, st);
    return q6k_check_launch("reorder_slots");
}
