// Drafts from a request's own text. With h its tokens, n of them (the newly verified ones appended first), the length of the match
// that ends in front of place e (1 <= e < n) is l(e) = the largest l <= max_match with h[e-l .. e) = h[n-l .. n). The place with the
// longest match of at least min_match tokens is taken, of several the latest, and the text is drafted to go on as it did there:
// draft t = h[e + t mod (n - e)] (a repetition shorter than the drafts repeats). One comparison decides most places, so the kernel
// reads the text once, 16 bytes a lane and four loads in flight, and is bound by that (256 texts of 131,071 tokens: 134 MB in 25.3 us, 81 % of
// the copy rate) or, short, by the chain length - last tokens - comparison; a long text is shared out over a cluster of blocks, whose best
// places (longest, then latest: the larger of two 64-bit numbers, in any order) meet in the first one's shared memory.
#include <cooperative_groups.h>

#include "draws.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int NG_THREADS = 256;
constexpr int NG_WARPS = NG_THREADS / 32;
constexpr int NG_MAX_MATCH = 32;
constexpr int NG_MAX_NEW = 512;
constexpr int NG_CTAS = 8;           // most blocks of a text
constexpr int NG_LEAST = 4096;       // tokens that a block of several has at least
constexpr int NG_LOADS = 4;

struct NgArgs {
    int* history;                    // [rows, room]
    const int* lengths;              // per request
    const int* state_slots;          // row of the history of each request, or null: its number
    const int* new_tokens;           // [requests, new_width] or null
    const int* new_counts;
    const int* limits;               // most drafts of each request, or null
    int* tokens;                     // [requests, max_drafts + 1]
    int *counts, *starts, *lengths_out;
    int* status;
    int requests, rows, room, new_width, max_drafts, min_match, max_match;
};

__device__ __forceinline__ unsigned long long warp_max64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long w = __shfl_xor_sync(~0u, v, o);
        v = w > v ? w : v;
    }
    return v;
}

__global__ void __launch_bounds__(NG_THREADS, 8) ngram_kernel(NgArgs a) {
    __shared__ unsigned long long best_sh[NG_WARPS], part_sh[NG_CTAS];
    __shared__ int last_sh[NG_MAX_MATCH];
    ti_grid_launch_dependents();
    if (gridDim.x > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    ti_grid_wait();
    const int r = blockIdx.y, rank = blockIdx.x, ctas = gridDim.x, tid = threadIdx.x, D = a.max_drafts;
    const int row = a.state_slots ? a.state_slots[r] : r;
    const int held = a.lengths[r];
    const int brought = a.new_tokens ? min(max(a.new_counts[r], 0), a.new_width) : 0;
    const bool known = row >= 0 && row < a.rows && held >= 0 && held <= a.room;
    const bool fits = known && brought <= a.room - held;
    int* h = a.history + (size_t)(known ? row : 0) * a.room;
    const int* fresh = a.new_tokens + (size_t)r * a.new_width;
    const int n = fits ? held + brought : (known ? held : 0);
    const bool there = fits && n > 0;
    auto token = [&](int i) { return i < held ? h[i] : fresh[i - held]; };        // nobody waits for the new ones to be written
    // tokens 0 .. end - 1 as they lie; group g has those from 4 g - shift on. What is wanted of the first groups is under way before it
    // is known what they are compared with.
    const int end = there ? min(held, n - 1) : 0, shift = (int)(((uintptr_t)h >> 2) & 3), groups = (end + shift + 3) >> 2;
    int4 v[NG_LOADS];
    auto load = [&](int first) {
#pragma unroll
        for (int k = 0; k < NG_LOADS; ++k) {
            const int g = first + k * NG_THREADS, i = 4 * g - shift;
            if (i >= 0 && i + 3 < end) {
                v[k] = *reinterpret_cast<const int4*>(h + i);
            } else {                                         // the text's ends, and behind them
                v[k].x = i >= 0 && i < end ? h[i] : 0;
                v[k].y = i + 1 >= 0 && i + 1 < end ? h[i + 1] : 0;
                v[k].z = i + 2 >= 0 && i + 2 < end ? h[i + 2] : 0;
                v[k].w = i + 3 >= 0 && i + 3 < end ? h[i + 3] : 0;
            }
        }
    };
    int first = rank * NG_LOADS * NG_THREADS + tid;
    load(first);
    if (there && tid < a.max_match && tid < n) last_sh[tid] = token(n - 1 - tid);
    __syncthreads();
    unsigned long long best = 0;
    if (there) {
        const int last = last_sh[0];
        auto look = [&](int i, int value) {                  // the match that ends with token i
            if (value != last || i < 0 || i >= n - 1) return;
            int l = 1;
            while (l < a.max_match && l <= i && token(i - l) == last_sh[l]) ++l;
            const unsigned long long key = ((unsigned long long)l << 32) | (unsigned)(i + 1);
            if (l >= a.min_match && key > best) best = key;
        };
        while (true) {
#pragma unroll
            for (int k = 0; k < NG_LOADS; ++k) {
                const int i = 4 * (first + k * NG_THREADS) - shift;
                if (i >= end || (v[k].x != last && v[k].y != last && v[k].z != last && v[k].w != last)) continue;
                const int token4[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (i + q < end) look(i + q, token4[q]);
            }
            first += ctas * NG_LOADS * NG_THREADS;
            if (first >= groups) break;
            load(first);
        }
        if (rank == 0)                                       // the new ones but the last
            for (int i = held + tid; i < n - 1; i += NG_THREADS) look(i, token(i));
    }
    best = warp_max64(best);
    if ((tid & 31) == 0) best_sh[tid >> 5] = best;
    __syncthreads();
    best = warp_max64((tid & 31) < NG_WARPS ? best_sh[tid & 31] : 0ull);
    if (ctas > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");           // every block runs
        if (tid == 0) *cluster.map_shared_rank(&part_sh[rank], 0) = best;
        cluster.sync();
        if (rank != 0) return;
        best = warp_max64((tid & 31) < ctas ? part_sh[tid & 31] : 0ull);
    }
    const int e = (int)(best & 0xFFFFFFFFull);
    const int most = a.limits ? min(max(a.limits[r], 0), D) : D;
    const int drafts = there && best ? most : 0;
    if (tid <= D) a.tokens[(size_t)r * (D + 1) + tid] = tid == 0 ? (there ? last_sh[0] : -1) : (tid <= drafts ? token(e + (tid - 1) % (n - e)) : -1);
    if (tid == 0) {
        a.counts[r] = there ? 1 + drafts : 0;
        a.starts[r] = there ? n - 1 : 0;
        a.lengths_out[r] = n;
        if (!fits && a.status) atomicExch(a.status, 6);      // a text without a row, or longer than its row
    }
    if (fits)
        for (int i = tid; i < brought; i += NG_THREADS) h[held + i] = fresh[i];
}

}  // namespace

TI_API int ti_ngram_drafts(int* tokens, int* counts, int* starts, int* lengths_out, int* history, const int* lengths, const int* state_slots,
                           const int* new_tokens, const int* new_counts, const int* limits, int* status, int requests, int rows, int room,
                           int new_width, int max_drafts, int min_match, int max_match, cudaStream_t stream) {
    TI_REQUIRE(requests >= 0 && requests <= 65535 && rows >= 0 && room >= 0 && room <= (1 << 30) && new_width >= 0 && new_width <= NG_MAX_NEW, "ngram_drafts: bad sizes");
    TI_REQUIRE(max_drafts >= 0 && max_drafts < NG_THREADS, "ngram_drafts: at most %d drafts", NG_THREADS - 1);
    TI_REQUIRE(min_match >= 1 && max_match >= min_match && max_match <= NG_MAX_MATCH, "ngram_drafts: matches of 1 to %d tokens", NG_MAX_MATCH);
    if (requests == 0) return 0;
    NgArgs a{history, lengths, state_slots, new_tokens, new_counts, limits, tokens, counts, starts, lengths_out, status,
             requests, rows, room, new_width, max_drafts, min_match, max_match};
    // Blocks of a text: until the machine has six on every SM. 256 texts of 131,071 tokens: 4 blocks each 25.3 us, 8 27.1, 2 34.3 (with eight
    // loads in flight a thread, and so five blocks an SM: 29.0, 31.0, 27.7).
    int ctas = 1;
    while (ctas < NG_CTAS && ctas * NG_LEAST < room && ctas * requests < 148 * 6) ctas *= 2;
    ti_launch_clusters(ngram_kernel, dim3(ctas, requests), ctas, NG_THREADS, 0, stream, a);
    TI_CHECK_LAUNCH("ngram_drafts");
    return 0;
}
