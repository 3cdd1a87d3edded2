// Drafts from a request's own text. With h its tokens, n of them (the newly verified ones appended first), the length of the match
// that ends in front of place e (1 <= e < n) is l(e) = the largest l <= max_match with h[e-l .. e) = h[n-l .. n). The place with the
// longest match of at least min_match tokens is taken, of several the latest, and the text is drafted to go on as it did there:
// draft t = h[e + t mod (n - e)] (a repetition shorter than the drafts repeats). One comparison decides most places, so the kernel
// reads the text once and is bound by that.
#include "common.cuh"

namespace {

constexpr int NG_THREADS = 512;
constexpr int NG_MAX_MATCH = 32;

struct NgArgs {
    int* history;                    // [rows, room], row stride `room`
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

__global__ void __launch_bounds__(NG_THREADS) ngram_kernel(NgArgs a) {
    __shared__ unsigned long long best_sh[NG_THREADS / 32];
    __shared__ int last_sh[NG_MAX_MATCH];
    ti_grid_launch_dependents();
    ti_grid_wait();
    const int r = blockIdx.x, tid = threadIdx.x, D = a.max_drafts;
    int* out = a.tokens + (size_t)r * (D + 1);
    const int row = a.state_slots ? a.state_slots[r] : r;
    const int held = a.lengths[r];
    const int brought = a.new_tokens ? min(max(a.new_counts[r], 0), a.new_width) : 0;
    const bool known = row >= 0 && row < a.rows && held >= 0 && held <= a.room;
    const bool fits = known && brought <= a.room - held;
    if (tid == 0 && !fits && a.status) atomicExch(a.status, 6);       // a text without a row, or longer than its row
    int* h = a.history + (size_t)(known ? row : 0) * a.room;
    const int n = fits ? held + brought : (known ? held : 0);
    if (fits && tid < brought) h[held + tid] = a.new_tokens[(size_t)r * a.new_width + tid];
    __syncthreads();
    unsigned long long best = 0;
    if (fits && n > 0) {
        if (tid < a.max_match) last_sh[tid] = n - 1 - tid >= 0 ? h[n - 1 - tid] : 0;
        __syncthreads();
        for (int e = 1 + tid; e < n; e += NG_THREADS) {
            int l = 0;
            while (l < a.max_match && l < e && h[e - 1 - l] == last_sh[l]) ++l;
            if (l >= a.min_match) {
                const unsigned long long key = ((unsigned long long)l << 32) | (unsigned)e;
                best = key > best ? key : best;
            }
        }
    }
    best = warp_max64(best);
    if ((tid & 31) == 0) best_sh[tid >> 5] = best;
    __syncthreads();
    if (tid < 32) {
        best = warp_max64(tid < NG_THREADS / 32 ? best_sh[tid] : 0ull);
        const int e = (int)(best & 0xFFFFFFFFull);
        const bool there = fits && n > 0;
        const int most = a.limits ? min(max(a.limits[r], 0), D) : D;
        const int drafts = there && best ? most : 0;
        for (int t = tid; t <= D; t += 32) out[t] = t == 0 ? (there ? h[n - 1] : -1) : (t <= drafts ? h[e + (t - 1) % (n - e)] : -1);
        if (tid == 0) {
            a.counts[r] = there ? 1 + drafts : 0;
            a.starts[r] = there ? n - 1 : 0;
            a.lengths_out[r] = n;
        }
    }
}

}  // namespace

TI_API int ti_ngram_drafts(int* tokens, int* counts, int* starts, int* lengths_out, int* history, const int* lengths, const int* state_slots,
                           const int* new_tokens, const int* new_counts, const int* limits, int* status, int requests, int rows, int room,
                           int new_width, int max_drafts, int min_match, int max_match, cudaStream_t stream) {
    TI_REQUIRE(requests >= 0 && requests <= 65535 && rows >= 0 && room >= 0 && max_drafts >= 0 && new_width >= 0 && new_width <= NG_THREADS,
               "ngram_drafts: bad sizes");
    TI_REQUIRE(min_match >= 1 && max_match >= min_match && max_match <= NG_MAX_MATCH, "ngram_drafts: matches of 1 to %d tokens", NG_MAX_MATCH);
    if (requests == 0) return 0;
    NgArgs a{history, lengths, state_slots, new_tokens, new_counts, limits, tokens, counts, starts, lengths_out, status,
             requests, rows, room, new_width, max_drafts, min_match, max_match};
    ti_launch(ngram_kernel, requests, NG_THREADS, 0, stream, a);
    TI_CHECK_LAUNCH("ngram_drafts");
    return 0;
}
