// The arrays of a step from the lengths of its requests, which need not be known on the host: request s has starts[s] tokens stored
// and brings counts[s]. Flat row cu[s] + i (cu: the sums of the counts before) is its token at position starts[s] + i, whose key goes to
// slot page * page_size + position % page_size of the page that the request's block table has for it. Rows behind the last
// request are position 0 of a request of their own (number `requests`) whose only page is pad_page.
// What is left out sets the status word, which keeps the larger of two codes: it does not depend on which block comes last.
// Pure data movement: every block adds up the counts before its request itself (they lie in L2), so one launch does it all.
#include "common.cuh"

namespace {

constexpr int SA_THREADS = 256;
constexpr int SA_TILE = 128;         // query rows of an attention tile

struct SaArgs {
    const int *starts, *counts;
    const int* state_slots;          // row of the tables of each request, or null: its number
    const int* tables;               // [groups, table_rows, width]
    const int* tokens;               // [requests, token_width] or null
    int* token_ids;                  // [rows] or null
    int *positions, *token_seq;      // [rows]
    int* cache_slots;                // [groups, rows]
    int* cu_seqlens;                 // [requests + 2]
    int *q_starts, *context_lens;    // [requests + 1]
    int4* tiles;                     // [requests * tiles_each]: request, first flat row, rows, first position
    int* block_tables;               // [groups, requests + 1, width]
    int* status;
    int requests, groups, table_rows, width, token_width, rows, max_count, tiles_each, page_size, pad_page;
};

// What request s brings: its count within the limits; none without a row of the tables or with a start that is no position.
__device__ __forceinline__ bool is_there(const SaArgs& a, int slot, int start) {
    return slot >= 0 && slot < a.table_rows && start >= 0 && start <= 0x7FFFFFFF - a.max_count;
}
__device__ __forceinline__ int brings(const SaArgs& a, int s, bool* cut) {
    const int slot = a.state_slots ? a.state_slots[s] : s, start = a.starts[s], count = a.counts[s];
    const int n = is_there(a, slot, start) ? min(max(count, 0), a.max_count) : 0;
    *cut = n != max(count, 0);
    return n;
}

__global__ void __launch_bounds__(SA_THREADS) step_arrays_kernel(SaArgs a) {
    __shared__ int sums[SA_THREADS / 32];
    ti_grid_launch_dependents();
    ti_grid_wait();
    const int s = blockIdx.y, tid = threadIdx.x, parts = gridDim.x, part = blockIdx.x;
    const bool pad = s == a.requests;
    const int slot = pad ? 0 : (a.state_slots ? a.state_slots[s] : s), given = pad ? 0 : a.starts[s];
    const bool there = pad || is_there(a, slot, given);
    const int start = there ? given : 0;
    bool cut = false;
    const int wanted = pad ? a.rows : brings(a, s, &cut);
    // the counts before this request; a sum that passes the rows stays there
    int before = 0;
    bool other;
#pragma unroll 4
    for (int i = tid; i < s; i += SA_THREADS) before = min(before + brings(a, i, &other), a.rows);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before = min(before + __shfl_xor_sync(~0u, before, o), a.rows);
    if ((tid & 31) == 0) sums[tid >> 5] = before;
    __syncthreads();
    before = 0;
#pragma unroll
    for (int w = 0; w < SA_THREADS / 32; ++w) before = min(before + sums[w], a.rows);
    const int n = min(wanted, a.rows - before);
    if (!pad && n < wanted) cut = true;
    const int context = pad ? 1 : start + n;
    if (part == 0) {
        if (tid == 0) {
            a.cu_seqlens[s] = before;
            if (pad) a.cu_seqlens[s + 1] = a.rows;
            a.q_starts[s] = start;
            a.context_lens[s] = context;
            if (cut && a.status) atomicMax(a.status, 5);
        }
        if (!pad)
            for (int i = tid; i < a.tiles_each; i += SA_THREADS) {
                const int off = min(i * SA_TILE, n);
                a.tiles[(size_t)s * a.tiles_each + i] = make_int4(s, before + off, min(n - off, SA_TILE), start + off);
            }
    }
    // the block tables: pages that the request holds, -1 behind them
    const int held = there ? (int)min((long long)a.width, ((long long)context + a.page_size - 1) / a.page_size) : 0;
    for (int g = 0; g < a.groups; ++g) {
        const int* table = a.tables + ((size_t)g * a.table_rows + slot) * a.width;
        int* to = a.block_tables + ((size_t)g * (a.requests + 1) + s) * a.width;
#pragma unroll 8
        for (int i = part * SA_THREADS + tid; i < a.width; i += parts * SA_THREADS) to[i] = i < held ? (pad ? a.pad_page : table[i]) : -1;
    }
    // the tokens
    for (int i = part * SA_THREADS + tid; i < n; i += parts * SA_THREADS) {
        const int row = before + i, pos = pad ? 0 : start + i;
        if (a.token_ids) a.token_ids[row] = pad ? 0 : a.tokens[(size_t)s * a.token_width + i];
        a.positions[row] = pos;
        a.token_seq[row] = s;
        const int logical = pos / a.page_size;
        for (int g = 0; g < a.groups; ++g) {
            const int page = pad ? -1 : (logical < a.width ? a.tables[((size_t)g * a.table_rows + slot) * a.width + logical] : -1);
            const long long at = (long long)page * a.page_size + pos % a.page_size;
            const bool ok = page >= 0 && at <= 0x7FFFFFFFll;
            a.cache_slots[(size_t)g * a.rows + row] = ok ? (int)at : -1;
            if (!ok && !pad && a.status) atomicMax(a.status, 1);      // a token without a page
        }
    }
}

}  // namespace

TI_API int ti_step_arrays(int* token_ids, int* positions, int* token_seq, int* cache_slots, int* cu_seqlens, int* q_starts, int* context_lens,
                          int* tiles, int* block_tables, const int* starts, const int* counts, const int* state_slots, const int* tables,
                          const int* tokens, int* status, int requests, int groups, int table_rows, int width, int token_width, int rows,
                          int max_count, int page_size, int pad_page, cudaStream_t stream) {
    TI_REQUIRE(requests >= 0 && requests < 65535 && groups >= 1 && table_rows >= 0 && width >= 1 && rows >= 0 && max_count >= 1 && page_size >= 1,
               "step_arrays: bad sizes");
    TI_REQUIRE(rows < (1 << 30) && max_count < (1 << 30), "step_arrays: fewer than 2^30 rows");     // two of them add up to less than 2^31
    // (an array without entries may have no address: without requests nothing is read from tokens, without rows nothing is written)
    TI_REQUIRE(requests == 0 || rows == 0 || (token_ids == nullptr) == (tokens == nullptr), "step_arrays: token_ids and tokens go together");
    TI_REQUIRE(!tokens || token_width >= max_count, "step_arrays: tokens narrower than max_count");
    SaArgs a{starts, counts, state_slots, tables, tokens, token_ids, positions, token_seq, cache_slots, cu_seqlens, q_starts, context_lens,
             (int4*)tiles, block_tables, status, requests, groups, table_rows, width, token_width, rows, max_count,
             (max_count + SA_TILE - 1) / SA_TILE, page_size, pad_page};
    // blocks a request: as many as keep a thread at four tokens and sixteen words of each table
    const int parts = max(1, min(64, max((max_count + 4 * SA_THREADS - 1) / (4 * SA_THREADS), (width + 16 * SA_THREADS - 1) / (16 * SA_THREADS))));
    ti_launch(step_arrays_kernel, dim3(parts, requests + 1), SA_THREADS, 0, stream, a);
    TI_CHECK_LAUNCH("step_arrays");
    return 0;
}
