// Verification of drafted tokens. A request brings rows of logits: row j says what follows the j-th token it was fed, and that
// token's successor among the fed ones is the draft d_j that row j judges; behind the last draft one row more.
//   s_i = x_i / T (a float32 division); kept: s_i at or above the k-th largest, neither NaN nor -inf;
//   p_i = exp(s_i - max s) / sum over the kept; q_i the same from the draft model's logits, or 1 at the draft without any.
// Drafts that come with the draft model's logits were drawn, and are judged by the ratio of the probabilities (rejection sampling):
//   a_j = min(1, p(d_j) / q(d_j)); draft j holds if u_j < a_j and all before it did; u_j is word 0 of the Philox block
//   (0, step + j, stream, 1) under the request's seed. The token behind comes from the row J behind the last draft that held: if all
//   held, argmax of s_i + G_i, what ti_sample draws from the row at step + J; if one failed, argmax of max(p_i - q_i, 0) / E_i,
//   E_i = -log U_i: an exponential race, token i wins with probability proportional to its numerator. Its noise is apart from
//   ti_sample's (fourth counter 2 for 0), which the draft may have been drawn with.
// Drafts without (looked up, or a draft model's argmax) are certain: whichever token the row's own draw gives, the draft holds if
//   it is that one. That is as likely as rejection sampling makes it, p(d), and the tokens are those of decoding one by one.
// Greedy requests draw the first largest logit.
// Sums and exponentials are float32 (the sum over a top-k row's few candidates is taken in fixed point, so that the order in which
// they were found does not show). The threshold and the draws go by the float32 quotients s; the weights of a row without a threshold go
// by x - max x, which comes closer to the softmax of x / T where logits or reciprocal temperatures are large.
//
// Bound by reading the logits once. Three kernels (two where every request is greedy):
//   parts_kernel   streams every row, 32 logits a thread in registers, and leaves of each warp's part the largest, the sum and the best
//                  draw, or of a top-k row the largest of every 32 neighbouring logits. No block waits for another: 64 x 4 rows of
//                  151,936 and as many of the draft model, less 64, 53 us = 6.6 TB/s; 64 x 7 open ones 86 us = 6.8 TB/s.
//   rows_kernel    a block a row. Of a top-k row: at least k of the row's lines of 32 reach a value close to the k-th largest of its lines'
//                  largest, which bounds the row's k-th largest from below; so the row's top k are in the few lines (some 110 for k = 100)
//                  that reach it, and those are read again and ranked. A chain of short steps on one block: 9 us for one row, 14 for 576.
//   verify_kernel  decides the request (1 to 2 us); behind a drawn draft that failed, clusters of blocks scan the two rows once more
//                  (64 requests of 151,936 tokens: 33 us, bound by the Philox words and exponentials of the tokens).
// A row held by a cluster of 16 blocks in shared memory, threshold and sum found there, read the logits once too, but spent 13 us of a
// block on meeting the others (a cluster's barrier 0.9 us) where its loads took 1.3: 291 us for the first of these cases.
#include <cooperative_groups.h>

#include <algorithm>

#include "draws.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int VD_MAX_DRAFTS = 31;    // a warp decides a request: a lane a draft, and one place more
constexpr int VD_THREADS = 256;
constexpr int VD_WARPS = VD_THREADS / 32;
constexpr int VD_GROUPS = 8;         // groups of four logits a thread holds
constexpr int VD_TILE = VD_THREADS * VD_GROUPS * 4;
constexpr int VD_LINE = 32;          // neighbouring logits that a top-k row's largest are taken of
constexpr int VD_CANDIDATES = 2048;  // of a top-k row, in shared memory
constexpr int VD_MAX_VOCAB = 1 << 19;        // so many weights of at most 2^44 fit 64 bits
constexpr int VD_LIST = 1024;        // of what the threshold keeps, for the draw behind a draft that failed
constexpr int VD_CTAS = 8, VD_MOST_CTAS = 16;         // blocks that share such a draw
constexpr int VD_STAGES = 3;         // groups of four tokens on their way to a thread there
constexpr float LOG2E = 1.4426950408889634f;

// A warp's part of a row: the largest logit, the sum of the weights relative to it, the best draw.
struct __align__(16) Part { float m, z, v; int i; };
// A row: the largest logit, the sum of the kept weights, the lowest kept key, the token that it draws (-1: none; of a
// sampled row that a draft model's logits judge: not drawn), the share of its draft, how many kept tokens are listed (-1: not).
struct __align__(16) RowStats { float m, z; unsigned threshold; int drawn; float share; int listed, unused[2]; };
struct __align__(8) Kept { float s; int i; };

struct VdArgs {
    const float* logits;             // [rows, vocab]
    const int* token_ids;            // [rows]
    const int* cu_rows;              // [requests + 1]
    const float* temperature;        // per request, or null with the others: every request is greedy
    const int *topk, *greedy;
    const long long* seed;
    const int *stream_id, *step;
    const float* draft_logits;       // element (r, j, i) at r * draft_request + j * draft_place + i, or null
    long long draft_request, draft_place;
    float* parts;                    // [requests, places, tiles, VD_THREADS]: lines' largest logits, or warps' Parts
    RowStats* stats;                 // [requests, places], where not all are greedy
    Kept* kept;                      // [requests, max_drafts, list]
    int* tokens;                     // [requests, max_drafts + 1]
    int* counts;
    float* accept;                   // [requests, max_drafts]
    int rows, vocab, requests, max_drafts, tiles, list;
    int places;                      // max_drafts + 1 rows of the target, then max_drafts of the draft model if there is one
};

// The request's rows: first flat row and how many (0 .. max_drafts + 1), inside the logits whatever cu_rows says.
__device__ __forceinline__ int2 rows_of(const VdArgs& a, int r) {
    const int lo = min(max(a.cu_rows[r], 0), a.rows), hi = min(max(a.cu_rows[r + 1], lo), a.rows);
    return make_int2(lo, min(hi - lo, a.max_drafts + 1));
}
__device__ __forceinline__ bool is_greedy(const VdArgs& a, int r) { return a.temperature == nullptr || a.greedy[r] != 0; }
__device__ __forceinline__ uint2 seed_of(const VdArgs& a, int r) {
    return make_uint2((unsigned)(a.seed[r] & 0xFFFFFFFFll), (unsigned)((unsigned long long)a.seed[r] >> 32));
}
// A place of a request: which of its rows (-1: none) and where it lies. draws: its token may be wanted as the row draws it.
struct Place { const float* x; int j; bool draws; };
__device__ __forceinline__ Place place_of(const VdArgs& a, int r, int place, int2 rows, bool greedy) {
    const bool of_draft = place > a.max_drafts;
    const int j = of_draft ? place - a.max_drafts - 1 : place;
    if (of_draft ? greedy || j >= rows.y - 1 : j >= rows.y) return Place{nullptr, -1, false};
    const float* x = of_draft ? a.draft_logits + r * a.draft_request + j * a.draft_place : a.logits + (size_t)(rows.x + j) * a.vocab;
    return Place{x, j, !greedy && !of_draft && (a.draft_logits == nullptr || j == rows.y - 1)};
}
__device__ __forceinline__ bool has_threshold(int topk, int vocab) { return topk > 0 && topk < vocab; }

__device__ __forceinline__ unsigned score_key(float s) { return order_key(s + 0.f); }        // -0 and +0 are one value

// 2^x, 2^-22 of itself off; nothing below 2^-126.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The weights of a row's logits by their distance from the largest, `most`: exp((v - most) / temp), which is 1 at the largest however far
// the logits lie from 0 (a mask's -1e10, a temperature near 0): an error in (v - most) c is one of the distance alone. Where a quotient
// is infinite, or the temperature's reciprocal 0 or nearly infinite, the quotients themselves are compared.
// `fast`, for many logits at once, is one multiply-add and one exponential, 2^(v c - m2) with m2 = most c rounded: that is 2^lost off,
// alike for all, and lost is an exact float32. At |m| < 2^20 (`near`) it is 0.09 at most; beyond, it may be anything (2^440 at -1e10).
constexpr float NEAR = 1048576.f;
struct Weights {
    float temp, most, m, c, m2;
    bool odd;
    __device__ __forceinline__ Weights(float temp_, float most_) : temp(temp_), most(most_), m(most_ / temp_), c(LOG2E / temp_), m2(most_ * c) {
        odd = !(fabsf(m) < INFINITY) || !(c > 0.f && c < 1e30f);
    }
    __device__ __forceinline__ bool near() const { return fabsf(m) < NEAR; }
    __device__ __forceinline__ float lost() const { return fmaf(most, c, -m2); }
    __device__ __forceinline__ float fast(float v) const { return ex2(fmaf(v, c, -m2)); }
    __device__ __forceinline__ float quotient(float v) const {
        const float s = v / temp;
        return !(s > -INFINITY) ? 0.f : (s == m ? 1.f : expf(s - m));
    }
    __device__ __forceinline__ float operator()(float v) const { return odd ? quotient(v) : ex2((v - most) * c); }
    // A factor on the weights that covers what they and a score s + G are off by, near 0: `lost`, 2^-24 of the scaled logits each for
    // two quotients and two sums, some steps of the functions; together below e^(4e-7 |m|) + 1e-4. (Farther off the quotients' own
    // roundings decide: equal ones are a tie, whatever their logits.)
    __device__ __forceinline__ float spare() const { return 1.001f + fabsf(m) * 1e-6f; }
};
// Whether s + G may reach a score: G is 16.7 at most, and the sum is rounded.
__device__ __forceinline__ bool may_reach(float s, float score) { return s > -INFINITY && s + fmaf(fabsf(s), 2.4e-7f, 17.f) >= score; }
// The same of a scaled logit at hand.
__device__ __forceinline__ float scaled_weight(float s, float m) { return !(s > -INFINITY) ? 0.f : (s == m ? 1.f : ex2((s - m) * LOG2E)); }

// Whether 1 - U < x * y may hold for the uniform number U of a word of the stream (never no where it does). 1 - U is 2 - 2^-24 - f, f the
// float in [1, 2) with the word's upper bits; so f + x y > 2 - 2^-24, which rounds to 2 at least, as the tie does.
__device__ __forceinline__ bool may_pass(unsigned word, float x, float y) { return fmaf(x, y, __uint_as_float(0x3F800000u | word >> 9)) >= 2.f; }

// s + G of a scaled logit s and its uniform number.
__device__ __forceinline__ float noisy(float s, float u) { return s - logf(-logf(u)); }

__device__ __forceinline__ Best warp_best(Best v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = better(v, Best{__shfl_xor_sync(~0u, v.v, o), __shfl_xor_sync(~0u, v.i, o)});
    return v;
}
__device__ __forceinline__ Best block_best(Best x, Best* sh) {
    x = warp_best(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = x;
    __syncthreads();
    return warp_best((threadIdx.x & 31) < VD_WARPS ? sh[threadIdx.x & 31] : Best{0.f, -1});
}

// A value that is below every logit whose quotient by temp reaches that of `bound`: quotients are rounded, by 2^-24 of themselves
// where they are normal numbers; elsewhere every logit may.
__device__ __forceinline__ float below_quotient(float bound, float temp) {
    const float s = fabsf(bound / temp);
    return s > 1e-35f && s < 1e37f ? bound - fabsf(bound) * 4.8e-7f : -INFINITY;
}

// Four neighbouring logits of a row; NaN behind its end. step: how many the row's place lets be read at once (rows off 16-byte
// boundaries: of an odd vocabulary, say). Which thread reads which logits goes by their number alone, and so does the order of sums.
__device__ __forceinline__ int row_step(const float* x) { return ((uintptr_t)x & 15) == 0 ? 4 : ((uintptr_t)x & 7) == 0 ? 2 : 1; }
__device__ __forceinline__ void load_four(const float* x, int e, int vocab, int step, float (&v)[4]) {
    if (step == 4 && e + 3 < vocab) {
        const float4 f = *reinterpret_cast<const float4*>(x + e);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else if (step == 2 && e + 3 < vocab) {
        const float2 f = *reinterpret_cast<const float2*>(x + e), g = *reinterpret_cast<const float2*>(x + e + 2);
        v[0] = f.x; v[1] = f.y; v[2] = g.x; v[3] = g.y;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = e + j < vocab ? x[e + j] : NAN;
    }
}

// f(logit, token) for all of a row, by the block; NaN for what lies behind it. Sixteen logits of a thread on their way at a time.
template <typename F>
__device__ __forceinline__ void each_of_row(const float* x, int vocab, int step, F f) {
#pragma unroll 1
    for (int first = 4 * (int)threadIdx.x; first < vocab; first += 16 * VD_THREADS) {
        float v[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) load_four(x, first + 4 * k * VD_THREADS, vocab, step, v[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q) f(v[k][q], first + 4 * k * VD_THREADS + q);
    }
}

// The tokens of thread t in a tile: a warp has 32 lines, a lane a group of four of every fourth.
__device__ __forceinline__ int token_of(int tile, int t, int k) { return tile * VD_TILE + (t >> 5) * (32 * VD_LINE) + 4 * (32 * k + (t & 31)); }

// DRAWS: open rows draw here, too (drafts that nothing judges: every row's token is wanted).
template <bool DRAWS>
__global__ void __launch_bounds__(VD_THREADS, DRAWS ? 4 : 5) parts_kernel(VdArgs a) {
    __shared__ float best_sh[VD_WARPS];
    ti_grid_launch_dependents();
    ti_grid_wait();
    const int tid = threadIdx.x, lane = tid & 31, r = blockIdx.z;
    const int2 rows = rows_of(a, r);
    const bool greedy = is_greedy(a, r);
    const Place at = place_of(a, r, blockIdx.y, rows, greedy);
    if (at.j < 0) return;
    const int step = row_step(at.x);
    float v[VD_GROUPS][4];
    if (step == 4 && token_of(blockIdx.x + 1, 0, 0) <= a.vocab) {
        const float4* from = reinterpret_cast<const float4*>(at.x + token_of(blockIdx.x, tid, 0));
#pragma unroll
        for (int k = 0; k < VD_GROUPS; ++k) {
            const float4 f = from[k * 32];
            v[k][0] = f.x; v[k][1] = f.y; v[k][2] = f.z; v[k][3] = f.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VD_GROUPS; ++k) load_four(at.x, token_of(blockIdx.x, tid, k), a.vocab, step, v[k]);
    }
    float* out = a.parts + (((size_t)r * a.places + blockIdx.y) * a.tiles + blockIdx.x) * VD_THREADS;
    Part* part = reinterpret_cast<Part*>(out) + (tid >> 5);

    if (greedy) {
        Best b{-INFINITY, -1};
#pragma unroll
        for (int k = 0; k < VD_GROUPS; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q)                      // a thread's tokens come in their order: the first of equals stays
                if (v[k][q] > b.v || (b.i < 0 && v[k][q] == v[k][q])) b = Best{v[k][q], token_of(blockIdx.x, tid, k) + q};
        b = warp_best(b);
        if (lane == 0) *part = Part{0.f, 0.f, b.v, b.i};
        return;
    }
#pragma unroll
    for (int k = 0; k < VD_GROUPS; ++k)
#pragma unroll
        for (int q = 0; q < 4; ++q) v[k][q] = fmaxf(v[k][q], -INFINITY);         // NaN, and what lies behind the row: -inf
    if (has_threshold(a.topk[r], a.vocab)) {
        // Eight neighbouring lanes share a line in each of their groups: after three exchanges, of four, two and one of the groups'
        // largest, each of the eight has one line's, group lane % 8's.
        float m[VD_GROUPS];
#pragma unroll
        for (int k = 0; k < VD_GROUPS; ++k) m[k] = fmaxf(fmaxf(v[k][0], v[k][1]), fmaxf(v[k][2], v[k][3]));
#pragma unroll
        for (int half = VD_GROUPS / 2; half > 0; half >>= 1) {
            const bool upper = lane & half;
#pragma unroll
            for (int k = 0; k < half; ++k) {
                const float other = __shfl_xor_sync(~0u, upper ? m[k] : m[k + half], half);
                m[k] = fmaxf(upper ? m[k + half] : m[k], other);
            }
        }
        out[(tid & ~31) + 4 * (lane & 7) + (lane >> 3)] = m[0];
        return;
    }
    float most = -INFINITY;
#pragma unroll
    for (int k = 0; k < VD_GROUPS; ++k) most = fmaxf(most, fmaxf(fmaxf(v[k][0], v[k][1]), fmaxf(v[k][2], v[k][3])));
    const float temp = a.temperature[r], largest = warp_max(most);
    Weights weight(temp, largest);
    const float m = weight.m;
    float z = 0.f;
    if (weight.odd) {
        if (m > -INFINITY) {
#pragma unroll 1
            for (int i = 0; i < 4 * VD_GROUPS; ++i) {
                const int e = token_of(blockIdx.x, tid, i >> 2) + (i & 3);
                if (e < a.vocab) z += weight.quotient(at.x[e]);
            }
        }
    } else {                                                 // from here on v is the weight
        if (!weight.near()) {                                // distances from the largest, which is 0 then
#pragma unroll
            for (int k = 0; k < VD_GROUPS; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q) v[k][q] -= largest;
            most -= largest;
            weight.most = weight.m2 = 0.f;
        }
#pragma unroll
        for (int k = 0; k < VD_GROUPS; ++k) {
#pragma unroll
            for (int q = 0; q < 4; ++q) v[k][q] = weight.fast(v[k][q]);
            z += (v[k][0] + v[k][1]) + (v[k][2] + v[k][3]);
        }
        z *= ex2(-weight.lost());
        most = weight.fast(most);
    }
    z = warp_sum(z);
    Best b{-INFINITY, -1};
    if (DRAWS) {
        // The largest of s + G, G = -log E, E = -log U. A token can pass a score B only if E < exp(s - B); E is 1 - U at least, and 1 - U
        // is exact: one comparison settles all but a few tokens once some B is known.
        const uint2 key2 = seed_of(a, r);
        const unsigned c1 = (unsigned)a.step[r] + (unsigned)at.j, stream = (unsigned)a.stream_id[r];
        float spare = 0.f, score = -INFINITY;                // exp(m - B), B
        // Beyond 2^29 a step of float32 is 64 and more: s + G is s, and the first of the largest quotients wins (a part behind a mask of
        // -1e9 ends here; 320 rows with all but 400 tokens at -1e9: 412 -> 52 us). Nothing wins where they are -inf.
        const bool silent = !(fabsf(m) <= 536870912.f);
        if (silent && m > -INFINITY) {
#pragma unroll 1
            for (int i = 0; i < 4 * VD_GROUPS && b.i < 0; ++i) {
                const int e = token_of(blockIdx.x, tid, i >> 2) + (i & 3);
                if (e < a.vocab && at.x[e] / temp == m) b = Best{m, e};
            }
        }
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {               // the threads' largest logits for a first B, then all
            unsigned left = 0u;
            if (silent) {                                    // b is the one
            } else if (half == 0) {
#pragma unroll
                for (int k = 0; k < VD_GROUPS; ++k)
#pragma unroll
                    for (int q = 0; q < 4; ++q) left = v[k][q] == most ? 1u << (4 * k + q) : left;
            } else if (weight.odd || !weight.near()) {       // by the quotients
#pragma unroll 1
                for (int i = 0; i < 4 * VD_GROUPS; ++i) {
                    const int e = token_of(blockIdx.x, tid, i >> 2) + (i & 3);
                    if (e < a.vocab && may_reach(at.x[e] / temp, score)) left |= 1u << i;
                }
            } else {
                // round by round for all groups: they share the key's bumps and what the first rounds make of the step and the stream
                // (320 open rows of 151,936 looked-up drafts 93 us; group by group 104)
                uint2 key = key2;
                asm volatile("" : "+r"(key.x), "+r"(key.y));             // bumped here, not ahead: that would take twenty registers
                uint4 w[VD_GROUPS];
#pragma unroll
                for (int k = 0; k < VD_GROUPS; ++k) w[k] = make_uint4((unsigned)token_of(blockIdx.x, tid, k) >> 2, c1, stream, 0u);
#pragma unroll
                for (int round = 0; round < 10; ++round) {
#pragma unroll
                    for (int k = 0; k < VD_GROUPS; ++k) w[k] = philox_round(w[k], key);
                    key.x += 0x9E3779B9u;
                    key.y += 0xBB67AE85u;
                }
#pragma unroll
                for (int k = 0; k < VD_GROUPS; ++k) {
                    const unsigned words[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        left |= may_pass(words[q], v[k][q], spare) ? 1u << (4 * k + q) : 0u;
                }
            }
            if (half == 0 && !(most > (weight.odd ? -INFINITY : 0.f))) left = 0u;       // (a weight of nothing is beaten by the largest)
            for (; left; left &= left - 1u) {                // (their numbers once more: the register file has no subscripts)
                const int bit = __ffs(left) - 1, i = token_of(blockIdx.x, tid, bit >> 2) + (bit & 3);
                const uint4 w = philox4x32_10(make_uint4((unsigned)i >> 2, c1, stream, 0u), key2);
                const float s = at.x[i] / temp;              // (-inf, too, of a finite logit at a temperature below 1)
                if (s > -INFINITY) b = better(b, Best{noisy(s, philox_uniform(word_of(w, i))), i});
            }
            if (half == 0) {                                 // the best that any warp of the block has found
                const float own = warp_max(b.i < 0 ? -INFINITY : b.v);
                if (lane == 0) best_sh[tid >> 5] = own;
                __syncthreads();
                score = warp_max(best_sh[lane & (VD_WARPS - 1)]);
                spare = ex2((m - score) * LOG2E) * weight.spare();
            }
        }
        b = warp_best(b);
    }
    if (lane == 0) *part = Part{largest, z, b.v, b.i};
}

// What a warp's parts of a row come to: all of it for the row's warp.
__device__ __forceinline__ RowStats whole_row(const VdArgs& a, const Place& at, size_t slot, bool greedy, float temp, int drafted) {
    const int lane = threadIdx.x & 31, n = a.tiles * VD_WARPS;
    const Part* part = reinterpret_cast<const Part*>(a.parts + slot * a.tiles * VD_THREADS);
    auto nth = [&](int i) { return part[(i / VD_WARPS) * (VD_THREADS / 4) + i % VD_WARPS]; };
    RowStats st{-INFINITY, 0.f, 0u, -1, 0.f, -1, {0, 0}};
    const float at_draft = !greedy && drafted >= 0 && drafted < a.vocab ? at.x[drafted] : NAN;
    Best b{0.f, -1};
    float z = 0.f;
    const float c = LOG2E / temp;
    for (int first = lane; first < n; first += 5 * 32) {     // five loads in flight
        Part p[5];
#pragma unroll
        for (int k = 0; k < 5; ++k) p[k] = first + 32 * k < n ? nth(first + 32 * k) : Part{-INFINITY, 0.f, 0.f, -1};
#pragma unroll
        for (int k = 0; k < 5; ++k) {
            b = better(b, Best{p[k].v, p[k].i});
            if (!greedy && p[k].z > 0.f) {
                if (p[k].m > st.m) { z *= ex2((st.m - p[k].m) * c); st.m = p[k].m; }
                z += p[k].z * ex2((p[k].m - st.m) * c);
            }
        }
    }
    st.drawn = warp_best(b).i;
    if (greedy) return st;
    const Weights weight(temp, warp_max(st.m));
    if (weight.odd) {                                        // once more, by the quotients
        z = 0.f;
        for (int i = lane; i < n; i += 32) {
            const Part p = nth(i);
            if (p.z > 0.f) z += p.z * weight.quotient(p.m);
        }
    } else if (z > 0.f) {
        z *= ex2((st.m - weight.most) * c);
    }
    st.z = warp_sum(z);
    st.m = weight.most;
    if (at_draft > -INFINITY && st.z > 0.f) st.share = weight(at_draft) / st.z;
    return st;
}

struct Range { unsigned least, most; };                       // of keys

struct RowShared {
    unsigned key[VD_CANDIDATES];
    int idx[VD_CANDIDATES];
    int line[VD_CANDIDATES];         // the lines that hold candidates
    unsigned hist[256], sel[2];
    Range range[VD_WARPS];
    float red[33];
    Best best[VD_WARPS];
    unsigned long long total[VD_WARPS];
    int lines, count, listed;
};

// Places in a shared list for the bits that a thread has set in `mask`: the first one's (a warp asks for all of its own at once).
__device__ __noinline__ int places_for(unsigned mask, int* counter) {
    const int lane = threadIdx.x & 31, n = __popc(mask);
    int upto = n, base = 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += w;
    }
    if (lane == 31 && upto > 0) base = atomicAdd(counter, upto);
    return __shfl_sync(~0u, base, 31) + upto - n;
}

// The least and the largest of the block's keys, two a thread; least: of those that are not 0.
__device__ __noinline__ Range key_range(unsigned one, unsigned two, Range* sh) {
    const unsigned least = __reduce_min_sync(~0u, min(one - 1u, two - 1u)), most = __reduce_max_sync(~0u, max(one, two));
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = Range{least, most};
    __syncthreads();
    const Range of = sh[threadIdx.x & (VD_WARPS - 1)];
    return Range{__reduce_min_sync(~0u, of.least) + 1u, __reduce_max_sync(~0u, of.most)};
}

// Of up to 512 keys, two a thread (0 where a thread has none; pairs: not all of the second are), of which at least k reach lo and none
// passes hi: a value that at least k reach, and no more than k + spare unless they are equal, by halving; a step is a count over the block.
__device__ __noinline__ unsigned reached_by(unsigned one, unsigned two, bool pairs, unsigned lo, unsigned hi, int k, int spare) {
#pragma unroll 1
    while (lo < hi) {
        const unsigned middle = lo + (hi - lo + 1) / 2;
        int n = __syncthreads_count(one >= middle);
        if (pairs) n += __syncthreads_count(two >= middle);
        if (n < k) {
            hi = middle - 1;
        } else {
            lo = middle;
            if (n <= k + spare) break;
        }
    }
    return lo;
}

// The same for any number of lines, none of which passes hi, by halving over all of them: a k in the hundreds.
__device__ __noinline__ unsigned lines_reached_by(RowShared& sh, const float* largest, int n, unsigned hi, int k, int spare) {
    unsigned lo = order_key(-INFINITY);                               // at least k reach lo
#pragma unroll 1
    for (int i = 0; i < 20 && lo < hi; ++i) {
        const unsigned middle = lo + (hi - lo + 1) / 2;
        int reach = 0;
        for (int j = threadIdx.x; j < n; j += VD_THREADS) reach += order_key(largest[j]) >= middle;
        reach = (int)block_sum((float)reach, sh.red);                 // at most 2^14 of them: exact
        if (reach < k) {
            hi = middle - 1;
        } else {
            lo = middle;
            if (reach <= k + spare) break;
        }
    }
    return lo;
}

__device__ __forceinline__ void copy_16(float* to, const float* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
// Copies four neighbouring logits (NaN behind the row's end) to shared memory, for the thread that asks.
__device__ __forceinline__ void copy_four(float* to, const float* x, int e, int vocab, int step) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(to);
    const float* from = x + e;
    if (step == 4 && e + 3 < vocab) {
        copy_16(to, from);
    } else if (step == 2 && e + 3 < vocab) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(from) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d + 8), "l"(from + 2) : "memory");
    } else {
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
            if (e + j < vocab) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d + 4 * j), "l"(from + j) : "memory");
            else to[j] = NAN;
        }
    }
}

// s + G of token i, and the share's time in the race: both are functions, there is one copy of their logarithms.
__device__ __noinline__ float exponential_of(int i, unsigned c1, unsigned stream, unsigned domain, uint2 key2) {
    uint4 c = make_uint4((unsigned)i >> 2, c1, stream, domain);
#pragma unroll 1
    for (int round = 0; round < 10; ++round) {
        c = philox_round(c, key2);
        key2.x += 0x9E3779B9u;
        key2.y += 0xBB67AE85u;
    }
    return -logf(philox_uniform(word_of(c, i)));
}

// Which of four logits reach `low`, as bits.
__device__ __forceinline__ unsigned reach_of(float4 f, float low) {
    auto bit = [&](float v, unsigned which) { return v >= low && v > -INFINITY ? which : 0u; };
    return bit(f.x, 1u) | bit(f.y, 2u) | bit(f.z, 4u) | bit(f.w, 8u);
}

constexpr int VD_STAGED = 16384;     // bytes of lines read again at a time, at least

__global__ void __launch_bounds__(VD_THREADS, 4) rows_kernel(VdArgs a) {
    extern __shared__ __align__(16) float largest[];         // the lines' largest, then lines
    __shared__ RowShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.y, D = a.max_drafts;
    ti_grid_launch_dependents();
    if (tid == 0) sh.lines = sh.count = sh.listed = 0;
    ti_grid_wait();
    const int2 rows = rows_of(a, r);
    const bool greedy = is_greedy(a, r);
    const Place at = place_of(a, r, blockIdx.x, rows, greedy);
    if (at.j < 0) return;
    const size_t slot = (size_t)r * a.places + blockIdx.x;
    const int topk = greedy ? 0 : a.topk[r];
    const float temp = greedy ? 1.f : a.temperature[r];
    const int drafted = at.j < rows.y - 1 ? a.token_ids[rows.x + at.j + 1] : -1;
    if (!has_threshold(topk, a.vocab)) {
        if (warp > 0) return;
        const RowStats st = whole_row(a, at, slot, greedy, temp, drafted);
        if (lane == 0) a.stats[slot] = st;
        return;
    }
    const int n_lines = a.tiles * VD_THREADS, step = row_step(at.x);
    const float* left = a.parts + slot * a.tiles * VD_THREADS;
#pragma unroll 1
    for (int i = 4 * tid; i < n_lines; i += 4 * VD_THREADS) copy_four(largest + i, left, i, n_lines, 4);
    const float at_draft = drafted >= 0 && drafted < a.vocab ? at.x[drafted] : NAN;
    const bool lists = !at.draws && (int)blockIdx.x <= D;    // a draw behind a failed draft may want them
    RowStats st{0.f, 0.f, 0u, -1, 0.f, -1, {0, 0}};
    float m = 0.f;                                           // the largest, scaled
    unsigned long long sum = 0;                              // weights of at most 1 in steps of 2^-44
    Best b{0.f, -1};
    asm volatile("cp.async.wait_all;" ::: "memory");

    __syncthreads();

    // A value that k lines' largest reach: by the largest of two shares of a thread's lines if those are enough, otherwise by all.
    float one = -INFINITY, two = -INFINITY;
#pragma unroll 2
    for (int i = tid; i < n_lines; i += 2 * VD_THREADS) {
        one = fmaxf(one, largest[i]);
        if (i + VD_THREADS < n_lines) two = fmaxf(two, largest[i + VD_THREADS]);
    }
    const Range offered = key_range(order_key(one), order_key(two), sh.range);
    // (near a k of all 512 shares their k-th largest is their least, which far too many lines reach: 64 x 3 rows and as many of the draft
    // model by the shares, by all lines, k = 100: 60, 78 us; k = 350: 79, 88 us; k = 400: 86, 88 us; k = 450: 414, 92 us)
    const unsigned bound = topk <= VD_THREADS * 3 / 2 ? reached_by(order_key(one), order_key(two), true, offered.least, offered.most, topk, topk / 8)
                                                      : lines_reached_by(sh, largest, n_lines, offered.most, topk, topk / 8);
    // (What lies 110 below the largest, scaled, has no weight in float32 and no noise that makes up for it: the tokens that a mask of the
    // type's lowest value leaves behind its own are not candidates, though the threshold may not drop them.)
    const float most = key_value(offered.most), floor = fabsf(most / temp) < 1e30f ? most - 110.f * temp - fabsf(most) * 4.8e-7f : -INFINITY;
    const float low = fmaxf(below_quotient(key_value(bound), temp), floor);
    constexpr int FOURS = 5;                                 // groups of four a thread looks at together
#pragma unroll 1
    for (int first = 0; first < n_lines; first += FOURS * 4 * VD_THREADS) {
        unsigned hits = 0u;
#pragma unroll
        for (int k = 0; k < FOURS; ++k) {
            const int i = first + 4 * (k * VD_THREADS + tid);
            if (i < n_lines) hits |= reach_of(*reinterpret_cast<const float4*>(largest + i), low) << (4 * k);
        }
        int to = places_for(hits, &sh.lines);
        for (; hits; hits &= hits - 1u, ++to) {
            const int bit = __ffs(hits) - 1;
            if (to < VD_CANDIDATES) sh.line[to] = first + 4 * ((bit >> 2) * VD_THREADS + tid) + (bit & 3);
        }
    }
    __syncthreads();
    bool fits = sh.lines <= VD_CANDIDATES;
    if (fits) {
        // their logits once more, a lane a group, as many lines at a time as there is room for where the largest were
        const int groups = sh.lines * (VD_LINE / 4), room = max(n_lines * 4, VD_STAGED) / 16;
        auto token = [&](int g) { return sh.line[g / (VD_LINE / 4)] * VD_LINE + g % (VD_LINE / 4) * 4; };
#pragma unroll 1
        for (int first = 0; first < groups; first += room) {
            const int some = min(room, groups - first);
            // (a thread copies, reads and copies over its own groups only)
#pragma unroll 1
            for (int g = tid; g < some; g += VD_THREADS) copy_four(largest + 4 * g, at.x, token(first + g), a.vocab, step);
            asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
            for (int base = 0; base < some; base += FOURS * VD_THREADS) {
                unsigned hits = 0u;
#pragma unroll
                for (int k = 0; k < FOURS; ++k) {
                    const int g = base + k * VD_THREADS + tid;
                    if (g < some) hits |= reach_of(*reinterpret_cast<const float4*>(largest + 4 * g), low) << (4 * k);
                }
                int to = places_for(hits, &sh.count);
                for (; hits; hits &= hits - 1u, ++to) {
                    const int bit = __ffs(hits) - 1, g = base + (bit >> 2) * VD_THREADS + tid;
                    if (to < VD_CANDIDATES) {
                        sh.key[to] = score_key(largest[4 * g + (bit & 3)] / temp);
                        sh.idx[to] = token(first + g) + (bit & 3);
                    }
                }
            }
        }
        __syncthreads();
        fits = sh.count <= VD_CANDIDATES;
    }
    const uint2 key2 = at.draws ? seed_of(a, r) : make_uint2(0u, 0u);
    const unsigned c1 = at.draws ? (unsigned)a.step[r] + (unsigned)at.j : 0u, stream = at.draws ? (unsigned)a.stream_id[r] : 0u;
    Kept* kept = lists ? a.kept + ((size_t)r * D + at.j) * a.list : nullptr;
    const int n = fits ? sh.count : a.vocab;
    auto take = [&](float s, int token) {
        if (score_key(s) < st.threshold || !(s > -INFINITY)) return;
        sum += __float2ull_rn(scaled_weight(s, m) * 17592186044416.f);
        if (at.draws) b = better(b, Best{s - logf(exponential_of(token, c1, stream, 0u, key2)), token});
        if (lists && fits) {
            const int to = atomicAdd(&sh.listed, 1);
            if (to < a.list) kept[to] = Kept{s, token};
        }
    };
    if (fits && n <= 2 * VD_THREADS) {
        // fewer than k: no finite logit of the row is missing, and all are kept
        const unsigned first = tid < n ? sh.key[tid] : 0u, second = tid + VD_THREADS < n ? sh.key[tid + VD_THREADS] : 0u;
        const Range found = key_range(first, second, sh.range);
        if (n >= topk) st.threshold = n == topk ? found.least : reached_by(first, second, n > VD_THREADS, found.least, found.most, topk, 0);
        m = n > 0 ? key_value(found.most) : -INFINITY;
    } else {
        // many candidates; or more than there is room for (a k in the thousands, thousands of equal logits): the row itself
        auto each = [&](auto f) {                            // every candidate's scaled logit
            if (fits) {
                for (int i = tid; i < n; i += VD_THREADS) f(key_value(sh.key[i]), sh.idx[i]);
            } else {
                each_of_row(at.x, a.vocab, step, [&](float v, int i) { if (v >= low && v > -INFINITY) f(v / temp, i); });
            }
        };
        if (n >= topk) st.threshold = select_kth(topk, sh.hist, sh.sel, [&](auto count) { each([&](float s, int) { count(score_key(s)); }); });
        m = most / temp;                                     // (quotients keep the order of what is divided)
        if (!fits) {
            each([&](float s, int token) { take(s, token); });
            if (tid == 0) sh.listed = a.list + 1;
        }
    }
    if (fits) {
#pragma unroll 1
        for (int i = tid; i < n; i += VD_THREADS) take(key_value(sh.key[i]), sh.idx[i]);
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    b = warp_best(b);
    if (lane == 0) { sh.total[warp] = sum; sh.best[warp] = b; }
    __syncthreads();
    if (warp > 0) return;
    sum = sh.total[lane & (VD_WARPS - 1)];
    b = sh.best[lane & (VD_WARPS - 1)];
#pragma unroll
    for (int o = VD_WARPS / 2; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(~0u, sum, o);
        b = better(b, Best{__shfl_xor_sync(~0u, b.v, o), __shfl_xor_sync(~0u, b.i, o)});
    }
    if (lane > 0) return;
    st.z = (float)((double)sum * (1.0 / 17592186044416.0));
    st.m = most;
    st.drawn = b.i;
    const float s = at_draft / temp;
    if (s > -INFINITY && score_key(s) >= st.threshold) st.share = scaled_weight(s, m) / st.z;
    if (lists && sh.listed <= a.list) st.listed = sh.listed;
    a.stats[slot] = st;
}

// Decides the request by its rows; if a drawn draft failed, draws from what is left of p beyond q. JUDGED: a cluster of blocks a
// request, which share that draw's rows out; otherwise a block. GREEDY: every request is, and the rows' parts are met here.
template <bool JUDGED, bool GREEDY>
__global__ void __launch_bounds__(VD_THREADS, JUDGED ? 4 : 1) verify_kernel(VdArgs a) {
    __shared__ RowStats row_sh[2 * VD_MAX_DRAFTS + 1];
    __shared__ Best best_sh[VD_WARPS], part_sh[VD_MOST_CTAS];
    __shared__ int held_sh;
    __shared__ unsigned beat_sh;
    ti_grid_launch_dependents();
    if (threadIdx.x == 0) beat_sh = 0u;
    ti_grid_wait();
    const int r = blockIdx.y, tid = threadIdx.x, D = a.max_drafts, rank = blockIdx.x;
    const int2 rows = rows_of(a, r);
    int* out = a.tokens + (size_t)r * (D + 1);
    const bool greedy = GREEDY || is_greedy(a, r);
    const int n = rows.y - 1;
    const bool judged = JUDGED && !greedy;                   // by the ratio of the probabilities
    const float temp = greedy ? 1.f : a.temperature[r];
    const bool thresholded = !greedy && has_threshold(a.topk[r], a.vocab);
    const uint2 key2 = judged ? seed_of(a, r) : make_uint2(0u, 0u);
    const unsigned step = judged ? (unsigned)a.step[r] : 0u, stream = judged ? (unsigned)a.stream_id[r] : 0u;
    const int fed = tid < n ? a.token_ids[rows.x + tid + 1] : -1;     // the draft of lane tid
    if (GREEDY) {
        for (int place = tid >> 5; place < rows.y; place += VD_WARPS) {
            const RowStats st = whole_row(a, place_of(a, r, place, rows, true), (size_t)r * a.places + place, true, 1.f, -1);
            if ((tid & 31) == 0) row_sh[place] = st;
        }
    } else if (tid < a.places && place_of(a, r, tid, rows, greedy).j >= 0) {
        row_sh[tid] = a.stats[(size_t)r * a.places + tid];
    }
    __syncthreads();
    if (tid < 32) {
        bool holds = false;
        if (tid < D) {
            float prob = 0.f;
            if (tid < n) {
                holds = fed >= 0 && fed == row_sh[tid].drawn;
                prob = greedy ? (holds ? 1.f : 0.f) : row_sh[tid].share;
                if (judged) {
                    const float q = row_sh[D + 1 + tid].share;
                    prob = q > 0.f ? fminf(prob / q, 1.f) : (prob > 0.f ? 1.f : 0.f);
                    holds = philox_uniform(philox4x32_10(make_uint4(0u, step + tid, stream, 1u), key2).x) < prob;
                }
            }
            if (rank == 0) a.accept[(size_t)r * D + tid] = prob;
        }
        const unsigned failed = __ballot_sync(~0u, !holds);  // at most 31 drafts: one lane at least does not hold
        if (tid == 0) held_sh = __ffs(failed) - 1;
    }
    __syncthreads();
    const int held = held_sh;
    Best b{0.f, -1};
    if (rows.y > 0) {
        const RowStats st = row_sh[held];
        b.i = st.drawn;
        const bool failed = held < n;
        if (JUDGED && judged && (failed || !thresholded)) {
            // What is left of p beyond q, or, if every draft held, an open row as ti_sample draws from it.
            const unsigned c1 = step + held, domain = failed ? 2u : 0u;
            const RowStats ds = failed ? row_sh[D + 1 + held] : RowStats{0.f, 0.f, 0u, -1, 0.f, -1, {0, 0}};
            const float* x = a.logits + (size_t)(rows.x + held) * a.vocab;
            const float* y = failed ? a.draft_logits + r * a.draft_request + held * a.draft_place : x;
            // By the quotients: rows with a threshold, whose sums were taken of them, and a draw from p alone far from 0, as sample's.
            Weights pw(temp, st.m), qw(temp, ds.m);
            pw.odd |= thresholded || (!failed && !pw.near());
            qw.odd |= thresholded;
            const float pz = st.z > 0.f ? 1.f / st.z : 0.f, qz = ds.z > 0.f ? 1.f / ds.z : 0.f;
            auto p_of = [&](float v) { return v > -INFINITY && (!st.threshold || score_key(v / temp) >= st.threshold) ? pw(v) * pz : 0.f; };
            auto q_of = [&](float v) { return v > -INFINITY && (!ds.threshold || score_key(v / temp) >= ds.threshold) ? qw(v) * qz : 0.f; };
            // An exponential race, the largest share / E, E = -log U; in ti_sample's terms the largest s + G.
            auto race = [&](float share, int i) {
                if (share > 0.f) b = better(b, Best{share / exponential_of(i, c1, stream, domain, key2), i});
            };
            b.i = -1;
            if (failed && st.listed >= 0) {                  // the threshold keeps few: the first block alone
                if (rank != 0) return;
                const Kept* list = a.kept + ((size_t)r * D + held) * a.list;
                // (second: nothing of p lies beyond q, they differ by a rounding: p itself)
#pragma unroll 1
                for (float q_share = 1.f; q_share >= 0.f && b.i < 0; q_share -= 1.f) {
                    for (int i = tid; i < st.listed; i += VD_THREADS) race(scaled_weight(list[i].s, pw.m) * pz - q_share * q_of(y[list[i].i]), list[i].i);
                    b = block_best(b, best_sh);
                }
            } else {
                cg::cluster_group cluster = cg::this_cluster();
                asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");     // this block runs (all of the cluster's come here)
                extern __shared__ __align__(16) float ring[];                  // [stage][row][thread][4]: a thread's own
                const int groups = (a.vocab + 3) / 4, ctas = gridDim.x, stride = ctas * VD_THREADS, x_step = row_step(x), y_step = row_step(y);
                const bool fours = x_step == 4 && y_step == 4;
                constexpr int ROW = 4 * VD_THREADS, STAGE = 2 * ROW;
                float* slot = ring + 4 * tid;                // of the stage whose turn it is
                auto fetch = [&](float* to, int g) {         // NaN where the row has no such tokens
                    if (fours && 4 * g + 3 < a.vocab) {
                        copy_16(to, x + 4 * g);
                        if (failed) copy_16(to + ROW, y + 4 * g);
                    } else {
                        copy_four(to, x, 4 * g, a.vocab, x_step);
                        if (failed) copy_four(to + ROW, y, 4 * g, a.vocab, y_step);
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                };
                // Logits that no threshold and no infinity cuts: a share is 2^(v c - most c - log2 z). Otherwise by p_of and q_of.
                // What rounding takes from the constants makes a factor, of p's share against q's.
                const bool plain = !st.threshold && !ds.threshold && pw.near() && !pw.odd && (!failed || (qw.near() && !qw.odd)) && st.z > 0.f;
                const float pl = log2f(st.z), p2 = pw.m2 + pl, ql = log2f(ds.z), q2 = failed ? qw.m2 + ql : INFINITY;
                auto rest = [](float a, float b, float sum) { return fabsf(a) < fabsf(b) ? (b - sum) + a : (a - sum) + b; };
                const float q_factor = failed ? ex2(rest(pw.m2, pl, p2) + pw.lost() - (rest(qw.m2, ql, q2) + qw.lost())) : 0.f;
                // Only tokens whose share can still pass the best B of the block run: share / E > B needs 1 - U < share / B.
                unsigned beaten = 0u;                        // B as a key, as this warp knows it
                float spare = INFINITY;                      // 1 / B, with something to spare
                auto beat = [&](unsigned key) {
                    beaten = key;
                    spare = pw.spare() * (failed ? 1.f / key_value(key) : ex2((pw.m - key_value(key)) * LOG2E) * st.z);
                };
#pragma unroll 1
                for (int k = 0; k < VD_STAGES; ++k) fetch(slot + k * STAGE, (rank + k * ctas) * VD_THREADS + tid);
#pragma unroll 1
                for (int g = rank * VD_THREADS + tid; g - tid < groups; g += stride) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(VD_STAGES - 1) : "memory");
                    const float4 f = *reinterpret_cast<const float4*>(slot);
                    float4 o = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (failed) o = *reinterpret_cast<const float4*>(slot + ROW);
                    const float v[4] = {f.x, f.y, f.z, f.w}, q[4] = {o.x, o.y, o.z, o.w};
                    float p[4];
                    if (plain) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float beyond = ex2(fmaf(fmaxf(q[i], -INFINITY), pw.c, -q2));
                            p[i] = fmaf(-q_factor, beyond, ex2(fmaf(fmaxf(v[i], -INFINITY), pw.c, -p2)));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[i] = p_of(v[i]) - (failed ? q_of(q[i]) : 0.f);
                    }
                    const float ahead = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
                    fetch(slot, g + VD_STAGES * stride);     // (what lay there is in registers)
                    slot = slot == ring + 4 * tid + (VD_STAGES - 1) * STAGE ? ring + 4 * tid : slot + STAGE;
                    // (one lane's view for all: another warp may write between two lanes' reads, and what follows is the warp's as a whole)
                    const unsigned now = __shfl_sync(~0u, *reinterpret_cast<volatile unsigned*>(&beat_sh), 0);
                    if (now != beaten) beat(now);
                    if (!__any_sync(~0u, plain ? ahead * spare > 5.9e-8f : ahead > 0.f)) continue;         // 1 - U is 2^-24 at least
                    const uint4 w = philox4x32_10(make_uint4((unsigned)g, c1, stream, domain), key2);
                    unsigned run = 0u;
                    auto run_all = [&]() {
#pragma unroll 1
                        for (; run; run &= run - 1u) {
                            const int i = __ffs(run) - 1;
                            const float e = -logf(philox_uniform(word_of(w, i)));
                            const float share = i & 2 ? (i & 1 ? p[3] : p[2]) : (i & 1 ? p[1] : p[0]);
                            const float own = i & 2 ? (i & 1 ? v[3] : v[2]) : (i & 1 ? v[1] : v[0]);
                            b = better(b, Best{failed ? share / e : own / temp - logf(e), 4 * g + i});
                        }
                        const unsigned best = __reduce_max_sync(~0u, b.i < 0 ? 0u : order_key(b.v));
                        if (best > beaten) {
                            if ((tid & 31) == 0) atomicMax(&beat_sh, best);
                            beat(best);
                        }
                    };
                    if (spare == INFINITY || !plain) {       // nothing to beat yet: the foremost of every thread first; or no telling: all
                        const float least = plain ? ahead : 0.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) run |= p[i] > 0.f && p[i] >= least ? 1u << i : 0u;
                        run_all();
                        if (!plain) continue;
                    }
                    const unsigned words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) run |= may_pass(words[i], p[i], spare) ? 1u << i : 0u;
                    if (__any_sync(~0u, run)) run_all();
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                b = block_best(b, best_sh);
                asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
                if (tid == 0) *cluster.map_shared_rank(&part_sh[rank], 0) = b;
                cluster.sync();
                if (rank != 0) return;
                b = warp_best((tid & 31) < ctas ? part_sh[tid & 31] : Best{0.f, -1});
            }
            if (b.i < 0 && failed) {                         // nothing of p lies beyond q, as above
                each_of_row(x, a.vocab, row_step(x), [&](float v, int i) { race(p_of(v), i); });
                b = block_best(b, best_sh);
            }
        }
    }
    if (rank == 0 && tid <= D) {
        const int token = rows.y > 0 && tid == held ? max(b.i, 0) : -1;
        out[tid] = rows.y > 0 && tid < held ? fed : token;
        if (tid == 0) a.counts[r] = rows.y > 0 ? held + 1 : 0;
    }
}

struct Scratch { long long parts, stats, kept, words; int list; };      // offsets in words (32 bits)
Scratch scratch_of(int requests, int max_drafts, int vocab, bool sampled, bool draft_logits) {
    const long long places = draft_logits ? 2 * max_drafts + 1 : max_drafts + 1, tiles = (vocab + VD_TILE - 1) / VD_TILE;
    Scratch s;
    s.parts = 0;
    s.stats = s.parts + requests * places * tiles * VD_THREADS;
    s.kept = s.stats + (sampled ? requests * places * (long long)(sizeof(RowStats) / 4) : 0);
    s.list = std::min(vocab, VD_LIST);
    s.words = s.kept + (draft_logits ? (long long)requests * max_drafts * s.list * (long long)(sizeof(Kept) / 4) : 0);
    return s;
}

}  // namespace

// Words (32 bits) of scratch a call needs, on a 16-byte boundary: what its rows leave for the kernels behind.
TI_API long long ti_verify_scratch_words(int requests, int max_drafts, int vocab, int sampled, int draft_logits) {
    return scratch_of(requests, max_drafts, vocab, sampled != 0, draft_logits != 0).words;
}

TI_API int ti_verify_drafts(int* tokens, int* counts, float* accept, const float* logits, const int* token_ids, const int* cu_rows,
                            int rows, int vocab, int requests, int max_drafts, const float* temperature, const int* topk,
                            const int* greedy, const long long* seed, const int* stream_id, const int* step, const float* draft_logits,
                            long long draft_request, long long draft_place, void* scratch, cudaStream_t stream) {
    TI_REQUIRE(rows >= 0 && vocab > 0 && requests >= 0 && requests <= 65535, "verify_drafts: bad sizes");
    TI_REQUIRE(max_drafts >= 0 && max_drafts <= VD_MAX_DRAFTS, "verify_drafts: at most %d drafts a request", VD_MAX_DRAFTS);
    TI_REQUIRE(vocab <= VD_MAX_VOCAB, "verify_drafts: at most %d tokens in the vocabulary", VD_MAX_VOCAB);
    TI_REQUIRE(temperature || !draft_logits, "verify_drafts: greedy requests have no use for draft logits");
    if (requests == 0) return 0;
    const Scratch s = scratch_of(requests, max_drafts, vocab, temperature != nullptr, draft_logits != nullptr);
    float* words = (float*)scratch;
    VdArgs a{logits, token_ids, cu_rows, temperature, topk, greedy, seed, stream_id, step, draft_logits, draft_request, draft_place,
             words + s.parts, (RowStats*)(words + s.stats), (Kept*)(words + s.kept), tokens, counts, accept, rows, vocab, requests, max_drafts,
             (vocab + VD_TILE - 1) / VD_TILE, s.list, draft_logits ? 2 * max_drafts + 1 : max_drafts + 1};
    ti_launch(draft_logits || !temperature ? parts_kernel<false> : parts_kernel<true>, dim3(a.tiles, a.places, requests), VD_THREADS, 0, stream, a);
    TI_CHECK_LAUNCH("verify_drafts: parts");
    if (temperature) {
        const int shared = std::max(a.tiles * VD_THREADS * 4, VD_STAGED);
        TI_REQUIRE(ti_allow_shared<rows_kernel>(shared) == cudaSuccess, "verify_drafts: %d bytes of shared memory are not to be had", shared);
        ti_launch(rows_kernel, dim3(a.places, requests), VD_THREADS, shared, stream, a);
        TI_CHECK_LAUNCH("verify_drafts: rows");
    }
    if (draft_logits) {
        constexpr int shared = VD_STAGES * 2 * VD_THREADS * 16;
        TI_REQUIRE((ti_allow_shared<verify_kernel<true, false>>(shared) == cudaSuccess), "verify_drafts: %d bytes of shared memory are not to be had", shared);
        // Sixteen blocks a request while all of them run at once, otherwise eight: 32 requests x 4 drafts, of which 8 are open, 40 us for 43;
        // 64 open requests x 7 drafts 137 us for 126 (captured).
        const bool wide = requests * VD_MOST_CTAS <= 148 * 4 && ti_allow_wide_clusters<verify_kernel<true, false>>() == cudaSuccess;
        const int ctas = wide ? VD_MOST_CTAS : VD_CTAS;
        ti_launch_clusters(verify_kernel<true, false>, dim3(ctas, requests), ctas, VD_THREADS, shared, stream, a);
    }
    else ti_launch(temperature ? verify_kernel<false, false> : verify_kernel<false, true>, dim3(1, requests), VD_THREADS, 0, stream, a);
    TI_CHECK_LAUNCH("verify_drafts");
    return 0;
}
