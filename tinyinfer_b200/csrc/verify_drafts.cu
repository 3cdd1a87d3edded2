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
// Sums and exponentials are float32.
#include "draws.cuh"

namespace {

constexpr int VD_MAX_DRAFTS = 31;    // a warp decides a request: a lane a draft, and one place more
constexpr int VD_THREADS = 512;

// What a row leaves: the largest scaled logit, the sum of the kept exponentials, the lowest kept key, the token that it draws (-1:
// none; of a sampled row that a draft model's logits judge: not drawn yet).
struct __align__(16) RowStats { float m, z; unsigned threshold; int drawn; };

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
    RowStats *target, *draft;        // [requests, max_drafts + 1], [requests, max_drafts]
    int* tokens;                     // [requests, max_drafts + 1]
    int* counts;
    float* accept;                   // [requests, max_drafts]
    int rows, vocab, requests, max_drafts;
};

// The request's rows: first flat row and how many (0 .. max_drafts + 1), inside the logits whatever cu_rows says.
__device__ __forceinline__ int2 rows_of(const VdArgs& a, int r) {
    const int lo = min(max(a.cu_rows[r], 0), a.rows), hi = min(max(a.cu_rows[r + 1], lo), a.rows);
    return make_int2(lo, min(hi - lo, a.max_drafts + 1));
}
__device__ __forceinline__ bool is_greedy(const VdArgs& a, int r) { return a.temperature == nullptr || a.greedy[r] != 0; }

__device__ __forceinline__ unsigned score_key(float s) { return order_key(s + 0.f); }        // -0 and +0 are one value

// exp(s - m) where the threshold keeps s, else 0. The largest is 1 even where it is infinite; -inf and NaN are never kept.
__device__ __forceinline__ float kept_weight(float s, const RowStats& st) {
    if (!(s > -INFINITY) || score_key(s) < st.threshold) return 0.f;
    return s == st.m ? 1.f : expf(s - st.m);
}

template <typename F>
__device__ __forceinline__ void each_logit(const float* x, int vocab, F f) {
    for (int i = threadIdx.x; i < vocab; i += VD_THREADS) f(x[i], i);
}

__device__ __forceinline__ Best block_best(Best x, Best* sh) {
    auto warp_best = [](Best v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = better(v, Best{__shfl_xor_sync(~0u, v.v, o), __shfl_xor_sync(~0u, v.i, o)});
        return v;
    };
    x = warp_best(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = x;
    __syncthreads();
    return warp_best((threadIdx.x & 31) < VD_THREADS / 32 ? sh[threadIdx.x & 31] : Best{0.f, -1});
}

// The row's draw: the best of s_i + G_i over what the threshold keeps.
__device__ __forceinline__ Best draw_row(const float* x, int vocab, float temp, unsigned threshold, unsigned c1, unsigned stream, uint2 key2,
                                         Best* sh) {
    Best b{0.f, -1};
    each_logit(x, vocab, [&](float v, int i) {
        const float s = v / temp;
        if (s > -INFINITY && score_key(s) >= threshold) {
            const uint4 w = philox4x32_10(make_uint4((unsigned)i >> 2, c1, stream, 0u), key2);
            const unsigned words[4] = {w.x, w.y, w.z, w.w};
            b = better(b, Best{s - logf(-logf(philox_uniform(words[i & 3]))), i});
        }
    });
    return block_best(b, sh);
}
__device__ __forceinline__ uint2 seed_of(const VdArgs& a, int r) {
    return make_uint2((unsigned)(a.seed[r] & 0xFFFFFFFFll), (unsigned)((unsigned long long)a.seed[r] >> 32));
}

__global__ void __launch_bounds__(VD_THREADS) row_stats_kernel(VdArgs a) {
    __shared__ unsigned hist[256], sel[2];
    __shared__ float red[33];
    __shared__ Best sh[VD_THREADS / 32];
    ti_grid_launch_dependents();
    ti_grid_wait();
    const int r = blockIdx.y, place = blockIdx.x;
    const int2 rows = rows_of(a, r);
    const bool greedy = is_greedy(a, r), of_draft = place > a.max_drafts;
    const int j = of_draft ? place - a.max_drafts - 1 : place;
    if (of_draft ? greedy || j >= rows.y - 1 : j >= rows.y) return;
    const float* x = of_draft ? a.draft_logits + r * a.draft_request + j * a.draft_place : a.logits + (size_t)(rows.x + j) * a.vocab;
    const float temp = greedy ? 1.f : a.temperature[r];
    const int k = greedy ? 0 : a.topk[r];
    RowStats st{0.f, 0.f, 0u, -1};
    Best b{0.f, -1};
    each_logit(x, a.vocab, [&](float v, int i) {
        const float s = v / temp;
        if (s == s) b = better(b, Best{s, i});
    });
    b = block_best(b, sh);
    st.m = b.v;
    st.drawn = greedy ? b.i : -1;
    if (!greedy) {
        if (k > 0 && k < a.vocab)
            st.threshold = select_kth(k, hist, sel, [&](auto count) {
                each_logit(x, a.vocab, [&](float v, int) {
                    const float s = v / temp;
                    if (s == s) count(score_key(s));
                });
            });
        float z = 0.f;
        each_logit(x, a.vocab, [&](float v, int) { z += kept_weight(v / temp, st); });
        st.z = block_sum(z, red);
        if (!a.draft_logits) st.drawn = draw_row(x, a.vocab, temp, st.threshold, (unsigned)(a.step[r] + j), (unsigned)a.stream_id[r], seed_of(a, r), sh).i;
    }
    if (threadIdx.x == 0) (of_draft ? a.draft[r * a.max_drafts + j] : a.target[r * (a.max_drafts + 1) + j]) = st;
}

__global__ void __launch_bounds__(VD_THREADS) verify_kernel(VdArgs a) {
    __shared__ Best sh[VD_THREADS / 32];
    __shared__ int held_sh;
    ti_grid_launch_dependents();
    ti_grid_wait();
    const int r = blockIdx.x, tid = threadIdx.x, D = a.max_drafts;
    const int2 rows = rows_of(a, r);
    int* out = a.tokens + (size_t)r * (D + 1);
    const bool greedy = is_greedy(a, r);
    const int n = rows.y - 1;
    const float temp = greedy ? 1.f : a.temperature[r];
    const bool judged = !greedy && a.draft_logits;            // by the ratio of the probabilities
    const uint2 key2 = greedy ? make_uint2(0u, 0u) : seed_of(a, r);
    const unsigned step = greedy ? 0u : (unsigned)a.step[r], stream = greedy ? 0u : (unsigned)a.stream_id[r];
    if (tid < 32) {
        const int j = tid;
        bool holds = false;
        if (j < D) {
            float prob = 0.f;
            if (j < n) {
                const int d = a.token_ids[rows.x + j + 1];
                const RowStats st = a.target[r * (D + 1) + j];
                const bool drawn = d >= 0 && d == st.drawn;
                if (greedy) {
                    prob = drawn ? 1.f : 0.f;
                } else if (d >= 0 && d < a.vocab && st.z > 0.f) {
                    const float p = kept_weight(a.logits[(size_t)(rows.x + j) * a.vocab + d] / temp, st) / st.z;
                    float q = 1.f;
                    if (judged) {
                        const RowStats ds = a.draft[r * D + j];
                        q = ds.z > 0.f ? kept_weight(a.draft_logits[r * a.draft_request + j * a.draft_place + d] / temp, ds) / ds.z : 0.f;
                    }
                    prob = q > 0.f ? fminf(p / q, 1.f) : (p > 0.f ? 1.f : 0.f);
                }
                holds = judged ? philox_uniform(philox4x32_10(make_uint4(0u, step + j, stream, 1u), key2).x) < prob : drawn;
            }
            a.accept[(size_t)r * D + j] = prob;
        }
        const unsigned failed = __ballot_sync(~0u, !holds);
        if (tid == 0) held_sh = __ffs(failed) - 1;           // at most 31 drafts: one lane at least does not hold
    }
    __syncthreads();
    const int held = held_sh;
    if (rows.y == 0) {
        if (tid <= D) out[tid] = -1;
        if (tid == 0) a.counts[r] = 0;
        return;
    }
    const RowStats st = a.target[r * (D + 1) + held];
    const float* x = a.logits + (size_t)(rows.x + held) * a.vocab;
    Best b{0.f, st.drawn};
    if (judged) {
        const unsigned c1 = step + held;
        b.i = -1;
        if (held == n) {
            b = draw_row(x, a.vocab, temp, st.threshold, c1, stream, key2, sh);
        } else {
            const RowStats ds = a.draft[r * D + held];
            const float* y = a.draft_logits + r * a.draft_request + held * a.draft_place;
            for (int beyond = 1; beyond >= 0 && b.i < 0; --beyond) {      // 0: nothing of p lies beyond q (they differ by a rounding): p itself
                each_logit(x, a.vocab, [&](float v, int i) {
                    float p = kept_weight(v / temp, st) / st.z;
                    if (beyond && ds.z > 0.f) p -= kept_weight(y[i] / temp, ds) / ds.z;
                    if (p > 0.f) {
                        const uint4 w = philox4x32_10(make_uint4((unsigned)i >> 2, c1, stream, 2u), key2);
                        const unsigned words[4] = {w.x, w.y, w.z, w.w};
                        b = better(b, Best{p / -logf(philox_uniform(words[i & 3])), i});
                    }
                });
                b = block_best(b, sh);
            }
        }
    }
    if (tid <= D) out[tid] = tid < held ? a.token_ids[rows.x + tid + 1] : (tid == held ? max(b.i, 0) : -1);
    if (tid == 0) a.counts[r] = held + 1;
}

}  // namespace

// Words (32 bits) of scratch a call needs, on a 16-byte boundary: what its rows leave for the kernel behind.
TI_API long long ti_verify_scratch_words(int requests, int max_drafts, int vocab) {
    (void)vocab;
    return 4ll * requests * (2 * max_drafts + 1);
}

TI_API int ti_verify_drafts(int* tokens, int* counts, float* accept, const float* logits, const int* token_ids, const int* cu_rows,
                            int rows, int vocab, int requests, int max_drafts, const float* temperature, const int* topk,
                            const int* greedy, const long long* seed, const int* stream_id, const int* step, const float* draft_logits,
                            long long draft_request, long long draft_place, void* scratch, cudaStream_t stream) {
    TI_REQUIRE(rows >= 0 && vocab > 0 && requests >= 0 && requests <= 65535, "verify_drafts: bad sizes");
    TI_REQUIRE(max_drafts >= 0 && max_drafts <= VD_MAX_DRAFTS, "verify_drafts: at most %d drafts a request", VD_MAX_DRAFTS);
    TI_REQUIRE(temperature || !draft_logits, "verify_drafts: greedy requests have no use for draft logits");
    if (requests == 0) return 0;
    VdArgs a{logits, token_ids, cu_rows, temperature, topk, greedy, seed, stream_id, step, draft_logits, draft_request, draft_place,
             (RowStats*)scratch, (RowStats*)scratch + (size_t)requests * (max_drafts + 1), tokens, counts, accept, rows, vocab, requests, max_drafts};
    ti_launch(row_stats_kernel, dim3(max_drafts + 1 + (draft_logits ? max_drafts : 0), requests), VD_THREADS, 0, stream, a);
    TI_CHECK_LAUNCH("verify_drafts: rows");
    ti_launch(verify_kernel, requests, VD_THREADS, 0, stream, a);
    TI_CHECK_LAUNCH("verify_drafts");
    return 0;
}
