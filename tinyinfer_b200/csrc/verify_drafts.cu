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
// they were found does not show).
//
// Bound by reading the logits once: a row is held by a cluster of blocks, 40 logits a thread in registers (all its loads in flight at
// once), so threshold, sum and draw take no second trip to memory. The blocks of a row meet in the first one's shared memory.
#include <cooperative_groups.h>

#include "draws.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int VD_MAX_DRAFTS = 31;    // a warp decides a request: a lane a draft, and one place more
constexpr int VD_THREADS = 512;
constexpr int VD_WARPS = VD_THREADS / 32;
constexpr int VD_GROUPS = 10;        // groups of four logits a thread holds
constexpr int VD_SLICE = VD_THREADS * VD_GROUPS * 4;
constexpr int VD_MAX_CTAS = 16;
constexpr int VD_CANDIDATES = 2048;  // of a top-k row, in the first block's shared memory
constexpr int VD_LIST = 256;         // of what the threshold keeps, for the draw behind a draft that failed
constexpr float LOG2E = 1.4426950408889634f;

// What a row leaves: the largest scaled logit, the sum of the kept exponentials, the lowest kept key, the token that it draws (-1:
// none; of a sampled row that a draft model's logits judge: not drawn yet), the share of its draft, how many kept tokens are listed.
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
    RowStats *target, *draft;        // [requests, max_drafts + 1], [requests, max_drafts]
    Kept* kept;                      // [requests, max_drafts, VD_LIST]
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
__device__ __forceinline__ uint2 seed_of(const VdArgs& a, int r) {
    return make_uint2((unsigned)(a.seed[r] & 0xFFFFFFFFll), (unsigned)((unsigned long long)a.seed[r] >> 32));
}
__device__ __forceinline__ unsigned score_key(float s) { return order_key(s + 0.f); }        // -0 and +0 are one value

// The weights of a row's logits, exp(v / temp - m): 2^(v * c - m * log2 e), one multiply-add and one exponential. Where that has
// infinities on both sides (an infinite logit; a temperature whose quotients leave float32) the quotient itself is compared.
struct Weights {
    float temp, m, c, m2;
    bool odd;
    __device__ __forceinline__ Weights(float temp_, float m_) : temp(temp_), m(m_), c(LOG2E / temp_), m2(m_ * LOG2E) {
        odd = !(fabsf(m) < 1e30f) || !(c < 1e30f);
    }
    __device__ __forceinline__ float operator()(float v) const {
        if (odd) {
            const float s = v / temp;
            return !(s > -INFINITY) ? 0.f : (s == m ? 1.f : expf(s - m));
        }
        return exp2f(fmaf(v, c, -m2));
    }
};
// The same of a scaled logit at hand.
__device__ __forceinline__ float scaled_weight(float s, float m) { return !(s > -INFINITY) ? 0.f : (s == m ? 1.f : exp2f((s - m) * LOG2E)); }

__device__ __forceinline__ Best warp_best(Best v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = better(v, Best{__shfl_xor_sync(~0u, v.v, o), __shfl_xor_sync(~0u, v.i, o)});
    return v;
}
__device__ __forceinline__ float warp_min(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(~0u, v, o));
    return v;
}
template <int WARPS>
__device__ __forceinline__ Best block_best(Best x, Best* sh) {
    x = warp_best(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = x;
    __syncthreads();
    return warp_best((threadIdx.x & 31) < WARPS ? sh[threadIdx.x & 31] : Best{0.f, -1});
}

// A value that is below every logit whose quotient by temp reaches that of `bound`: quotients are rounded, by 2^-24 of themselves
// where they are normal numbers; elsewhere every logit may.
__device__ __forceinline__ float below_quotient(float bound, float temp) {
    const float s = fabsf(bound / temp);
    return s > 1e-35f && s < 1e37f ? bound - fabsf(bound) * 4.8e-7f : -INFINITY;
}

// A thread's part of a row, in groups of four logits: group (k * ctas + rank) * threads + tid. Which thread holds which logits goes by
// their number alone, not by where the row lies, so that the order of sums does not either: a row off 16-byte boundaries (of an odd
// vocabulary, say) is read 8 or 4 bytes at a time.
struct Slice {
    const float* x;                  // the row
    int first, stride, vocab, step;
    __device__ __forceinline__ Slice(const float* x_, int vocab_, int rank, int ctas)
        : x(x_), first(4 * (rank * VD_THREADS + (int)threadIdx.x)), stride(4 * ctas * VD_THREADS), vocab(vocab_),
          step(((uintptr_t)x_ & 15) == 0 ? 4 : ((uintptr_t)x_ & 7) == 0 ? 2 : 1) {}
    __device__ __forceinline__ int token(int k) const { return first + k * stride; }        // the group's first
    __device__ __forceinline__ void load(int k, float (&v)[4]) const {
        const int e = token(k);
        if (step == 4 && e + 3 < vocab) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(x + e));
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else if (step == 2 && e + 3 < vocab) {
            const float2 f = *reinterpret_cast<const float2*>(x + e), g = *reinterpret_cast<const float2*>(x + e + 2);
            v[0] = f.x; v[1] = f.y; v[2] = g.x; v[3] = g.y;
        } else {                                         // also the row's end, and places behind it
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = e + j < vocab ? x[e + j] : NAN;
        }
    }
};

struct RowShared {
    unsigned key[VD_CANDIDATES];
    int idx[VD_CANDIDATES];
    unsigned sums[4][256];           // the first block's: the row's histogram of each byte
    unsigned hist[256], sel[2];
    float bound[VD_MAX_CTAS], m[VD_MAX_CTAS], z[VD_MAX_CTAS];
    Best part[VD_MAX_CTAS];
    float warp[VD_WARPS], red[33];
    Best best[VD_WARPS];
    unsigned long long total[VD_WARPS];
    int count, over, listed;
};

// The k-th largest key of the row by radix selection over what the blocks hold, all blocks together; any k, any number of ties.
__device__ __forceinline__ unsigned row_threshold(RowShared& sh, cg::cluster_group& cluster, const float (&v)[VD_GROUPS][4], const Slice& s, float temp, int k) {
    const int tid = threadIdx.x;
    unsigned prefix = 0u, left = (unsigned)k;
    for (int pass = 0; pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
        const unsigned mask = pass == 0 ? 0u : 0xFFFFFFFFu << (shift + 8);
        if (tid < 256) sh.hist[tid] = 0u;
        __syncthreads();
#pragma unroll
        for (int g = 0; g < VD_GROUPS; ++g) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned key = score_key(v[g][j] / temp);
                if (v[g][j] > -INFINITY && (key & mask) == prefix) {
                    const unsigned bin = (key >> shift) & 0xFFu, same = __match_any_sync(__activemask(), bin);
                    if ((tid & 31) == __ffs(same) - 1) atomicAdd(&sh.hist[bin], (unsigned)__popc(same));
                }
            }
        }
        __syncthreads();
        if (tid < 256 && sh.hist[tid]) atomicAdd(cluster.map_shared_rank(&sh.sums[pass][tid], 0), sh.hist[tid]);
        cluster.sync();
        if (cluster.block_rank() == 0 && tid < 32) {         // a lane eight bins; the highest whose bins, with all above, reach the k-th
            unsigned mine[8], sum = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) { mine[i] = sh.sums[pass][8 * tid + i]; sum += mine[i]; }
            unsigned above = sum;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const unsigned w = __shfl_down_sync(~0u, above, off);
                if (tid + off < 32) above += w;
            }
            const unsigned reach = __ballot_sync(~0u, above >= left);
            if (reach ? tid == 31 - __clz(reach) : tid == 0) {
                unsigned want = left - (above - sum);
                int b = 7;
                if (reach) {
                    for (; b > 0 && mine[b] < want; --b) want -= mine[b];
                } else {                                     // fewer than k: all of them
                    b = 0;
                    want = 0u;
                }
                sh.sel[0] = reach ? prefix | ((unsigned)(8 * tid + b) << shift) : 0u;
                sh.sel[1] = want;
            }
        }
        cluster.sync();
        prefix = *cluster.map_shared_rank(&sh.sel[0], 0);
        left = *cluster.map_shared_rank(&sh.sel[1], 0);
        if (left == 0u) break;
    }
    cluster.sync();                                          // the first block goes on only when all have read
    return left == 0u ? 0u : prefix;
}

__global__ void __launch_bounds__(VD_THREADS, 2) row_kernel(VdArgs a) {
    __shared__ RowShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = blockIdx.x, ctas = gridDim.x;
    const int r = blockIdx.z, place = blockIdx.y, D = a.max_drafts;
    ti_grid_launch_dependents();
    ti_grid_wait();
    const int2 rows = rows_of(a, r);
    const bool greedy = is_greedy(a, r), of_draft = place > D;
    const int j = of_draft ? place - D - 1 : place;
    if (of_draft ? greedy || j >= rows.y - 1 : j >= rows.y) return;
    const float* x = of_draft ? a.draft_logits + r * a.draft_request + j * a.draft_place : a.logits + (size_t)(rows.x + j) * a.vocab;
    const Slice slice(x, a.vocab, rank, ctas);
    float v[VD_GROUPS][4];
#pragma unroll
    for (int k = 0; k < VD_GROUPS; ++k) slice.load(k, v[k]);
    const int drafted = j < rows.y - 1 ? a.token_ids[rows.x + j + 1] : -1;
    const float at_draft = drafted >= 0 && drafted < a.vocab ? x[drafted] : NAN;
    const float temp = greedy ? 1.f : a.temperature[r];
    const int topk = greedy ? 0 : a.topk[r];
    const bool draws = !greedy && !of_draft && (a.draft_logits == nullptr || j == rows.y - 1);
    const uint2 key2 = draws ? seed_of(a, r) : make_uint2(0u, 0u);
    const unsigned c1 = draws ? (unsigned)(a.step[r] + j) : 0u, stream = draws ? (unsigned)a.stream_id[r] : 0u;
    // what the other blocks write to or count in
    if (tid < 256)
        for (int p = 0; p < 4; ++p) sh.sums[p][tid] = 0u;
    if (tid == 0) sh.count = sh.over = sh.listed = 0;
    cluster.sync();
    RowStats* out = of_draft ? a.draft + r * D + j : a.target + r * (D + 1) + j;
    RowStats st{0.f, 0.f, 0u, -1, 0.f, -1, {0, 0}};

    if (greedy) {
        Best b{-INFINITY, -1};
#pragma unroll
        for (int k = 0; k < VD_GROUPS; ++k) {
#pragma unroll
            for (int q = 0; q < 4; ++q)                      // a thread's tokens come in their order: the first of equals stays
                if (v[k][q] > b.v || (b.i < 0 && v[k][q] == v[k][q])) b = Best{v[k][q], slice.token(k) + q};
        }
        b = block_best<VD_WARPS>(b, sh.best);
        if (tid == 0) *cluster.map_shared_rank(&sh.part[rank], 0) = b;
        cluster.sync();
        if (rank == 0 && warp == 0) {
            b = warp_best(lane < ctas ? sh.part[lane] : Best{0.f, -1});
            st.drawn = b.i;
            if (lane == 0) *out = st;
        }
        return;
    }

    float most = -INFINITY;
#pragma unroll
    for (int k = 0; k < VD_GROUPS; ++k) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            v[k][q] = fmaxf(v[k][q], -INFINITY);             // NaN and places outside the row: -inf
            most = fmaxf(most, v[k][q]);
        }
    }
    if (topk > 0 && topk < a.vocab) {
        bool wide = topk > ctas * VD_THREADS;                // more than there are threads to offer a value each
        if (!wide) {
            // Every warp offers the u-th largest of its threads' largest logits, u * warps >= k: at least k logits of the row
            // reach the least of these offers, and few more do. Those are the row's candidates.
            const int u = (topk + ctas * VD_WARPS - 1) / (ctas * VD_WARPS);
            float offer = 0.f, rest = most;
            for (int i = 0; i < u; ++i) {
                offer = warp_max(rest);
                const unsigned who = __ballot_sync(~0u, rest == offer);
                if (lane == __ffs(who) - 1) rest = -INFINITY;
            }
            if (lane == 0) sh.warp[warp] = offer;
            __syncthreads();
            const float least = warp_min(lane < VD_WARPS ? sh.warp[lane] : INFINITY);
            if (tid < ctas) *cluster.map_shared_rank(&sh.bound[rank], tid) = least;
            cluster.sync();
            const float low = below_quotient(warp_min(lane < ctas ? sh.bound[lane] : INFINITY), temp);
            int n = 0;
            if (most >= low && most > -INFINITY) {
#pragma unroll
                for (int k = 0; k < VD_GROUPS; ++k) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) n += v[k][q] >= low && v[k][q] > -INFINITY;
                }
            }
            int before = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int w = __shfl_up_sync(~0u, before, o);
                if (lane >= o) before += w;
            }
            int base = 0;
            if (lane == 31 && before > 0) {
                base = atomicAdd(cluster.map_shared_rank(&sh.count, 0), before);
                if (base + before > VD_CANDIDATES)
                    for (int c = 0; c < ctas; ++c) *cluster.map_shared_rank(&sh.over, c) = 1;
            }
            int at = __shfl_sync(~0u, base, 31) + before - n;
            if (n > 0) {
                unsigned* keys = cluster.map_shared_rank(sh.key, 0);
                int* idx = cluster.map_shared_rank(sh.idx, 0);
#pragma unroll
                for (int k = 0; k < VD_GROUPS; ++k) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (v[k][q] >= low && v[k][q] > -INFINITY) {
                            if (at < VD_CANDIDATES) { keys[at] = score_key(v[k][q] / temp); idx[at] = slice.token(k) + q; }
                            ++at;
                        }
                }
            }
            cluster.sync();
            wide = sh.over != 0;
        }
        if (!wide) {
            if (rank != 0) return;
            // the first block alone, on the candidates
            const int n = sh.count;
            if (n > topk)
                st.threshold = select_kth(topk, sh.hist, sh.sel, [&](auto count) {
                    for (int i = tid; i < n; i += VD_THREADS) count(sh.key[i]);
                });
            unsigned top = 0u;
            for (int i = tid; i < n; i += VD_THREADS) top = max(top, sh.key[i]);
            top = __reduce_max_sync(~0u, top);
            if (lane == 0) sh.warp[warp] = __uint_as_float(top);
            __syncthreads();
            top = __reduce_max_sync(~0u, lane < VD_WARPS ? __float_as_uint(sh.warp[lane]) : 0u);
            st.m = n > 0 ? key_value(top) : -INFINITY;
            unsigned long long sum = 0;                      // weights of at most 1 in steps of 2^-44
            Best b{0.f, -1};
            const bool lists = !draws && !of_draft;
            for (int i = tid; i < n; i += VD_THREADS) {
                if (sh.key[i] < st.threshold) continue;
                const float s = key_value(sh.key[i]);
                sum += __float2ull_rn(scaled_weight(s, st.m) * 17592186044416.f);
                if (draws) {
                    const uint4 w = philox4x32_10(make_uint4((unsigned)sh.idx[i] >> 2, c1, stream, 0u), key2);
                    const unsigned words[4] = {w.x, w.y, w.z, w.w};
                    b = better(b, Best{s - logf(-logf(philox_uniform(words[sh.idx[i] & 3]))), sh.idx[i]});
                }
                if (lists) {
                    const int slot = atomicAdd(&sh.listed, 1);
                    if (slot < VD_LIST) a.kept[((size_t)r * D + j) * VD_LIST + slot] = Kept{s, sh.idx[i]};
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            if (lane == 0) sh.total[warp] = sum;
            b = block_best<VD_WARPS>(b, sh.best);
            if (tid == 0) {
                sum = 0;
                for (int w = 0; w < VD_WARPS; ++w) sum += sh.total[w];
                st.z = (float)((double)sum * (1.0 / 17592186044416.0));
                st.drawn = b.i;
                const float s = at_draft / temp;
                if (s > -INFINITY && score_key(s) >= st.threshold) st.share = scaled_weight(s, st.m) / st.z;
                if (lists && sh.listed <= VD_LIST) st.listed = sh.listed;
                *out = st;
            }
            return;
        }
        st.threshold = row_threshold(sh, cluster, v, slice, temp, topk);
    }

    // Every kept logit of the row counts: the blocks' sums and best draws, each relative to its own largest.
    most = warp_max(most);
    if (lane == 0) sh.warp[warp] = most;
    __syncthreads();
    const float m = warp_max(lane < VD_WARPS ? sh.warp[lane] : -INFINITY) / temp;
    const Weights weight(temp, m);
    const unsigned threshold = st.threshold;
    float z = 0.f;
#pragma unroll
    for (int k = 0; k < VD_GROUPS; ++k) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (threshold && score_key(v[k][q] / temp) < threshold) v[k][q] = -INFINITY;
            if (v[k][q] > -INFINITY) z += weight(v[k][q]);
        }
    }
    z = block_sum(z, sh.red);
    Best b{-INFINITY, -1};
    if (draws) {
        // The largest of s + G, G = -log E, E = -log U. A token can pass the best score B so far only if E < exp(s - B), that is, since
        // exp(-y) >= 1 - y, if U > 1 - exp(s - B): one comparison (with a thousandth to spare) settles all but a few tokens.
        float spare = INFINITY;                              // exp(m - B)
#pragma unroll
        for (int k = 0; k < VD_GROUPS; ++k) {
            const int e = slice.token(k);
            if (e < a.vocab) {
                const uint4 w = philox4x32_10(make_uint4((unsigned)e >> 2, c1, stream, 0u), key2);
                const unsigned words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float u = philox_uniform(words[q]);
                    if (v[k][q] > -INFINITY && !(u <= 1.f - weight(v[k][q]) * spare)) b = better(b, Best{v[k][q] / temp - logf(-logf(u)), e + q});
                }
            }
            if (k == 0 || k == 1 || k == 3) spare = exp2f((m - warp_max(b.v)) * LOG2E) * 1.001f;
        }
        b = block_best<VD_WARPS>(b, sh.best);
    }
    if (tid == 0) {
        *cluster.map_shared_rank(&sh.m[rank], 0) = m;
        *cluster.map_shared_rank(&sh.z[rank], 0) = z;
        *cluster.map_shared_rank(&sh.part[rank], 0) = b;
    }
    cluster.sync();
    if (rank == 0 && warp == 0) {
        b = warp_best(lane < ctas ? sh.part[lane] : Best{0.f, -1});
        const float mine = lane < ctas ? sh.m[lane] : -INFINITY;
        st.m = warp_max(mine);
        st.z = warp_sum(lane < ctas && sh.z[lane] > 0.f ? sh.z[lane] * scaled_weight(mine, st.m) : 0.f);
        st.drawn = draws ? b.i : -1;
        const float s = at_draft / temp;
        if (s > -INFINITY && score_key(s) >= threshold) st.share = Weights(temp, st.m)(at_draft) / st.z;
        if (lane == 0) *out = st;
    }
}

// Decides the request by its rows; if a drawn draft failed, draws from what is left of p beyond q. JUDGED: clusters of blocks share that
// draw's row out; otherwise a warp a request.
constexpr int VF_THREADS = 256;
constexpr int VF_CTAS = 8;

template <bool JUDGED>
__global__ void __launch_bounds__(JUDGED ? VF_THREADS : 32) verify_kernel(VdArgs a) {
    __shared__ Best best_sh[VF_THREADS / 32], part_sh[VF_CTAS];
    __shared__ int held_sh;
    ti_grid_launch_dependents();
    ti_grid_wait();
    const int r = blockIdx.y, tid = threadIdx.x, D = a.max_drafts, rank = blockIdx.x;
    const int2 rows = rows_of(a, r);
    int* out = a.tokens + (size_t)r * (D + 1);
    const bool greedy = is_greedy(a, r);
    const int n = rows.y - 1;
    const bool judged = JUDGED && !greedy;                   // by the ratio of the probabilities
    const uint2 key2 = judged ? seed_of(a, r) : make_uint2(0u, 0u);
    const unsigned step = judged ? (unsigned)a.step[r] : 0u, stream = judged ? (unsigned)a.stream_id[r] : 0u;
    int fed = -1;                                            // lane j: the draft j
    if (tid < 32) {
        bool holds = false;
        if (tid < D) {
            float prob = 0.f;
            if (tid < n) {
                fed = a.token_ids[rows.x + tid + 1];
                const RowStats st = a.target[r * (D + 1) + tid];
                holds = fed >= 0 && fed == st.drawn;
                prob = greedy ? (holds ? 1.f : 0.f) : st.share;
                if (judged) {
                    const float q = a.draft[r * D + tid].share;
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
        const RowStats st = a.target[r * (D + 1) + held];
        b.i = st.drawn;
        if (JUDGED && judged && held < n) {
            const unsigned c1 = step + held;
            const RowStats ds = a.draft[r * D + held];
            const float temp = a.temperature[r];
            const float* x = a.logits + (size_t)(rows.x + held) * a.vocab;
            const float* y = a.draft_logits + r * a.draft_request + held * a.draft_place;
            const Weights pw(temp, st.m), qw(temp, ds.m);
            const float pz = st.z > 0.f ? 1.f / st.z : 0.f, qz = ds.z > 0.f ? 1.f / ds.z : 0.f;
            auto p_of = [&](float v) { return v > -INFINITY && (!st.threshold || score_key(v / temp) >= st.threshold) ? pw(v) * pz : 0.f; };
            auto q_of = [&](float v) { return v > -INFINITY && (!ds.threshold || score_key(v / temp) >= ds.threshold) ? qw(v) * qz : 0.f; };
            // an exponential race: the largest share / E, E = -log U
            auto race = [&](float share, int i) {
                if (!(share > 0.f)) return;
                const uint4 w = philox4x32_10(make_uint4((unsigned)i >> 2, c1, stream, 2u), key2);
                const unsigned words[4] = {w.x, w.y, w.z, w.w};
                b = better(b, Best{share / -logf(philox_uniform(words[i & 3])), i});
            };
            b.i = -1;
            if (st.listed >= 0) {                            // the threshold keeps few: the first block alone
                if (rank != 0) return;
                const Kept* list = a.kept + ((size_t)r * D + held) * VD_LIST;
                for (int i = tid; i < st.listed; i += VF_THREADS) race(scaled_weight(list[i].s, st.m) * pz - q_of(y[list[i].i]), list[i].i);
                b = block_best<VF_THREADS / 32>(b, best_sh);
            } else {
                cg::cluster_group cluster = cg::this_cluster();
                for (int i = rank * VF_THREADS + tid; i < a.vocab; i += VF_CTAS * VF_THREADS) race(p_of(x[i]) - q_of(y[i]), i);
                b = block_best<VF_THREADS / 32>(b, best_sh);
                cluster.sync();                              // every block runs
                if (tid == 0) *cluster.map_shared_rank(&part_sh[rank], 0) = b;
                cluster.sync();
                if (rank != 0) return;
                b = warp_best((tid & 31) < VF_CTAS ? part_sh[tid & 31] : Best{0.f, -1});
            }
            if (b.i < 0) {                                   // nothing of p lies beyond q (they differ by a rounding): p itself
                for (int i = tid; i < a.vocab; i += VF_THREADS) race(p_of(x[i]), i);
                b = block_best<VF_THREADS / 32>(b, best_sh);
            }
        }
    }
    if (rank == 0 && tid <= D) {
        const int token = rows.y > 0 && tid == held ? max(b.i, 0) : -1;
        out[tid] = rows.y > 0 && tid < held ? fed : token;
        if (tid == 0) a.counts[r] = rows.y > 0 ? held + 1 : 0;
    }
}

// How many blocks hold a row.
int row_ctas(int vocab) {
    int ctas = 1;
    while (ctas < VD_MAX_CTAS && (long long)ctas * VD_SLICE < vocab) ctas *= 2;
    return ctas;
}

}  // namespace

// Words (32 bits) of scratch a call needs, on a 16-byte boundary: what its rows leave for the kernel behind.
TI_API long long ti_verify_scratch_words(int requests, int max_drafts, int draft_logits) {
    return (long long)requests * ((2 * max_drafts + 1) * (long long)(sizeof(RowStats) / 4) + (draft_logits ? 2ll * VD_LIST * max_drafts : 0));
}

TI_API int ti_verify_drafts(int* tokens, int* counts, float* accept, const float* logits, const int* token_ids, const int* cu_rows,
                            int rows, int vocab, int requests, int max_drafts, const float* temperature, const int* topk,
                            const int* greedy, const long long* seed, const int* stream_id, const int* step, const float* draft_logits,
                            long long draft_request, long long draft_place, void* scratch, cudaStream_t stream) {
    TI_REQUIRE(rows >= 0 && vocab > 0 && requests >= 0 && requests <= 65535, "verify_drafts: bad sizes");
    TI_REQUIRE(max_drafts >= 0 && max_drafts <= VD_MAX_DRAFTS, "verify_drafts: at most %d drafts a request", VD_MAX_DRAFTS);
    TI_REQUIRE(vocab <= VD_MAX_CTAS * VD_SLICE, "verify_drafts: at most %d tokens in the vocabulary", VD_MAX_CTAS * VD_SLICE);
    TI_REQUIRE(temperature || !draft_logits, "verify_drafts: greedy requests have no use for draft logits");
    if (requests == 0) return 0;
    RowStats* target = (RowStats*)scratch;
    RowStats* draft = target + (size_t)requests * (max_drafts + 1);
    VdArgs a{logits, token_ids, cu_rows, temperature, topk, greedy, seed, stream_id, step, draft_logits, draft_request, draft_place,
             target, draft, (Kept*)(draft + (size_t)requests * max_drafts), tokens, counts, accept, rows, vocab, requests, max_drafts};
    const int ctas = row_ctas(vocab);
    if (ctas > 8) {
        static bool allowed[64] = {};
        int dev = -1;
        TI_REQUIRE(cudaGetDevice(&dev) == cudaSuccess, "verify_drafts: no device");
        if (dev >= 64 || !allowed[dev]) {
            TI_REQUIRE(cudaFuncSetAttribute(row_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess,
                       "verify_drafts: clusters of %d blocks are not allowed", ctas);
            if (dev < 64) allowed[dev] = true;
        }
    }
    ti_launch_clusters(row_kernel, dim3(ctas, max_drafts + 1 + (draft_logits ? max_drafts : 0), requests), ctas, VD_THREADS, stream, a);
    TI_CHECK_LAUNCH("verify_drafts: rows");
    if (draft_logits) ti_launch_clusters(verify_kernel<true>, dim3(VF_CTAS, requests), VF_CTAS, VF_THREADS, stream, a);
    else ti_launch(verify_kernel<false>, dim3(1, requests), 32, 0, stream, a);
    TI_CHECK_LAUNCH("verify_drafts");
    return 0;
}
