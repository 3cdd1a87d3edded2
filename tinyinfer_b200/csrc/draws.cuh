// What the kernels that choose tokens share: the counter-based random stream of a request (Philox-4x32-10), the order of
// floats as integers, and the better of two candidates (the larger value, on ties the lower index).
#pragma once
#include "common.cuh"

__device__ __forceinline__ uint4 philox_round(uint4 c, uint2 k) {      // (a product's two words in one instruction)
    const unsigned long long p0 = 0xD2511F53ull * c.x, p1 = 0xCD9E8D57ull * c.z;
    return make_uint4((unsigned)(p1 >> 32) ^ c.y ^ k.x, (unsigned)p1, (unsigned)(p0 >> 32) ^ c.w ^ k.y, (unsigned)p0);
}
__device__ __forceinline__ uint4 philox4x32_10(uint4 c, uint2 k) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        c = philox_round(c, k);
        k.x += 0x9E3779B9u;
        k.y += 0xBB67AE85u;
    }
    return c;
}
__device__ __forceinline__ unsigned word_of(uint4 w, int i) {       // word i mod 4
    const unsigned lo = (i & 1) ? w.y : w.x, hi = (i & 1) ? w.w : w.z;
    return (i & 2) ? hi : lo;
}
__device__ __forceinline__ float philox_uniform(unsigned word) {   // in (0, 1), exact in float32
    return ((float)(word >> 9) + 0.5f) * (1.0f / 8388608.0f);
}
__device__ __forceinline__ unsigned order_key(float v) {           // larger float -> larger key
    const unsigned b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Launches `kernel` on clusters of `ctas` blocks along x, otherwise as ti_launch does.
template <typename... KArgs, typename... Args>
cudaError_t ti_launch_clusters(void (*kernel)(KArgs...), dim3 grid, int ctas, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ti_pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

// Lets KERNEL run on clusters of more than 8 blocks on the current device (the record as in ti_allow_shared).
template <auto KERNEL>
cudaError_t ti_allow_wide_clusters() {
    constexpr int DEVICES = 64;
    static bool allowed[DEVICES] = {};
    int dev = -1;
    const cudaError_t got = cudaGetDevice(&dev);
    if (got != cudaSuccess || (dev < DEVICES && allowed[dev])) return got;
    const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev < DEVICES) allowed[dev] = true;
    return e;
}

struct Best { float v; int i; };
__device__ __forceinline__ Best better(Best a, Best b) {
    if (b.i < 0) return a;
    if (a.i < 0) return b;
    if (b.v > a.v || (b.v == a.v && b.i < a.i)) return b;
    return a;
}
__device__ __forceinline__ float key_value(unsigned key) {          // the inverse of order_key
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

// Radix select, one byte per pass from the top: the k-th largest of the keys that `each` hands out (it calls
// its argument once per key; every thread of the block calls select_kth with the same k). 0 if k <= 0.
// hist: 256 shared words; sel: 2 shared words. The counts of a pass go into the histogram warp by warp: lanes
// that hold the same byte count themselves once together (most logits share their sign and exponent, so a
// plain atomic per key would make a warp wait for itself 32 times over); the bin that holds the k-th largest
// is found by the first warp together (a suffix sum over lanes of eight bins each), not by one thread.
// One pass: sel[0] holds the bytes found so far (from the top), sel[1] which of the keys that begin with them,
// counted from the largest, is looked for; afterwards one byte more and the rank among those.
template <typename Each>
__device__ __forceinline__ void radix_pass(int pass, unsigned* hist, unsigned* sel, Each each) {
    {
        const int shift = 24 - 8 * pass;
        for (int i = threadIdx.x; i < 256; i += blockDim.x) hist[i] = 0u;
        __syncthreads();
        const unsigned prefix = sel[0];
        const unsigned mask = pass == 0 ? 0u : (0xFFFFFFFFu << (shift + 8));
        each([&](unsigned key) {
            if ((key & mask) == prefix) {
                const unsigned bin = (key >> shift) & 0xFFu;
                const unsigned same = __match_any_sync(__activemask(), bin);
                if ((threadIdx.x & 31) == (unsigned)(__ffs(same) - 1)) atomicAdd(&hist[bin], (unsigned)__popc(same));
            }
        });
        __syncthreads();
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x;
            unsigned mine[8], sum = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) { mine[i] = hist[8 * lane + i]; sum += mine[i]; }
            unsigned above = sum;                                  // keys in this lane's bins and all higher ones
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const unsigned v = __shfl_down_sync(0xffffffffu, above, off);
                if (lane + off < 32) above += v;
            }
            const unsigned remaining = sel[1];
            // the highest lane whose bins, with all above them, reach the k-th largest; lane 0 if none does
            const unsigned reach = __ballot_sync(0xffffffffu, above >= remaining);
            const int owner = reach ? 31 - __clz(reach) : 0;
            if (lane == owner) {
                unsigned left = remaining - (above - sum);         // still to find inside this lane's bins
                int b = 7;
                if (reach) {
                    for (; b > 0; --b) {
                        if (mine[b] >= left) break;
                        left -= mine[b];
                    }
                } else {
                    b = 0;                                         // fewer keys than k: bin 0, as the plain walk does
                    left = remaining;
                    for (int i = 255; i > 0; --i) left -= hist[i];
                }
                sel[0] = prefix | ((unsigned)(8 * lane + b) << shift);
                sel[1] = left;
            }
        }
        __syncthreads();
    }
}
template <typename Each>
__device__ __forceinline__ unsigned select_kth(int k, unsigned* hist, unsigned* sel, Each each) {
    if (k <= 0) return 0u;
    if (threadIdx.x == 0) { sel[0] = 0u; sel[1] = (unsigned)k; }
    for (int pass = 0; pass < 4; ++pass) radix_pass(pass, hist, sel, each);
    return sel[0];
}
