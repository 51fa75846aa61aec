// Next tokens from logits and given random numbers: temperature, top-k, top-p, min-p.
//
//   w_i = exp((x_i - max) / T),  Z = sum w_i;  order: x descending, index ascending
//   kept = front part with rank < top_k, mass before < top_p Z, w_i >= min_p (at least the first)
//   token = first i by index with (running kept mass) > u (kept mass)
//
// Every filter keeps a front part of one order, so together they keep everything above one logit and, of the tokens
// with exactly that logit, the first m by index.  That logit is found by a radix descent on the monotone image of the
// f32 bits, on counts and masses.  Masses are fixed point, w * 2^44 rounded to an integer, and exact from there on: sums
// do not depend on the order they are taken in, so a launch repeats to the bit, and a border is decided to 2^-44 of
// the largest weight (f32 sums would decide it to 2^-20 or so, which draws other tokens where many are alike).
#include "mono_common.cuh"

extern void mono_set_error(const char* fmt, ...);

namespace sampling {
using namespace mono;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr double kOne = 17592186044416.0;  // 2^44
typedef unsigned long long u64;

// Order-preserving image of a logit; NaN goes with -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x == x)) x = -INFINITY;
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);  // -0 counts as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }
constexpr uint32_t kKeyNegInf = 0x007FFFFFu;

struct Row {
    float mx;        // largest logit
    double inv_t;
    u64 k;           // rank below this
    double p;        // < 1: share of the mass
    u64 floor_w;     // weight at least this
    float u;
    bool greedy;
};

__device__ __forceinline__ u64 weight_of(float x, const Row& r) {
    if (x == r.mx) return (u64)kOne;
    const double d = ((double)x - (double)r.mx) * r.inv_t;
    if (!(d > -31.0)) return 0;  // below 2^-44; also -inf and NaN
    return (u64)(exp(d) * kOne + 0.5);
}
// floor(u W) for a 24-bit u below 1
__device__ __forceinline__ u64 share_of(float u, u64 W) {
    const int e = (int)((__float_as_uint(u) >> 23) & 0xFF);
    if (e == 0) return 0;  // below 2^-126
    const u64 mant = (__float_as_uint(u) & 0x7FFFFFu) | 0x800000u;  // u = mant 2^(e - 150)
    const int sh = 150 - e;                                        // at least 24 for u < 1
    const u64 lo = mant * W, hi = __umul64hi(mant, W);
    if (sh >= 128) return 0;
    if (sh >= 64) return hi >> (sh - 64);
    return (hi << (64 - sh)) | (lo >> sh);
}

__device__ __forceinline__ u64 block_sum_u64(u64 v, u64* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 s = 0;
    for (int i = 0; i < kWarps; ++i) s += red[i];
    return s;
}

template <typename T>
__device__ __forceinline__ float load_logit(const T* p, int i);
template <>
__device__ __forceinline__ float load_logit<float>(const float* p, int i) { return __ldg(p + i); }
template <>
__device__ __forceinline__ float load_logit<__nv_bfloat16>(const __nv_bfloat16* p, int i) { return __bfloat162float(p[i]); }

// One CTA per row.
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const mono_sample_args a) {
    pdl_prologue();
    __shared__ u64 red[kWarps], hist_m[256];
    __shared__ uint32_t hist_n[256], red32[kWarps];
    __shared__ u64 s_above, s_bin_mass;
    __shared__ uint32_t s_count, s_bin, s_bin_n;
    __shared__ int s_token;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x, V = a.vocab;
    const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld;
    // ---- the largest logit and its first index
    uint32_t kmax = 0;
    for (int i = tid; i < V; i += kThreads) kmax = max(kmax, key_of(load_logit(x, i)));
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (lane == 0) red32[warp] = kmax;
    if (tid == 0) s_token = INT32_MAX;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) kmax = max(kmax, red32[i]);
    if (kmax <= kKeyNegInf) {  // no logit above -inf
        if (tid == 0) {
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = -INFINITY;
        }
        return;
    }
    Row r;
    r.mx = logit_of(kmax);
    const float temp = a.temperature ? a.temperature[row] : 1.f;
    r.greedy = !(temp > 0.f);
    r.inv_t = r.greedy ? 1.0 : 1.0 / (double)temp;
    const int tk = a.top_k ? a.top_k[row] : 0;
    r.k = tk < 1 || tk > V ? (u64)V : (u64)tk;
    r.p = a.top_p && a.top_p[row] < 1.f ? fmax((double)a.top_p[row], 0.0) : 1.0;
    const float mp = a.min_p && a.min_p[row] > 0.f ? fminf(a.min_p[row], 1.f) : 0.f;
    r.floor_w = (u64)ceil((double)mp * kOne);
    r.u = a.u[row];
    if (!(r.u > 0.f)) r.u = 0.f;
    if (r.greedy) r.k = 1;
    // ---- the whole mass
    u64 z = 0;
    for (int i = tid; i < V; i += kThreads) z += weight_of(load_logit(x, i), r);
    z = block_sum_u64(z, red);
    // ---- the border: keys above `lo` bits in all, the bin [lo, lo + 2^shift) holds it
    // "mass before < top_p Z" for a whole number of units of mass: before < ceil(top_p Z)
    const u64 limit = r.p < 1.0 ? max((u64)ceil(r.p * (double)z), 1ull) : ~0ull;
    uint32_t lo = 0;      // the border key's known high bits
    uint32_t count = 0;   // tokens above
    u64 above = 0;        // their mass
    uint32_t ties = 0;    // tokens at the border key that are kept
    if (r.k < (u64)V || r.p < 1.0 || r.floor_w) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) { hist_n[tid] = 0; hist_m[tid] = 0; }
            __syncthreads();
            for (int i = tid; i < V; i += kThreads) {
                const float v = load_logit(x, i);
                const uint32_t k = key_of(v);
                if (shift == 24 || (k >> (shift + 8)) == (lo >> (shift + 8))) {
                    atomicAdd(&hist_n[(k >> shift) & 255], 1u);
                    atomicAdd(&hist_m[(k >> shift) & 255], weight_of(v, r));
                }
            }
            __syncthreads();
            if (tid == 0) {
                // down to the first bin that is not kept whole
                uint32_t c = count;
                u64 m = above;
                int b = 255;
                for (; b > 0; --b) {
                    const uint32_t low_key = lo | ((uint32_t)b << shift);
                    if (hist_n[b] == 0) continue;
                    if (c + hist_n[b] > r.k || m + hist_m[b] >= limit || weight_of(logit_of(low_key), r) < r.floor_w) break;
                    c += hist_n[b];
                    m += hist_m[b];
                }
                s_bin = b;
                s_count = c;
                s_above = m;
                s_bin_n = hist_n[b];
                s_bin_mass = hist_m[b];
            }
            __syncthreads();
            lo |= s_bin << shift;
            count = s_count;
            above = s_above;
        }
        // of the tokens with the border's logit: rank and mass before the j-th are count + j and above + j w
        const u64 w = weight_of(logit_of(lo), r);
        u64 m = s_bin_n;
        if (w < r.floor_w) m = 0;
        m = min(m, r.k - count);
        if (limit != ~0ull) m = above >= limit ? 0 : w == 0 ? m : min(m, (limit - above + w - 1) / w);
        ties = (uint32_t)m;
        if (count + ties == 0) ties = 1;
    }
    const u64 tie_w = weight_of(logit_of(lo), r);
    const u64 kept = (r.k < (u64)V || r.p < 1.0 || r.floor_w) ? above + ties * tie_w : z;
    const u64 target = r.u >= 1.f ? kept - 1 : share_of(r.u, kept);
    // ---- the draw: every warp sums a run of consecutive tokens; the run that holds the target walks itself
    const int run = (V + kWarps - 1) / kWarps, i0 = min(warp * run, V), i1 = min(i0 + run, V);
    const bool all = !(r.k < (u64)V || r.p < 1.0 || r.floor_w);
    uint32_t my_ties = 0;
    u64 mine = 0;
    for (int i = i0 + lane; i < i1; i += 32) {
        const float v = load_logit(x, i);
        const uint32_t k = key_of(v);
        if (all || k > lo) mine += weight_of(v, r);
        else if (k == lo) ++my_ties;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    my_ties = __reduce_add_sync(0xffffffffu, my_ties);
    __syncthreads();
    if (lane == 0) { red32[warp] = my_ties; red[warp] = mine; }
    __syncthreads();
    u64 before = 0;
    uint32_t ties_before = 0;
    auto kept_ties = [&](uint32_t first, uint32_t n) { return first >= ties ? 0u : min(n, ties - first); };
    for (int w = 0; w < warp; ++w) {
        before += red[w] + (all ? 0ull : kept_ties(ties_before, red32[w]) * tie_w);
        ties_before += red32[w];
    }
    const u64 after = before + mine + (all ? 0ull : kept_ties(ties_before, my_ties) * tie_w);
    if (before <= target && target < after) {  // one warp
        for (int b = i0; b < i1; b += 32) {
            const int i = b + lane;
            const float v = i < i1 ? load_logit(x, i) : -INFINITY;
            const uint32_t k = i < i1 ? key_of(v) : 0;
            const uint32_t tie_mask = __ballot_sync(0xffffffffu, !all && i < i1 && k == lo);
            const bool tie_kept = ties_before + __popc(tie_mask & ((1u << lane) - 1)) < ties;
            u64 w = 0;
            if (i < i1 && (all || k > lo || (k == lo && tie_kept))) w = weight_of(v, r);
            u64 s = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 t = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += t;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, w > 0 && before + s > target);
            if (hit) {
                const int token = b + __ffs(hit) - 1;
                if (lane == 0) {
                    const float xt = load_logit(x, token);
                    const double y = xt == r.mx ? 0.0 : ((double)xt - (double)r.mx) * r.inv_t;
                    a.tokens[row] = token;
                    if (a.logprobs) a.logprobs[row] = (float)(y - log((double)z / kOne));
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, s, 31);
            ties_before += __popc(tie_mask);
        }
    }
}

}  // namespace sampling

extern "C" int mono_sample_launch(const mono_sample_args* a, void* stream) {
    const char* who = "mono_sample_launch";
    if (!a || a->rows < 1 || a->rows > 65535 || a->vocab < 1 || a->vocab > MONO_SAMPLE_MAX_VOCAB) {
        mono_set_error("%s: 1..65535 rows of 1..%d logits required", who, MONO_SAMPLE_MAX_VOCAB);
        return MONO_E_ARG;
    }
    if (!a->logits || !a->u || !a->tokens || a->ld < a->vocab) {
        mono_set_error("%s: logits with rows at least vocab apart, u and tokens required", who);
        return MONO_E_ARG;
    }
    if ((reinterpret_cast<uintptr_t>(a->logits) & (a->logits_bf16 ? 1 : 3)) || (reinterpret_cast<uintptr_t>(a->tokens) & 7)) {
        mono_set_error("%s: logits and tokens must be aligned to their type", who);
        return MONO_E_ARG;
    }
    const cudaError_t e = a->logits_bf16 ? mono::launch_k(sampling::sample_kernel<__nv_bfloat16>, a->rows, sampling::kThreads, 0, (cudaStream_t)stream, *a)
                                         : mono::launch_k(sampling::sample_kernel<float>, a->rows, sampling::kThreads, 0, (cudaStream_t)stream, *a);
    if (e != cudaSuccess) mono_set_error("%s: %s", who, cudaGetErrorString(e));
    return (int)e;
}
