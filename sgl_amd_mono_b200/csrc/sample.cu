// Next tokens from logits and given random numbers: temperature, top-k, top-p, min-p.
//
//   w_i = exp((x_i - max) / T),  Z = sum w_i;  order: x descending, index ascending
//   kept = front part with rank < top_k, mass before < top_p Z, w_i >= min_p (at least the first)
//   token = first i by index with (running kept mass) > u (kept mass)
//
// Every filter keeps a front part of one order, so together they keep everything above one logit and, of the tokens
// with exactly that logit, the first m by index.  Masses are fixed point, w * 2^44 rounded to an integer, and exact from
// there on: sums do not depend on the order they are taken in, so a launch repeats to the bit, and a border is decided
// to 2^-44 of the largest weight (f32 sums would decide it to 2^-20 or so, which draws other tokens where many are
// alike).  A token whose weight rounds to 0 is never drawn, so it counts in no rank either.
//
// Layout: a cluster of eight CTAs per row (short or many rows: fewer); each reads its share of the row once from HBM into shared memory and all
// passes run on that.  The border is found in steps that all eight CTAs decide alike from merged histograms (read over
// distributed shared memory; one cluster barrier a step):
//   1. the largest logit;
//   2. Z, and a histogram over 1024 equal steps of log2 w of the tokens' number and of how far into its step each lies;
//      the weights of a step differ by 3 % and these two sums give its mass to 2^-11, so the border lies in one step as a
//      rule;
//   3. the mass above those steps, and a list of the logits in them.  Up to 256 of the row are sent to all CTAs and ranked
//      one against another, which ends the search; more go by keys (the order-preserving image of the f32 bits) into 1024
//      bins with counts and masses, and the bin that holds the border is searched again.
// Then each warp's run of kept mass says which warp walks to the token.
//
// Bound: latency.  For few rows of the cluster's barriers, and of code that a launch runs once.  Many rows go in waves of
// clusters, two CTAs an SM, whose loads, maxima and weights take turns and hardly cover each other: HBM alone would take 20
// us for 256 rows, the f64 pipe (some 12 operations a weight) 22.  Measured, 129280 f32 logits: 1 row 22 us, 16 rows with all
// filters 36 us, 256 rows, one in eight with top-p, 158 us (835 GB/s); without a filter 121 us, of bf16 logits 102 us; 129281
// logits, rows at any address, as 129280.  A row's CTAs live 12 us without a filter: 4 for the load, 1 for the maximum, 5 to
// 7 for Z; 30 with a top-p border deep in the bulk, whose rows are weighed a second time.  (Two CTAs an SM leave 64 registers a
// thread; the kernel of two CTAs a row spills 44 bytes of them.)
#include <cooperative_groups.h>

#include <cmath>

#include "mono_common.cuh"

extern void mono_set_error(const char* fmt, ...);

namespace sampling {
using namespace mono;
namespace cg = cooperative_groups;

constexpr int kCtas = 8;  // of a row, at most: the portable cluster size; a slice of the largest vocabulary fits shared memory
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kPerThread = kBins / kThreads;
constexpr double kOne = 17592186044416.0;  // 2^44
constexpr float kSteps = kBins / 44.001f;  // histogram steps per factor of two: weights down to 2^-44
typedef unsigned long long u64;
MONO_TL_DECLARE(tl_sample)

// Order-preserving image of a logit (NaN has been taken to -inf).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);  // -0 counts as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }
// The logit f for which x <= f says key_of(x) <= key.  One key has no logit, that of -0, and -0 compares as 0 does.
__device__ __forceinline__ float below_or_at(uint32_t key) { return logit_of(key == 0x7FFFFFFFu ? key - 1 : key); }
constexpr uint32_t kKeyNegInf = 0x007FFFFFu, kKeyInf = 0xFF800000u;

constexpr int kTable = 32, kCopies = 16;  // a copy of the table per pair of banks: looked up by all lanes, it has no conflicts
constexpr double kTwo52 = 4503599627370496.0;             // 2^52: a number below it, added, leaves its whole part in the mantissa
constexpr double kRound32 = 6755399441055744.0 / kTable;  // (2^52 + 2^51) / 32

struct Powers {
    double p[kTable];  // 2^(44 + i / 32)
};
struct Row {
    float mx;           // largest logit (finite)
    float c;            // log2(e) / T, f32: for histogram steps only
    double mx64, c64;   // the same, f64
    u64 k;              // rank below this
    u64 floor_w;        // weight at least this
    const double* tab;  // 2^(44 + i / 32), this lane's copy
};

// round(2^44 exp((x - mx) / T)).  y = (x - mx) log2(e) / T = n + i / 32 + r, 0 <= i < 32, |r| <= 1/64:
// 2^y = 2^n 2^(i/32) 2^r, the last by its series in r ln 2 (at most 0.0109: the sixth power's term is below 2^-48).  The
// f64 pipe bounds the passes that weigh, so what integers can do they do: the sign tests, the exponent, the sums.
__device__ __forceinline__ u64 weight_of(float x, const Row& r) {
    const double y = ((double)x - r.mx64) * r.c64;
    const double shifted = y + kRound32;  // rounded to a multiple of 1/32: the low word holds 32 y
    const int q = __double2loint(shifted);
    const double t = y - (shifted - kRound32);
    constexpr double L = 0.69314718055994530942;
    double e = fma(t, L * L * L * L * L / 120, L * L * L * L / 24);
    e = fma(t, e, L * L * L / 6);
    e = fma(t, e, L * L / 2);
    e = fma(t, e, L);
    e = fma(t, e, 1.0);
    e *= r.tab[(q & (kTable - 1)) * kCopies];
    // times 2^n, by the exponent.  At -45 and below (and for -inf) the exponent may leave its range: a high word of 0 leaves
    // a number next to 0.  y <= 0, so its high word, unsigned, grows with |y|.
    const int hi = __double2hiint(e) + ((q & ~(kTable - 1)) << 15);
    e = __hiloint2double((uint32_t)__double2hiint(y) < 0xC0468000u ? hi : 0, __double2loint(e));
    return (u64)__double_as_longlong(e + kTwo52) - (u64)__double_as_longlong(kTwo52);  // to a whole number, below 2^52
}
// floor(u W) for 0 <= u < 1
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
__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct Hist {
    uint32_t n[2][kBins], lo[2][kBins], hi[2][kBins];  // counts, and masses in two words; two sets, used in turn
};
constexpr int kRank = 256;  // tokens that are ranked one against another (0.8 us; a round of bins takes 3.5)
constexpr int kSlice = 20480;  // logits that a CTA holds beside another CTA on its SM
constexpr int kList = 64;  // logits of the border's first range that a warp lists
constexpr size_t kAfter = sizeof(Hist) + kWarps * kList * sizeof(uint16_t);  // shared memory behind the slice
// One word atomics are native in shared memory, 64-bit ones are not: the carry is taken from the value that was there.
__device__ __forceinline__ void hist_add(Hist& h, int set, int bin, uint32_t n, u64 w) {
    atomicAdd(&h.n[set][bin], n);
    const uint32_t wl = (uint32_t)w, old = atomicAdd(&h.lo[set][bin], wl);
    const uint32_t wh = (uint32_t)(w >> 32) + (old + wl < old ? 1u : 0u);
    if (wh) atomicAdd(&h.hi[set][bin], wh);
}

// CTA c's keys of the tokens to be ranked, in a set of the histograms that is not in use (the rest of it holds the ranked).
__device__ __forceinline__ uint32_t* candidates(Hist& h, int set, int c) {
    static_assert(kRank * kCtas <= 2 * kBins && kRank * 3 <= kBins, "fits a set");
    return c < kCtas / 2 ? &h.n[set][c * kRank] : &h.lo[set][(c - kCtas / 2) * kRank];
}

__device__ __forceinline__ uint32_t peer_address(const void* p, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ uint32_t ld_peer(const uint32_t* p, int rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_address(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void st_peer(uint32_t* p, int rank, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_address(p, rank)), "r"(v) : "memory");
}
// The CTAs' histograms of set `set`, added into set `set ^ 1` of all of them: each CTA adds its share of the bins and
// writes it to every CTA.  (Shared memory of other CTAs is read at some 8 bytes a cycle: with every CTA reading all
// bins of all others a level took 3 us.)  Barriers before and after.
template <int CTAS>
__device__ __forceinline__ void hist_merge(Hist& h, int set, int rank, cg::cluster_group& cluster) {
    if (CTAS == 1) {
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) { h.n[set ^ 1][i] = h.n[set][i]; h.lo[set ^ 1][i] = h.lo[set][i]; h.hi[set ^ 1][i] = h.hi[set][i]; }
        __syncthreads();
        return;
    }
    constexpr int kShare = kBins / CTAS;
    cluster.sync();
    for (int x = threadIdx.x; x < 2 * kShare; x += kThreads) {
        const int b = rank * kShare + (x & (kShare - 1));
        if (x < kShare) {
            uint32_t v[CTAS], n = 0;
#pragma unroll
            for (int c = 0; c < CTAS; ++c) v[c] = ld_peer(&h.n[set][b], c);
#pragma unroll
            for (int c = 0; c < CTAS; ++c) n += v[c];
#pragma unroll
            for (int c = 0; c < CTAS; ++c) st_peer(&h.n[set ^ 1][b], c, n);
        } else {
            uint32_t lo[CTAS], hi[CTAS];
            u64 m = 0;
#pragma unroll
            for (int c = 0; c < CTAS; ++c) { lo[c] = ld_peer(&h.lo[set][b], c); hi[c] = ld_peer(&h.hi[set][b], c); }
#pragma unroll
            for (int c = 0; c < CTAS; ++c) m += ((u64)hi[c] << 32) + lo[c];
#pragma unroll
            for (int c = 0; c < CTAS; ++c) { st_peer(&h.lo[set ^ 1][b], c, (uint32_t)m); st_peer(&h.hi[set ^ 1][b], c, (uint32_t)(m >> 32)); }
        }
    }
    cluster.sync();
}

// The histogram step of a weight above 0, and how far into the step it lies, in 2^-16 (clamped to the step).  Rounding to
// the nearest whole number by adding 2^23 + 2^22 keeps the order of the logits; f32 places a logit within 2^-12 of its
// true step number.
__device__ __forceinline__ int step_of(float x, const Row& r, uint32_t* within) {
    const float at = x == r.mx ? 0.f : fminf((r.mx - x) * r.c * kSteps, 2000.f);
    const int b = min(max(__float_as_int(at - 0.5f + 12582912.f) - 0x4B400000, 0), kBins - 1);
    *within = (uint32_t)(__float_as_int(fminf(fmaxf(at - (float)b, 0.f), 1.f) * 65535.f + 12582912.f) - 0x4B400000);
    return b;
}
// The sum of `v` over the threads before this one.
template <typename A>
__device__ __forceinline__ A block_before(A v, A* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    A s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const A t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    if (lane == 31) red[warp] = s;
    __syncthreads();
    A b = s - v;
    for (int i = 0; i < warp; ++i) b += red[i];
    return b;
}

// `slice`: logits of a CTA (a multiple of 4); runs: a warp's consecutive logits (a multiple of 128)
template <typename T, int CTAS>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(kThreads, 2) sample_kernel(const mono_sample_args a, int slice, int run, const __grid_constant__ Powers powers) {
    extern __shared__ __align__(16) float xs[];  // [slice], then the histograms and the warps' lists
    Hist& h = *reinterpret_cast<Hist*>(xs + slice);
    __shared__ u64 s_wsum[kWarps], red64[kWarps], s_z[CTAS], s_kept[CTAS], s_part[CTAS], s_cut[2];
    __shared__ uint32_t s_wties[kWarps], red32[kWarps], s_key[CTAS], s_num[CTAS], s_cnt[2];
    __shared__ float redf[2][kWarps];
    __shared__ int s_bin[2];
    __shared__ uint32_t s_found, s_cand[CTAS], s_border;
    __shared__ double s_tab[kTable * kCopies];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x / CTAS, V = a.vocab;
    const int rank = (int)cluster.block_rank();
    // The row's CTAs write into one another's shared memory once all of them are known to run: the wait for that comes
    // after the load.
    if (CTAS > 1) cluster.barrier_arrive();
    if (tid < kTable * kCopies) s_tab[tid] = powers.p[tid / kCopies];
    for (int i = tid; i < kBins; i += kThreads) { h.n[0][i] = 0; h.lo[0][i] = 0; h.hi[0][i] = 0; }
    if (tid == 0) { s_bin[0] = kBins; s_bin[1] = kBins; s_found = 0; s_border = 0; }
    MONO_TL(tl_sample, 0);
    pdl_prologue();
    MONO_TL(tl_sample, 1);
    const int first = min(rank * slice, V), count = min(slice, V - first);  // this CTA's tokens
    const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld + first;
    const float temp = a.temperature ? a.temperature[row] : 1.f;
    const int tk = a.top_k ? a.top_k[row] : 0;
    const float tp = a.top_p ? a.top_p[row] : 1.f, mp = a.min_p ? a.min_p[row] : 0.f;
    float u = a.u[row];
    // ---- the slice into shared memory, and its largest logit; places behind the vocabulary hold -inf
    float top = -INFINITY;
    {
        constexpr int N = sizeof(T) == 4 ? 4 : 8;  // logits of a 16-byte load
        auto clean = [&](float v) {  // fmaxf takes the number beside NaN
            v = fmaxf(v, -INFINITY);
            top = fmaxf(top, v);
            return v;
        };
        const int vecs = (reinterpret_cast<uintptr_t>(x) & 15) ? 0 : count / N;
        constexpr int B = 8;
        for (int v0 = tid; v0 < vecs; v0 += kThreads * B) {
            uint4 w[B];
#pragma unroll
            for (int j = 0; j < B; ++j) w[j] = __ldg(reinterpret_cast<const uint4*>(x) + min(v0 + j * kThreads, vecs - 1));
#pragma unroll
            for (int j = 0; j < B; ++j) {
                const int i = v0 + j * kThreads;
                if (i >= vecs) break;
                if (sizeof(T) == 4) {
                    reinterpret_cast<float4*>(xs)[i] = make_float4(clean(__uint_as_float(w[j].x)), clean(__uint_as_float(w[j].y)), clean(__uint_as_float(w[j].z)),
                                                                   clean(__uint_as_float(w[j].w)));
                } else {
                    const uint32_t ws[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
                    float f[8];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        f[2 * q] = clean(__uint_as_float(ws[q] << 16));
                        f[2 * q + 1] = clean(__uint_as_float(ws[q] & 0xFFFF0000u));
                    }
                    reinterpret_cast<float4*>(xs)[2 * i] = make_float4(f[0], f[1], f[2], f[3]);
                    reinterpret_cast<float4*>(xs)[2 * i + 1] = make_float4(f[4], f[5], f[6], f[7]);
                }
            }
        }
        for (int i = vecs * N + tid; i < slice; i += kThreads) xs[i] = clean(i < count ? (float)x[i] : -INFINITY);
    }
    uint32_t kmax = key_of(top);
    MONO_TL(tl_sample, 2);
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (lane == 0) red32[warp] = kmax;
    __syncthreads();
    if (CTAS > 1) cluster.barrier_wait();
    if (tid < CTAS) {
        for (int i = 0; i < kWarps; ++i) kmax = max(kmax, red32[i]);
        *cluster.map_shared_rank(&s_key[rank], tid) = kmax;
    }
    cluster.sync();
    MONO_TL(tl_sample, 3);
    kmax = 0;
    for (int i = 0; i < CTAS; ++i) kmax = max(kmax, s_key[i]);
    if (kmax <= kKeyNegInf) {  // no logit above -inf: all CTAs of the row leave
        if (tid == 0 && rank == 0) {
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = -INFINITY;
        }
        return;
    }
    if (kmax == kKeyInf) {  // beside an infinite logit nothing has weight: its likes become 0, the others -inf
        for (int i = tid; i < slice; i += kThreads) xs[i] = xs[i] == INFINITY ? 0.f : -INFINITY;
        kmax = key_of(0.f);
        __syncthreads();
    }
    Row r;
    r.tab = s_tab + (lane & (kCopies - 1));
    r.mx = logit_of(kmax);
    const bool greedy = !(temp > 0.f);
    // Temperatures beyond 2^-100 and 2^100 weigh no logits otherwise than those do, short of logits of 2^-93 or 2^55.
    r.c64 = greedy ? 1.4426950408889634 : 1.4426950408889634 / fmin(fmax((double)temp, 7.888609052210118e-31), 1.2676506002282294e30);
    r.c = (float)r.c64;
    r.mx64 = (double)r.mx;
    r.k = greedy || mp > 1.f ? 1ull : tk < 1 || tk > V ? (u64)V : (u64)tk;
    const double p = !greedy && tp < 1.f ? fmax((double)tp, 0.0) : 1.0;
    r.floor_w = !greedy && mp > 0.f ? (u64)ceil((double)fminf(mp, 1.f) * kOne) : 0ull;  // (above 1: no weight passes, and the first stays)
    const bool filtered = r.k < (u64)V || p < 1.0 || r.floor_w;
    const bool search = filtered && r.k != 1;  // with rank 0 alone the border is the largest logit
    // ---- Z, and the histogram of counts over steps of log2 w
    const int i0 = min(warp * run, slice), i1 = min(i0 + run, slice);
    {
        u64 z = 0;
        for (int i = i0 + lane * 4; i < i1; i += 256) {  // eight weights at a time: f64 arithmetic answers late
            const bool second = i + 128 < i1;
            const float4 a4 = *reinterpret_cast<const float4*>(xs + i), b4 = second ? *reinterpret_cast<const float4*>(xs + i + 128) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            const float v[8] = {a4.x, a4.y, a4.z, a4.w, b4.x, b4.y, b4.z, b4.w};
            u64 w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = weight_of(v[j], r);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                z += w[j];
                if (search && w[j] != 0) {
                    uint32_t within;
                    const int b = step_of(v[j], r, &within);
                    atomicAdd(&h.n[0][b], 1u);
                    atomicAdd(&h.lo[0][b], within);  // at most 49152 x 65535: below 2^32
                }
            }
        }
        z = warp_sum_u64(z);
        if (lane == 0) s_wsum[warp] = z;
    }
    __syncthreads();
    MONO_TL(tl_sample, 4);
    if (tid < CTAS) {
        u64 z = 0;
        for (int i = 0; i < kWarps; ++i) z += s_wsum[i];
        *cluster.map_shared_rank(&s_z[rank], tid) = z;
    }
    if (search) hist_merge<CTAS>(h, 0, rank, cluster); else cluster.sync();
    MONO_TL(tl_sample, 5);
    u64 Z = 0;
    for (int i = 0; i < CTAS; ++i) Z += s_z[i];
    // kept: keys above khi; of the keys klo .. khi (one key, or one token) the first `ties` of `tied`
    uint32_t khi = 0, klo = 1, tied = 0, ties = 0;
    u64 kept = Z, tie_w = 0;
    bool all = !filtered;
    u64 run_above = 0;       // of this warp's run: the mass above the range that the keys were first searched in,
    float first_hi = 0.f;    // which ends here
    // The run's logits of that range, as places in the run: a few of a hundred as a rule, and all that later steps look at.
    uint16_t* list = reinterpret_cast<uint16_t*>(&h + 1) + warp * kList;
    int listed = kList + 1;  // more than kList: not all are there, and later steps walk the run
    if (filtered && !search) {
        khi = klo = kmax;
        kept = tie_w = (u64)kOne;
        ties = 1;
        tied = 2;  // or more, or no more than one
    }
    if (search) {
        // "mass before < p Z", for masses in whole units
        const u64 limit = p < 1.0 ? max((u64)ceil(p * (double)Z), 1ull) : ~0ull;
        // ---- bounds of the border among the steps
        uint32_t n_before[kPerThread + 1];
        {
            const uint2 n2 = *reinterpret_cast<const uint2*>(&h.n[1][tid * kPerThread]);
            const uint32_t n[kPerThread] = {n2.x, n2.y};
            static_assert(kPerThread == 2, "two bins per thread");
            const uint2 l2 = *reinterpret_cast<const uint2*>(&h.lo[1][tid * kPerThread]), h2 = *reinterpret_cast<const uint2*>(&h.hi[1][tid * kPerThread]);
            const float f[kPerThread] = {((float)h2.x * 65536.f + (float)l2.x * (1.f / 65536.f)), ((float)h2.y * 65536.f + (float)l2.y * (1.f / 65536.f))};
            // A weight f steps into a step is 2^(-f / kSteps) of the step's first: 1 - a f, plus at most (a f)^2 / 2 <= a^2 / 2 f.
            constexpr float a = 0.69314718f / kSteps, a2 = a * a * 0.5f;
            float top[kPerThread + 1], m_lo[kPerThread], m_hi[kPerThread];
#pragma unroll
            for (int j = 0; j <= kPerThread; ++j) top[j] = exp2f(-(float)(tid * kPerThread + j) / kSteps);
#pragma unroll
            for (int j = 0; j < kPerThread; ++j) {
                m_lo[j] = fmaxf(top[j] * ((float)n[j] - a * f[j]), 0.f);
                m_hi[j] = top[j] * ((float)n[j] - a * f[j] + a2 * f[j]);
            }
            uint32_t c = block_before<uint32_t>(n[0] + n[1], red32);
            float hi = block_before<float>(m_hi[0] + m_hi[1], redf[0]), lo = block_before<float>(m_lo[0] + m_lo[1], redf[1]);
            // f32 sums of at most 1024 terms (2^-14 at worst), the places' 2^-12 of a step (2^-17 of a weight) and their
            // rounding: 2^-12 covers them.  The last step also holds weights below it, 2^-44 of the largest each.
            constexpr float up = 1.f + 0x1p-12f, down = 1.f - 0x1p-12f;
            const float lim = limit == ~0ull ? INFINITY : (float)((double)limit / kOne), fl = (float)((double)r.floor_w / kOne);
#pragma unroll
            for (int j = 0; j < kPerThread; ++j) {
                n_before[j] = c;
                c += n[j];
                hi += m_hi[j];
                lo += m_lo[j];
                const int b = tid * kPerThread + j;
                if (c > r.k || hi * up >= lim || top[j + 1] * down < fl) atomicMin(&s_bin[0], b);  // may not be kept whole
                if (c > r.k || lo * down >= lim || top[j] * up < fl) atomicMin(&s_bin[1], b);      // the border is not behind it
            }
            n_before[kPerThread] = c;
        }
        __syncthreads();
        const int b0 = s_bin[0], b1 = min(s_bin[1], kBins - 1);
        if (b0 / kPerThread == tid) s_cnt[0] = b0 % kPerThread ? n_before[1] : n_before[0];
        if (b1 / kPerThread == tid) s_cnt[1] = b1 % kPerThread ? n_before[2] : n_before[1];
        __syncthreads();
        uint32_t in_range = s_cnt[1] - s_cnt[0];  // as the steps were counted
        if (b0 >= kBins) {
            all = true;
        } else {
            // the steps' range of logits, with room for the rounding of the step's number
            const double per = 1.0 / ((double)r.c * (double)kSteps);
            float xh = b0 == 0 ? r.mx : (float)((double)r.mx - ((double)b0 - 0x1p-10) * per);
            float xl = (float)((double)r.mx - ((double)(b1 + 1) + 0x1p-10) * per);
            if (!(xh <= r.mx)) xh = r.mx;
            if (!(xl <= xh)) xl = -INFINITY;  // no number: infinite temperature, infinite logits
            khi = min(key_of(xh) + 2u, kmax);
            // (the last step also holds what lies behind it)
            klo = b1 < kBins - 1 && key_of(xl) > kKeyNegInf + 2u ? key_of(xl) - 2u : kKeyNegInf + 1u;
            u64 above = 0;
            uint32_t n_above = 0;
            MONO_TL(tl_sample, 6);
            int idle = 0;  // the histograms' set that no CTA of the row reads now
            // One key, or one token, holds the border: of its `tied` the first `ties` are kept.
            auto settle = [&]() {
                // rank and mass before the j-th of them are n_above + j and above + j tie_w
                u64 t = tied;
                if (tie_w < r.floor_w) t = 0;
                t = min(t, r.k - n_above);
                if (limit != ~0ull) t = above >= limit ? 0 : min(t, (limit - above + tie_w - 1) / tie_w);
                if (n_above + t == 0) t = 1;
                ties = (uint32_t)t;
                kept = above + t * tie_w;
            };
            for (int level = 1;; ++level) {
                const float fhi = below_or_at(khi), flo = logit_of(klo);  // order as the keys do, and cost nothing to compare
                if (level == 1) {  // what is above the range is weighed, what is in it listed
                    u64 m_ab = 0;
                    uint32_t n_ab = 0;
                    int found = 0;
                    for (int b = i0; b < i1; b += 256) {  // whole warps: the lanes vote
                        float v[8];
                        bool over = false, near = false;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const int i = b + q * 128 + lane * 4;
                            const float4 v4 = i < i1 ? *reinterpret_cast<const float4*>(xs + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                            v[4 * q] = v4.x; v[4 * q + 1] = v4.y; v[4 * q + 2] = v4.z; v[4 * q + 3] = v4.w;
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            over = over || v[j] > fhi;
                            near = near || (v[j] >= flo && v[j] <= fhi);
                        }
                        if (__any_sync(0xffffffffu, over)) {
                            u64 w[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) w[j] = weight_of(v[j], r);
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const u64 kept_w = v[j] > fhi ? w[j] : 0;  // surely kept
                                m_ab += kept_w;
                                n_ab += kept_w != 0;
                            }
                        }
                        if (!__any_sync(0xffffffffu, near)) continue;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const bool here = v[j] >= flo && v[j] <= fhi;
                            const unsigned in = __ballot_sync(0xffffffffu, here);
                            const int at = found + __popc(in & ((1u << lane) - 1));
                            if (here && at < kList) list[at] = (uint16_t)(b - i0 + (j >> 2) * 128 + lane * 4 + (j & 3));
                            found += __popc(in);
                        }
                    }
                    listed = found;
                    m_ab = warp_sum_u64(m_ab);
                    n_ab = __reduce_add_sync(0xffffffffu, n_ab);
                    if (lane == 0) { red64[warp] = m_ab; red32[warp] = n_ab; }
                    run_above = m_ab;
                    first_hi = fhi;
                    __syncwarp();
                }
                bool summed = level > 1;
                auto sum_above = [&]() {
                    for (int i = 0; i < CTAS; ++i) { above += s_part[i]; n_above += s_num[i]; }
                    summed = true;
                };
                auto send_above = [&]() {
                    u64 m = 0;
                    uint32_t n = 0;
                    for (int i = 0; i < kWarps; ++i) { m += red64[i]; n += red32[i]; }
                    *cluster.map_shared_rank(&s_part[rank], tid) = m;
                    *cluster.map_shared_rank(&s_num[rank], tid) = n;
                };
                // ---- few tokens left: all CTAs get all of them, and rank them
                if (in_range <= kRank) {
                    if (listed <= kList) {
                        for (int b = 0; b < listed; b += 32) {
                            const float v = b + lane < listed ? xs[i0 + list[b + lane]] : -INFINITY;
                            const bool here = v >= flo && v <= fhi && weight_of(v, r) != 0;
                            const unsigned in = __ballot_sync(0xffffffffu, here);
                            uint32_t at = lane == 0 && in ? atomicAdd(&s_found, __popc(in)) : 0;
                            at = __shfl_sync(0xffffffffu, at, 0) + __popc(in & ((1u << lane) - 1));
                            if (here && at < kRank) {
#pragma unroll
                                for (int c = 0; c < CTAS; ++c) st_peer(candidates(h, idle, rank) + at, c, key_of(v));
                            }
                        }
                    } else if (lane == 0) {
                        atomicAdd(&s_found, kRank + 1);
                    }
                    __syncthreads();
                    if (tid < CTAS) {
                        *cluster.map_shared_rank(&s_cand[rank], tid) = s_found;
                        if (level == 1) send_above();
                    }
                    cluster.sync();
                    if (tid == 0) s_found = 0;
                    if (!summed) sum_above();
                    uint32_t total = 0;
                    for (int c = 0; c < CTAS; ++c) total += min(s_cand[c], (uint32_t)kRank + 1);
                    if (total <= kRank) {
                        uint32_t* keys = h.hi[idle];
                        u64* ws = reinterpret_cast<u64*>(h.hi[idle] + kRank);
                        uint32_t from = 0;
                        for (int c = 0; c < CTAS; ++c) {
                            if (tid < (int)s_cand[c]) {
                                const uint32_t key = candidates(h, idle, c)[tid];
                                keys[from + tid] = key;
                                ws[from + tid] = weight_of(logit_of(key), r);
                            }
                            from += s_cand[c];
                        }
                        __syncthreads();
                        static_assert(2 * kRank <= kThreads, "two threads per token");
                        const int i = tid >> 1;
                        uint32_t n_more = 0, alike = 0;
                        u64 m_more = 0;
                        const uint32_t key = i < (int)total ? keys[i] : 0xFFFFFFFFu;
                        for (int j = tid & 1; j < (int)total; j += 2) {
                            const uint32_t kj = keys[j];
                            if (kj > key) { ++n_more; m_more += ws[j]; }
                            alike += kj == key;
                        }
                        n_more += __shfl_xor_sync(0xffffffffu, n_more, 1);
                        alike += __shfl_xor_sync(0xffffffffu, alike, 1);
                        m_more += __shfl_xor_sync(0xffffffffu, m_more, 1);
                        const u64 w = i < (int)total ? ws[i] : 0, m_to = above + m_more + alike * w;
                        const uint32_t n_to = n_above + n_more + alike;  // rank and mass up to this key
                        if (i < (int)total) {
                            if (n_to > r.k || m_to >= limit || w < r.floor_w) atomicMax(&s_border, key);
                            if (n_more + alike == total) s_part[0] = m_to;
                        } else if (total == 0 && tid == 0) {
                            s_part[0] = above;
                        }
                        __syncthreads();
                        if (s_border == 0) {  // everything in the range is kept
                            kept = s_part[0];
                            khi = klo - 1;  // and nobody is tied
                            break;
                        }
                        if (i < (int)total && key == s_border) {
                            red32[0] = alike;
                            red32[1] = n_above + n_more;
                            red64[0] = w;
                            red64[1] = above + m_more;
                        }
                        __syncthreads();
                        khi = klo = s_border;
                        tied = red32[0];
                        n_above = red32[1];
                        tie_w = red64[0];
                        above = red64[1];
                        settle();
                        break;
                    }
                }
                const int set = (level & 1) ^ 1;
                const uint32_t width = khi - klo;
                const int sh = width < kBins ? 0 : 22 - __clz(width);
                for (int i = tid; i < kBins; i += kThreads) { h.n[set][i] = 0; h.lo[set][i] = 0; h.hi[set][i] = 0; }
                if (tid == 0) s_bin[set] = kBins;
                __syncthreads();
                // adds the logits of the range that a warp's lanes hold
                auto add = [&](float v) {
                    bool here = v >= flo && v <= fhi;
                    if (!__any_sync(0xffffffffu, here)) return;
                    const u64 wi = weight_of(v, r);
                    here = here && wi > 0;
                    const unsigned in = __ballot_sync(0xffffffffu, here);
                    if (in == 0) return;
                    const int bin = (int)((khi - key_of(v)) >> sh), lead = __ffs(in) - 1;
                    const int lb = __shfl_sync(0xffffffffu, bin, lead);
                    if (__popc(in) > 4 && __all_sync(0xffffffffu, !here || bin == lb)) {  // many equal logits: one addition for all
                        const u64 sum = warp_sum_u64(here ? wi : 0);
                        if (lane == lead) hist_add(h, set, bin, __popc(in), sum);
                    } else if (here) {
                        hist_add(h, set, bin, 1, wi);
                    }
                    __syncwarp();
                };
                if (listed <= kList) {
                    for (int b = 0; b < listed; b += 32) add(b + lane < listed ? xs[i0 + list[b + lane]] : -INFINITY);
                } else {
                    for (int b = i0; b < i1; b += 32) add(b + lane < i1 ? xs[b + lane] : -INFINITY);
                }
                __syncthreads();
                if (!summed && tid < CTAS) send_above();
                hist_merge<CTAS>(h, set, rank, cluster);
                idle = set;
                MONO_TL(tl_sample, 5 + 2 * level);
                if (!summed) sum_above();
                const uint2 n2 = *reinterpret_cast<const uint2*>(&h.n[set ^ 1][tid * kPerThread]), l2 = *reinterpret_cast<const uint2*>(&h.lo[set ^ 1][tid * kPerThread]),
                            h2 = *reinterpret_cast<const uint2*>(&h.hi[set ^ 1][tid * kPerThread]);
                const uint32_t n[kPerThread] = {n2.x, n2.y};
                const u64 m[kPerThread] = {((u64)h2.x << 32) + l2.x, ((u64)h2.y << 32) + l2.y};
                uint32_t c = n_above + block_before<uint32_t>(n[0] + n[1], red32);
                u64 mass = above + block_before<u64>(m[0] + m[1], red64);
                uint32_t c_at[kPerThread];
                u64 m_at[kPerThread];
                int mine = -1;
#pragma unroll
                for (int j = 0; j < kPerThread; ++j) {
                    c_at[j] = c;
                    m_at[j] = mass;
                    c += n[j];
                    mass += m[j];
                    const int b = tid * kPerThread + j;
                    if (n[j] == 0 || mine >= 0) continue;
                    const uint32_t top = khi - ((uint32_t)b << sh);
                    const uint32_t low = top - klo < (1u << sh) ? klo : top - ((1u << sh) - 1);
                    if (c > r.k || mass >= limit || weight_of(logit_of(low), r) < r.floor_w) mine = j;
                }
                MONO_TL(tl_sample, 6 + 2 * level);
                if (mine >= 0) atomicMin(&s_bin[set], tid * kPerThread + mine);
                __syncthreads();
                const int b = s_bin[set];
                if (b >= kBins) {  // everything in the range is kept
                    if (tid == kThreads - 1) { s_cut[set] = mass; s_cnt[set] = c; }
                    __syncthreads();
                    kept = s_cut[set];
                    khi = klo - 1;  // and nobody is tied
                    break;
                }
                if (tid == b / kPerThread) {
                    const int j = b % kPerThread;
                    s_cut[set] = j ? m_at[1] : m_at[0];
                    s_cnt[set] = j ? c_at[1] : c_at[0];
                    red64[0] = j ? m[1] : m[0];
                    red32[0] = j ? n[1] : n[0];
                }
                __syncthreads();
                above = s_cut[set];
                n_above = s_cnt[set];
                const u64 bin_m = red64[0];
                tied = red32[0];
                khi -= (uint32_t)b << sh;
                klo = khi - klo < (1u << sh) ? klo : khi - ((1u << sh) - 1);
                if (sh == 0 || tied == 1) {
                    tie_w = bin_m / tied;
                    settle();
                    break;
                }
                in_range = tied;
                __syncthreads();  // red32 / red64 have been read
            }
        }
    }
    MONO_TL(tl_sample, 13);
    if (!(u > 0.f)) u = 0.f;
    const u64 target = u >= 1.f ? kept - 1 : share_of(u, kept);
    // ---- the draw: every warp's run of kept mass; where only some of the tied tokens are kept, their number apart
    const bool some = !all && ties > 0 && ties < tied;
    if (!all && !some && ties == tied) khi = klo - 1;  // all of the tied are kept: so is every key from klo on
    if (!all) {
        u64 m = 0;
        uint32_t t = 0;
        const float fhi = below_or_at(khi), flo = logit_of(klo);
        auto take = [&](float v) {  // what lies above the first range has been added up
            if (v > fhi) {
                if (v <= first_hi) m += weight_of(v, r);
            } else if (some && v >= flo) {
                ++t;
            }
        };
        if (listed <= kList) {
            for (int b = lane; b < listed; b += 32) take(xs[i0 + list[b]]);
        } else {
            for (int i = i0 + lane * 4; i < i1; i += 128) {
                const float4 v4 = *reinterpret_cast<const float4*>(xs + i);
                take(v4.x);
                take(v4.y);
                take(v4.z);
                take(v4.w);
            }
        }
        m = warp_sum_u64(m) + run_above;
        t = __reduce_add_sync(0xffffffffu, t);
        if (lane == 0) { s_wsum[warp] = m; s_wties[warp] = t; }
        __syncthreads();
        if (tid < CTAS) {
            u64 sm = 0;
            uint32_t st = 0;
            for (int i = 0; i < kWarps; ++i) { sm += s_wsum[i]; st += s_wties[i]; }
            // (not into s_z: without a search no barrier lies behind the other CTAs' reading of Z)
            *cluster.map_shared_rank(&s_kept[rank], tid) = sm;
            *cluster.map_shared_rank(&s_key[rank], tid) = st;
        }
        cluster.sync();
    }
    MONO_TL(tl_sample, 14);
    // from here on a CTA reads only what is its own
    u64 before = 0;
    uint32_t t_before = 0;
    auto kept_of = [&](uint32_t from, uint32_t n) { return some && from < ties ? (u64)min(n, ties - from) * tie_w : 0ull; };
    const u64* sums = all ? s_z : s_kept;
    for (int c = 0; c < rank; ++c) {
        before += sums[c];
        if (some) { before += kept_of(t_before, s_key[c]); t_before += s_key[c]; }
    }
    for (int w = 0; w < warp; ++w) {
        before += s_wsum[w];
        if (some) { before += kept_of(t_before, s_wties[w]); t_before += s_wties[w]; }
    }
    const u64 after = before + s_wsum[warp] + (some ? kept_of(t_before, s_wties[warp]) : 0ull);
    if (before <= target && target < after) {  // one warp of the eight CTAs
        for (int b = i0; b < i1; b += 128) {
            const float4 v4 = *reinterpret_cast<const float4*>(xs + min(b + lane * 4, i1 - 4));
            const float v[4] = {v4.x, v4.y, v4.z, v4.w};
            const bool in = b + lane * 4 < i1;
            u64 w[4];
            uint32_t tie = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t k = key_of(v[j]);
                w[j] = in && (all || k > khi) ? weight_of(v[j], r) : 0;
                if (in && some && k <= khi && k >= klo) tie |= 1u << j;
            }
            if (some) {
                uint32_t n = __popc(tie), s = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t t = __shfl_up_sync(0xffffffffu, s, o);
                    if (lane >= o) s += t;
                }
                uint32_t at = t_before + s - n;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (tie >> j & 1) w[j] = at++ < ties ? tie_w : 0;
                t_before += __shfl_sync(0xffffffffu, s, 31);
            }
            const u64 own = w[0] + w[1] + w[2] + w[3];
            u64 s = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 t = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += t;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, before + s > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    u64 at = before + s - own;
                    int j = 0;
                    while (j < 3 && at + w[j] <= target) at += w[j++];
                    const float xt = v[j];
                    const double y = xt == r.mx ? 0.0 : ((double)xt - (double)r.mx) * r.c64 * 0.69314718055994530942;
                    a.tokens[row] = first + b + lane * 4 + j;
                    if (a.logprobs) a.logprobs[row] = (float)(y - log((double)Z / kOne));
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, s, 31);
        }
    }
    MONO_TL(tl_sample, 15);
}

template <typename T, int CTAS>
static cudaError_t launch_with(const mono_sample_args* a, cudaStream_t st) {
    int slice = (a->vocab + CTAS - 1) / CTAS;
    slice = (slice + 7) & ~7;  // slices start on 16-byte addresses where the row does
    int run = (slice + kWarps - 1) / kWarps;
    run = (run + 127) & ~127;
    const size_t smem = (size_t)slice * 4 + kAfter;
    static std::atomic<uint64_t> attr_once{0};  // bit d: set on device d
    if (attr_needed(attr_once)) {
        const cudaError_t e = cudaFuncSetAttribute(sample_kernel<T, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (CTAS < kCtas ? kSlice : MONO_SAMPLE_MAX_VOCAB / kCtas) * 4 + (int)kAfter);
        if (e != cudaSuccess) return e;
        attr_done(attr_once);
    }
    static const Powers powers = [] {  // (made by every CTA, they cost its start a microsecond)
        Powers w;
        for (int i = 0; i < kTable; ++i) w.p[i] = std::exp2(44.0 + i / (double)kTable);
        return w;
    }();
    return launch_k(sample_kernel<T, CTAS>, a->rows * CTAS, kThreads, smem, st, *a, slice, run, powers);
}
// CTAs of a row.  One where it holds a short row: no barriers between CTAs, and nothing to merge.  Fewer than eight where there
// are more rows than clusters run at once (two CTAs an SM) and a smaller cluster holds the row.  Measured with filters, us by
// CTAs and by clusters of eight: 1 row of 4000 logits 11.6 and 12.8, of 8000 14.8 and 13.2; 24 rows of 8000 16.7 and 18.1, of
// 16000 24.4 and 19.1; 256 rows of 1000 14 and 107, of 20000 41 and 120; by two CTAs 256 rows of 40000 75 and 153, by four 256
// rows of 80000 129 and 188.
template <typename T>
static cudaError_t launch(const mono_sample_args* a, cudaStream_t st) {
    const int sms = mono_sm_count() > 0 ? mono_sm_count() : 148;
    if (a->vocab <= 4096 || (a->vocab <= 8192 && a->rows * kCtas > sms)) return launch_with<T, 1>(a, st);
    int ctas = kCtas;
    while (ctas > 1 && a->rows * ctas > 2 * sms && a->vocab <= kSlice * (ctas / 2)) ctas /= 2;
    return ctas == 1 ? launch_with<T, 1>(a, st) : ctas == 2 ? launch_with<T, 2>(a, st) : ctas == 4 ? launch_with<T, 4>(a, st) : launch_with<T, kCtas>(a, st);
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
    const cudaError_t e = a->logits_bf16 ? sampling::launch<__nv_bfloat16>(a, (cudaStream_t)stream) : sampling::launch<float>(a, (cudaStream_t)stream);
    if (e != cudaSuccess) mono_set_error("%s: %s", who, cudaGetErrorString(e));
    return (int)e;
}

#ifdef MONO_TIMELINE
// Copies the kernel's stamps of the last launch to `out` (MONO_TL_CTAS x MONO_TL_POINTS); blocks the host.
extern "C" int mono_timeline_read_sample(unsigned long long* out, int* ctas, int* points) {
    *ctas = MONO_TL_CTAS;
    *points = MONO_TL_POINTS;
    return (int)cudaMemcpyFromSymbol(out, sampling::tl_sample, sizeof(unsigned long long) * MONO_TL_CTAS * MONO_TL_POINTS);
}
#endif
