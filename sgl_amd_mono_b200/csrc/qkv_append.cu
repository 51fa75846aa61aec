// Rows of the fused q | k | v projection -> normed and rotated queries, and keys and values in the paged E4M3 cache.
//
// Per q and k head:  y = x / sqrt(mean(x^2) + eps) * (1 + g)          (no norm where g is absent)
//                    (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin) on the first R dims, pairs (i, i + R/2) or (2i, 2i+1)
// q is stored as bf16, k as E4M3(y / k_scale), v as E4M3(x / v_scale), saturating.  Everything between the load and the
// store is f32 with one rounding at the store; the step kernel of gqa.cu, which also makes the index keys, rounds to
// bf16 after the norm and after the rotation instead.
//
// Bound: memory.  A token's row is read once and written once (bf16 q, one byte per K and V value).  Sixteen lanes hold
// a head, eight dims (16 bytes) each, so a warp takes two heads at a time and a norm is four shuffles.  Four pairs of heads
// are in flight, and what a token and kind multiply by is made once for all its heads.  Measured (48 q heads on 8, B200):
// 16384 tokens 87 us, 5804 GB/s, 89 % of a copy (pairs by halves 91 us); 2001 tokens 16.3 us; 16 tokens of 12 heads on 2
// 2.3 us, a launch, from four partial sums 2.8 us.
#include "mono_common.cuh"

extern void mono_set_error(const char* fmt, ...);

namespace qkv_append {
using namespace mono;

constexpr int kDim = 128;
constexpr int kThreads = 256;
// CTAs of an SM: with four, halves that turn with one another (their partners come by shuffles) do not fit 64 registers
// (16384 tokens 100 us, with three 91), interleaved pairs do (87 us either way).  Partial sums have at most 16 rows.
constexpr int ctas_per_sm(bool interleaved, bool f32) { return f32 ? 2 : interleaved ? 4 : 3; }

typedef unsigned long long f32x2;  // two f32 that one instruction works on
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 halves(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 swapped(f32x2 v) {
    const float2 h = halves(v);
    return pair(h.y, h.x);
}
__device__ __forceinline__ f32x2 unpack2(uint32_t w) { return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ void unpack8(const uint4 w, f32x2 v[4]) {
    v[0] = unpack2(w.x); v[1] = unpack2(w.y); v[2] = unpack2(w.z); v[3] = unpack2(w.w);
}
__device__ __forceinline__ uint32_t pack2(f32x2 v) {
    const float2 h = halves(v);
    const __nv_bfloat162 b = __floats2bfloat162_rn(h.x, h.y);
    return *reinterpret_cast<const uint32_t*>(&b);
}
// two table entries from entry `at` on (at even)
__device__ __forceinline__ f32x2 load2(const void* table, int is_f32, size_t at) {
    if (is_f32) {
        const float2 f = __ldg(reinterpret_cast<const float2*>(reinterpret_cast<const float*>(table) + at));
        return pair(f.x, f.y);
    }
    return unpack2(__ldg(reinterpret_cast<const uint32_t*>(reinterpret_cast<const __nv_bfloat16*>(table) + at)));
}

// What a lane multiplies its eight dims of a q or k head by: out = f (x A + other B), other being the dims' partners.
// Norm and rotation are linear in the head up to the factor f = 1 / rms, so A = (1 + g) cos and B = -+(1 + g of the
// partner) sin serve all heads of a token and kind.
struct Coef {
    f32x2 a[4], b[4];
};
template <bool INTERLEAVED>
__device__ __forceinline__ void make_coef(const mono_qkv_append_args& args, const void* gain, size_t row, int sub, int psub, bool turned, bool low, Coef& c) {
    const f32x2 one = pair(1.f, 1.f);
    f32x2 g[4] = {one, one, one, one}, o[4] = {one, one, one, one};
    if (gain) {
        unpack8(__ldg(reinterpret_cast<const uint4*>(gain) + sub), g);
        unpack8(__ldg(reinterpret_cast<const uint4*>(gain) + psub), o);
#pragma unroll
        for (int j = 0; j < 4; ++j) { g[j] = fma2(one, one, g[j]); o[j] = fma2(one, one, o[j]); }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        c.a[j] = g[j];
        c.b[j] = pair(0.f, 0.f);
        if (!turned) continue;
        if (INTERLEAVED) {  // two dims share an angle: (x0, x1) -> (x0 c - x1 s, x1 c + x0 s)
            const size_t at = row + sub * 4 + (j & 2);
            const float2 cs = halves(load2(args.cos, args.table_f32, at)), sn = halves(load2(args.sin, args.table_f32, at));
            const float cj = j & 1 ? cs.y : cs.x, sj = j & 1 ? sn.y : sn.x;
            c.a[j] = mul2(g[j], pair(cj, cj));
            c.b[j] = mul2(swapped(g[j]), pair(-sj, sj));
        } else {  // this lane holds the first or the second dims of eight pairs
            const size_t at = row + (low ? sub : psub) * 8 + 2 * j;
            const float2 sn = halves(load2(args.sin, args.table_f32, at));
            c.a[j] = mul2(g[j], load2(args.cos, args.table_f32, at));
            c.b[j] = mul2(o[j], low ? pair(-sn.x, -sn.y) : pair(sn.x, sn.y));
        }
    }
}

// Per warp: where it reads and writes.
struct Lane {
    int sub, half, psub;  // piece of the head, head of the pair, piece that holds the partners
    bool turned, low;     // its dims are rotated; they are the first of their pairs
    size_t row;           // of the tables
};

// The pairs of heads p0 .. p1 - 1 of one kind (0 q, 1 k, 2 v); kBatch of them are in flight.
template <int KIND, bool INTERLEAVED, bool F32SRC>
__device__ __forceinline__ void do_heads(const mono_qkv_append_args& a, const Lane& n, int token, int p0, int p1, uint8_t* to) {
    if (p0 >= p1) return;
    constexpr int kBatch = F32SRC ? 1 : 4;
    const int count = KIND == 0 ? a.q_heads : a.kv_heads, first = KIND == 0 ? 0 : KIND == 1 ? a.q_heads : a.q_heads + a.kv_heads;
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.src_bf16) + (size_t)token * a.src_ld) + first * (kDim / 8) + n.sub;
    const void* gain = KIND == 0 ? a.g_q : a.g_k;
    Coef cf;
    const float scale = KIND == 0 ? 1.f : 1.f / (KIND == 1 ? a.k_scale : a.v_scale);
    uint4 raw[kBatch];
    if (!F32SRC) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) raw[j] = __ldg(src + min(2 * (p0 + j) + n.half, count - 1) * (kDim / 8));
    }
    if (KIND != 2) make_coef<INTERLEAVED>(a, gain, n.row, n.sub, n.psub, n.turned, n.low, cf);
    for (int p = p0; p < p1; p += kBatch) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (p + j >= p1) break;
            const int h = 2 * (p + j) + n.half;
            f32x2 x[4], other[4];
            if (F32SRC) {
                const float* f = a.src_f32 + (size_t)token * a.src_ld + (size_t)(first + min(h, count - 1)) * kDim + n.sub * 8;
                const float4 lo = sum_partials4<4>(f, (size_t)a.sum_stride, a.nsum), hi = sum_partials4<4>(f + 4, (size_t)a.sum_stride, a.nsum);
                x[0] = pair(lo.x, lo.y); x[1] = pair(lo.z, lo.w);
                x[2] = pair(hi.x, hi.y); x[3] = pair(hi.z, hi.w);
                if (KIND != 2) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) other[i] = INTERLEAVED ? swapped(x[i]) : __shfl_sync(0xffffffffu, x[i], n.half * 16 + n.psub);
                }
            } else {
                const uint4 w = raw[j];
                unpack8(w, x);
                if (KIND != 2 && INTERLEAVED) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) other[i] = swapped(x[i]);
                } else if (KIND != 2) {
                    const int from = n.half * 16 + n.psub;
                    unpack8(make_uint4(__shfl_sync(0xffffffffu, w.x, from), __shfl_sync(0xffffffffu, w.y, from), __shfl_sync(0xffffffffu, w.z, from),
                                       __shfl_sync(0xffffffffu, w.w, from)), other);
                }
                raw[j] = __ldg(src + min(h + 2 * kBatch, count - 1) * (kDim / 8));
            }
            float f = scale;
            if (KIND != 2) {
                if (gain) {
                    f32x2 sq = mul2(x[0], x[0]);
#pragma unroll
                    for (int i = 1; i < 4; ++i) sq = fma2(x[i], x[i], sq);
                    const float2 sh = halves(sq);
                    float ssq = sh.x + sh.y;
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1) ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
                    f *= rsqrtf(ssq * (1.f / kDim) + a.eps);
                }
                // dims that are not turned keep no trace of others, infinite or not
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = n.turned ? fma2(other[i], cf.b[i], mul2(x[i], cf.a[i])) : mul2(x[i], cf.a[i]);
            }
            const f32x2 ff = pair(f, f);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = mul2(x[i], ff);
            if (h < count && to) {
                if (KIND == 0) {
                    *reinterpret_cast<uint4*>(to + h * kDim * 2) = make_uint4(pack2(x[0]), pack2(x[1]), pack2(x[2]), pack2(x[3]));
                } else {
                    uint32_t b[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[i] = __nv_cvt_float2_to_fp8x2(halves(x[i]), __NV_SATFINITE, __NV_E4M3);
                    *reinterpret_cast<uint2*>(to + h * kDim) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
                }
            }
        }
    }
}

// A warp takes `pairs` pairs of heads of one token (q pairs, then k, then v); lanes 0..15 hold the even head of a pair,
// 16..31 the odd one.
template <bool INTERLEAVED, bool F32SRC>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(INTERLEAVED, F32SRC)) qkv_append_kernel(const __grid_constant__ mono_qkv_append_args a, int chunks, int pairs) {
    pdl_prologue();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned work = blockIdx.x * (kThreads / 32) + warp;
    const int token = (int)(work / (unsigned)chunks);
    if (token >= a.tokens) return;  // whole warps leave together
    const int p0 = (int)(work - (unsigned)token * chunks) * pairs, p1 = p0 + pairs;
    const int64_t slot = a.slots ? a.slots[token] : -1;
    const bool insert = slot >= 0 && slot < a.n_pages * kPage;
    Lane n;
    n.sub = lane & 15;
    n.half = lane >> 4;
    const int lanes_half = a.rot_dim >> 4;  // lanes that hold the first half of the rotated dims
    n.turned = n.sub < 2 * lanes_half;
    n.low = n.sub < lanes_half;
    n.psub = INTERLEAVED || !n.turned ? n.sub : n.low ? n.sub + lanes_half : n.sub - lanes_half;
    int64_t pos = a.positions[token];
    pos = pos < 0 ? 0 : pos >= a.table_rows ? a.table_rows - 1 : pos;
    n.row = (size_t)pos * (a.rot_dim >> 1);
    const int pq = (a.q_heads + 1) >> 1, pk = (a.kv_heads + 1) >> 1;
    uint8_t* q_to = reinterpret_cast<uint8_t*>(a.q_out) + (size_t)token * a.q_heads * kDim * 2 + n.sub * 16;
    const size_t kv_at = (size_t)(insert ? slot : 0) * a.kv_heads * kDim + n.sub * 8;
    do_heads<0, INTERLEAVED, F32SRC>(a, n, token, p0, min(p1, pq), q_to);
    if (!insert) return;
    do_heads<1, INTERLEAVED, F32SRC>(a, n, token, max(p0 - pq, 0), min(p1 - pq, pk), a.k_cache + kv_at);
    do_heads<2, INTERLEAVED, F32SRC>(a, n, token, max(p0 - pq - pk, 0), min(p1 - pq - pk, pk), a.v_cache + kv_at);
}

template <bool INTERLEAVED>
static cudaError_t launch(const mono_qkv_append_args* a, cudaStream_t st) {
    const int pairs = (a->q_heads + 1) / 2 + 2 * ((a->kv_heads + 1) / 2);
    // How many warps share a token: what takes least, reckoned as rounds of the warps that the GPU holds, a round as long as a
    // warp's pairs of heads and kStart more (angles and latency).  With 32 warps an SM and 48 heads on 8: 2001 tokens, two
    // warps, one round, 17 us (five warps, which fill it 2.1 times, 20.6); 3000: three warps 23 us, one 28; 6000: two 41, one 45.
    constexpr int kStart = 6;
    const long long held = (mono_sm_count() > 0 ? mono_sm_count() : 148) * ctas_per_sm(INTERLEAVED, a->src_f32 != nullptr) * (kThreads / 32);
    int chunks = 1;
    long long least = -1;
    for (int c = 1; c <= pairs && (c == 1 || a->tokens * (long long)c <= 8 * held); ++c) {
        const long long cost = (a->tokens * (long long)c + held - 1) / held * ((pairs + c - 1) / c + kStart);
        if (least < 0 || cost < least) { least = cost; chunks = c; }
    }
    const int per = (pairs + chunks - 1) / chunks;
    chunks = (pairs + per - 1) / per;
    const long long warps = (long long)a->tokens * chunks;
    const unsigned grid = (unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32));
    return a->src_f32 ? launch_k(qkv_append_kernel<INTERLEAVED, true>, grid, kThreads, 0, st, *a, chunks, per)
                      : launch_k(qkv_append_kernel<INTERLEAVED, false>, grid, kThreads, 0, st, *a, chunks, per);
}

}  // namespace qkv_append

extern "C" int mono_qkv_append_launch(const mono_qkv_append_args* a, void* stream) {
    const char* who = "mono_qkv_append_launch";
    if (!a || a->tokens < 1 || a->tokens > (1 << 24) || a->q_heads < 1 || a->kv_heads < 1 || a->q_heads > 256 || a->kv_heads > 256) {
        mono_set_error("%s: 1..2^24 tokens, 1..256 q heads and 1..256 kv heads required", who);
        return MONO_E_ARG;
    }
    if (a->rot_dim < 16 || a->rot_dim > 128 || (a->rot_dim & 15)) {
        mono_set_error("%s: rot_dim %d, needs a multiple of 16 in 16..128", who, a->rot_dim);
        return MONO_E_ARG;
    }
    if ((a->src_bf16 == nullptr) == (a->src_f32 == nullptr) || (a->src_f32 && (a->nsum < 1 || a->tokens > MONO_MAX_ROWS || (a->sum_stride & 3)))) {
        mono_set_error("%s: bf16 rows, or f32 partial sums of at most %d rows, required", who, MONO_MAX_ROWS);
        return MONO_E_ARG;
    }
    const long width = (long)(a->q_heads + 2 * a->kv_heads) * 128;
    if (a->src_ld < width || (a->src_ld & 7) || (reinterpret_cast<uintptr_t>(a->src_bf16) & 15) || (reinterpret_cast<uintptr_t>(a->src_f32) & 15)) {
        mono_set_error("%s: rows of %ld values needed at a 16-byte aligned address, their distance a multiple of 8 values (got %ld)", who, width, a->src_ld);
        return MONO_E_ARG;
    }
    const uintptr_t all = reinterpret_cast<uintptr_t>(a->g_q) | reinterpret_cast<uintptr_t>(a->g_k) | reinterpret_cast<uintptr_t>(a->cos) |
                          reinterpret_cast<uintptr_t>(a->sin) | reinterpret_cast<uintptr_t>(a->q_out) | reinterpret_cast<uintptr_t>(a->k_cache) |
                          reinterpret_cast<uintptr_t>(a->v_cache);
    if (!a->cos || !a->sin || a->table_rows < 1 || !a->positions || !a->q_out || !a->k_cache || !a->v_cache || a->n_pages < 1 || !mono::scale_ok(a->k_scale) || !mono::scale_ok(a->v_scale) || !(a->eps >= 0.f) || (all & 15)) {
        mono_set_error("%s: rope tables, positions, q output and caches with scales of 2^-100 .. 2^100 required, 16-byte aligned", who);
        return MONO_E_ARG;
    }
    const cudaError_t e = a->interleaved ? qkv_append::launch<true>(a, (cudaStream_t)stream) : qkv_append::launch<false>(a, (cudaStream_t)stream);
    if (e != cudaSuccess) mono_set_error("%s: %s", who, cudaGetErrorString(e));
    return (int)e;
}
