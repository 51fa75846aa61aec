// Rows of the fused q | k | v projection -> normed and rotated queries, and keys and values in the paged E4M3 cache.
//
// Per q and k head:  y = x / sqrt(mean(x^2) + eps) * (1 + g)          (no norm where g is absent)
//                    (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin) on the first R dims, pairs (i, i + R/2) or (2i, 2i+1)
// q is stored as bf16, k as E4M3(y / k_scale), v as E4M3(x / v_scale), saturating.  Everything between the load and the
// store is f32 with one rounding at the store; the step kernel of gqa.cu, which also makes the index keys, rounds to
// bf16 after the norm and after the rotation instead.
//
// Bound: memory.  A token's row is read once and written once (bf16 q, one byte per K and V value).  Sixteen lanes hold
// a head, eight dims (16 bytes) each, so a warp takes two heads at a time and a norm is four shuffles.
#include "mono_common.cuh"

extern void mono_set_error(const char* fmt, ...);

namespace qkv_append {
using namespace mono;

constexpr int kDim = 128;
constexpr int kThreads = 256;

__device__ __forceinline__ void unpack8(const uint4 w, float v[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(u[j] << 16);
        v[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint4 pack8(const float v[8]) {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}
// n table entries from entry i of a row (n = 4 or 8, i a multiple of n)
template <int N>
__device__ __forceinline__ void load_table(const void* table, int is_f32, size_t at, float v[N]) {
    if (is_f32) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(table) + at);
#pragma unroll
        for (int j = 0; j < N / 4; ++j) {
            const float4 f = __ldg(p + j);
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        }
    } else {
        const uint2* p = reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(table) + at);
#pragma unroll
        for (int j = 0; j < N / 4; ++j) {
            const uint2 w = __ldg(p + j);
            v[4 * j] = __uint_as_float(w.x << 16); v[4 * j + 1] = __uint_as_float(w.x & 0xFFFF0000u);
            v[4 * j + 2] = __uint_as_float(w.y << 16); v[4 * j + 3] = __uint_as_float(w.y & 0xFFFF0000u);
        }
    }
}

// A warp takes PAIRS pairs of heads of one token; lanes 0..15 hold the even head of a pair, 16..31 the odd one.
template <int PAIRS, bool F32SRC>
__global__ void __launch_bounds__(kThreads) qkv_append_kernel(const mono_qkv_append_args a, int chunks) {
    pdl_prologue();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 15, half = lane >> 4;
    const long long work = (long long)blockIdx.x * (kThreads / 32) + warp;
    const long long token = work / chunks;
    if (token >= a.tokens) return;  // whole warps leave together
    const int chunk = (int)(work - token * chunks);
    const int heads = a.q_heads + 2 * a.kv_heads;
    const int head0 = chunk * PAIRS * 2 + half;
    float x[PAIRS][8];
    if (F32SRC) {
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
            const int h = min(head0 + 2 * p, heads - 1);
            const float* src = a.src_f32 + (size_t)token * a.src_ld + (size_t)h * kDim + sub * 8;
            const float4 lo = sum_partials4<4>(src, (size_t)a.sum_stride, a.nsum);
            const float4 hi = sum_partials4<4>(src + 4, (size_t)a.sum_stride, a.nsum);
            x[p][0] = lo.x; x[p][1] = lo.y; x[p][2] = lo.z; x[p][3] = lo.w;
            x[p][4] = hi.x; x[p][5] = hi.y; x[p][6] = hi.z; x[p][7] = hi.w;
        }
    } else {
        const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(a.src_bf16) + (size_t)token * a.src_ld + sub * 8;
        uint4 raw[PAIRS];  // every load is issued before the first is used
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) raw[p] = __ldg(reinterpret_cast<const uint4*>(src + (size_t)min(head0 + 2 * p, heads - 1) * kDim));
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) unpack8(raw[p], x[p]);
    }
    // the token's angles: this lane's eight dims are one side of eight pairs (half layout) or four whole pairs
    const int lanes_half = a.rot_dim >> 4;  // lanes that hold the first half of the rotated dims
    const bool turned = sub < 2 * lanes_half;
    int partner = lane;
    float c[8], s[8];
    {
        int64_t pos = a.positions[token];
        pos = pos < 0 ? 0 : pos >= a.table_rows ? a.table_rows - 1 : pos;
        const size_t row = (size_t)pos * (a.rot_dim >> 1);
        if (turned && !a.interleaved) {
            partner = sub < lanes_half ? lane + lanes_half : lane - lanes_half;
            const int i = (sub < lanes_half ? sub : sub - lanes_half) * 8;
            load_table<8>(a.cos, a.table_f32, row + i, c);
            load_table<8>(a.sin, a.table_f32, row + i, s);
        } else if (turned) {
            load_table<4>(a.cos, a.table_f32, row + sub * 4, c);
            load_table<4>(a.sin, a.table_f32, row + sub * 4, s);
        }
    }
    const int64_t slot = a.slots ? a.slots[token] : -1;
    const bool insert = slot >= 0 && slot < a.n_pages * kPage;
#pragma unroll
    for (int p = 0; p < PAIRS; ++p) {
        const int h = head0 + 2 * p;
        const int kind = h < a.q_heads ? 0 : h < a.q_heads + a.kv_heads ? 1 : 2;
        const void* gp = kind == 0 ? a.g_q : kind == 1 ? a.g_k : nullptr;
        float ssq = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ssq += x[p][j] * x[p][j];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
        if (gp) {
            const float rstd = rsqrtf(ssq * (1.f / kDim) + a.eps);
            float g[8];
            unpack8(__ldg(reinterpret_cast<const uint4*>(gp) + sub), g);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[p][j] = x[p][j] * rstd * (1.f + g[j]);
        }
        if (!a.interleaved) {
            const float sign = sub < lanes_half ? -1.f : 1.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float other = __shfl_sync(0xffffffffu, x[p][j], partner);
                if (turned && kind != 2) x[p][j] = x[p][j] * c[j] + sign * other * s[j];
            }
        } else if (turned && kind != 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float lo = x[p][2 * j], hi = x[p][2 * j + 1];
                x[p][2 * j] = lo * c[j] - hi * s[j];
                x[p][2 * j + 1] = hi * c[j] + lo * s[j];
            }
        }
        if (h >= heads) continue;
        if (kind == 0) {
            reinterpret_cast<uint4*>(a.q_out)[((size_t)token * a.q_heads + h) * (kDim / 8) + sub] = pack8(x[p]);
        } else if (insert) {
            const float sc = kind == 1 ? a.k_scale : a.v_scale;
            uint8_t* cache = kind == 1 ? a.k_cache : a.v_cache;
            const int kh = h - a.q_heads - (kind == 1 ? 0 : a.kv_heads);
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                w[j >> 2] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[p][j], sc), __fdiv_rn(x[p][j + 1], sc)), __NV_SATFINITE, __NV_E4M3)
                             << (8 * (j & 3));
            *reinterpret_cast<uint2*>(cache + ((size_t)slot * a.kv_heads + kh) * kDim + sub * 8) = make_uint2(w[0], w[1]);
        }
    }
}

template <int PAIRS>
static cudaError_t launch(const mono_qkv_append_args* a, cudaStream_t st) {
    const int pairs = (a->q_heads + 2 * a->kv_heads + 1) / 2;
    const int chunks = (pairs + PAIRS - 1) / PAIRS;
    const long long warps = (long long)a->tokens * chunks;
    const unsigned grid = (unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32));
    return a->src_f32 ? launch_k(qkv_append_kernel<PAIRS, true>, grid, kThreads, 0, st, *a, chunks)
                      : launch_k(qkv_append_kernel<PAIRS, false>, grid, kThreads, 0, st, *a, chunks);
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
    if (!a->cos || !a->sin || a->table_rows < 1 || !a->positions || !a->q_out || !a->k_cache || !a->v_cache || a->n_pages < 1 || !(a->k_scale > 0.f) ||
        !(a->v_scale > 0.f) || !(a->eps >= 0.f) || (all & 15)) {
        mono_set_error("%s: rope tables, positions, q output and caches with positive scales required, 16-byte aligned", who);
        return MONO_E_ARG;
    }
    // A warp that takes four pairs has four row loads in flight and reads its angles once for eight heads; a small
    // step is spread over more warps instead.
    const long long pairs = (long long)a->tokens * ((a->q_heads + 2 * a->kv_heads + 1) / 2);
    const int sms = mono_sm_count();
    const cudaError_t e = pairs >= (long long)(sms > 0 ? sms : 148) * 64 ? qkv_append::launch<4>(a, (cudaStream_t)stream)
                                                                         : qkv_append::launch<1>(a, (cudaStream_t)stream);
    if (e != cudaSuccess) mono_set_error("%s: %s", who, cudaGetErrorString(e));
    return (int)e;
}
