// Attention of a batch whose sequences share long prefixes, over the paged E4M3 K and V caches: narrow split and merge.
//
//   out[t][h] = softmax over the keys that token t sees (its group's prefix, its sequence's own keys up to itself) of
//               (q[t][h] . k) k_scale sm_scale,  times v v_scale
//
// A prefix is read once for all tokens of its group: the rows of a tile come from every sequence of the group.
// prefix_attn.cuh says how the work is cut.  This file holds the kernel for few rows and the merge; prefix_attn_tc.cu
// the kernel for many.
#include "prefix_attn.cuh"

extern void mono_set_error(const char* fmt, ...);

namespace prefix_attn {

constexpr int kConsumers = 4;                        // warps that compute; one more fetches
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kStages = 4;
constexpr int kTileBytes = kPage * kDim;             // one page of one kv head: 64 keys x 128 bytes
constexpr int kPitch = kDim + 4;                     // floats of a combine row
constexpr float kPBias = 14.f;                       // P is formed as 2^14 p, so that f16 keeps small weights

// D(16x8,f32) += A(16x16,f16,row) * B(16x8,f16,col)
__device__ __forceinline__ void mma_f16(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t lo16) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(lo16 & 0xFFFFu), __NV_E4M3);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// a maximum that keeps NaN: a row with a NaN score is a row of NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// The queries of one tile in the layout of the A fragments, and their scales.  The contraction's order is free as long
// as both operands share it, so thread (g, t) of a fragment takes dims 32 t .. 32 t + 31 of its rows: a key's 32 bytes
// are then two 16-byte shared loads.  A row is scaled by a power of two so that its largest value lies in
// [2^13, 2^14): f16 then holds every bf16 value down to 2^-28 of that exactly.
__device__ __forceinline__ void load_q(const mono_prefix_attn_args& a, const Entry& n, int head, int row0, int G, uint32_t q[8][4], float qscale[2],
                                       int lim[2]) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    uint4 raw[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = row0 + g + 8 * i;
        const bool live = row < n.ntok * G;
        const int r = live ? row : 0;
        const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)(n.tok0 + r / G) * a.q_ld + (size_t)(head * G + r % G) * kDim + t * 32;
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[i][j] = live ? __ldg(reinterpret_cast<const uint4*>(src) + j) : make_uint4(0, 0, 0, 0);
        lim[i] = live ? row_limit(n, row, G) : 0;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(raw[i]);
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[j] << 16)), fabsf(__uint_as_float(w[j] & 0xFFFF0000u))));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // exponent field of the largest value, kept where 2^(13 - e) and its inverse are normal numbers
        const int e = clamp_int((int)(__float_as_uint(amax) >> 23), 30, 254);
        const float up = __uint_as_float((uint32_t)(267 - e) << 23);  // 2^(13 - (e - 127))
        qscale[i] = __uint_as_float((uint32_t)(e - 13) << 23) * (a.sm_scale * a.k_scale * 1.4426950408889634f);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            q[s][i] = pack_f16(__uint_as_float(w[2 * s] << 16) * up, __uint_as_float(w[2 * s] & 0xFFFF0000u) * up);
            q[s][2 + i] = pack_f16(__uint_as_float(w[2 * s + 1] << 16) * up, __uint_as_float(w[2 * s + 1] & 0xFFFF0000u) * up);
        }
    }
}

// Up to 16 rows per tile.  Four warps take 16 of a page's 64 keys each, for all rows of the tile, with a running
// maximum and sum of their own; the fifth warp keeps a ring of pages in flight by TMA (128-byte swizzle, which makes
// the 16-byte shared loads below free of bank conflicts).  Bound: HBM; K and V stay bytes until a warp has them in
// registers, where they become f16 exactly.
__global__ void __launch_bounds__(kThreads, 2) prefix_narrow_kernel(const __grid_constant__ Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* comb = reinterpret_cast<float*>(ring + kStages * 2 * kTileBytes);  // [4 warps][16 rows][kPitch]
    const mono_prefix_attn_args& a = p.a;
    const int E = a.groups + a.seqs;
    uint32_t* off = reinterpret_cast<uint32_t*>(comb + kConsumers * 16 * kPitch);
    uint32_t* item = off + E + 1;
    __shared__ uint64_t full[kStages], empty[kStages];
    __shared__ int page_ok[kStages];
    __shared__ uint32_t red[64];
    __shared__ float s_m[kConsumers][16], s_l[kConsumers][16];
    __shared__ int abort_flag;
    volatile int* abortp = &abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kConsumers);
        }
        mbar_fence_init();
        prefetch_tmap(&p.kmap);
        prefetch_tmap(&p.vmap);
    }
    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0 && guard_failed(a.guard)) abort_flag = 1;
    make_plan<false, kThreads>(a, off, item, red);
    if (blockIdx.x == 0) {  // the merge reads it
        for (int e = tid; e <= E; e += kThreads) {
            p.s.off[0][e] = off[e];
            p.s.item[0][e] = item[e];
        }
    }
    const uint32_t U = off[E], n = min(gridDim.x, U);
    const int G = a.q_heads / a.kv_heads;
    const uint64_t wait_ns = a.wait_ns ? a.wait_ns : kWaitLimitNs;
    if (blockIdx.x < n) {
        const uint32_t u0 = cut(U, blockIdx.x, n), u1 = cut(U, blockIdx.x + 1, n);
        if (warp == kConsumers) {
            // ---- fetch: 32 units' pages at a time are looked up by the lanes, then requested in order
            int it = 0;
            for (uint32_t base = u0; base < u1 && !*abortp; base += 32) {
                const uint32_t u = min(base + lane, u1 - 1);
                const int e = find_entry(off, E, u);
                const Entry en = entry_of(a, e);
                int tiles, units;
                entry_work<false>(a, en, &tiles, &units);
                const uint32_t local = u - off[e];
                const int head = (int)(local / units) / tiles;
                const int page = en.table[local % units];
                const bool ok = page >= 0 && page < a.n_pages;
                const int cnt = (int)min(32u, u1 - base);
                for (int j = 0; j < cnt; ++j, ++it) {
                    const int pj = __shfl_sync(0xffffffffu, page, j), hj = __shfl_sync(0xffffffffu, head, j), okj = __shfl_sync(0xffffffffu, (int)ok, j);
                    if (lane == 0) {
                        const int st = it % kStages;
                        if (*abortp || (it >= kStages && !mbar_wait(&empty[st], ((it / kStages) - 1) & 1, abortp, wait_ns))) {
                            // given up: the consumers' waits see the flag
                        } else {
                            page_ok[st] = okj;
                            if (okj) {
                                uint8_t* dst = ring + st * 2 * kTileBytes;
                                mbar_expect_tx(&full[st], 2 * kTileBytes);
                                tma_load_3d(dst, &p.kmap, hj * kDim, pj * kPage, 0, &full[st]);
                                tma_load_3d(dst + kTileBytes, &p.vmap, hj * kDim, pj * kPage, 0, &full[st]);
                            } else {
                                mbar_arrive(&full[st]);
                            }
                        }
                    }
                }
                __syncwarp();
            }
        } else {
            const int g = lane >> 2, t = lane & 3;
            int it = 0, e = find_entry(off, E, u0);
            for (uint32_t u = u0; u < u1;) {
                while (off[e + 1] <= u) ++e;
                const Entry en = entry_of(a, e);
                int tiles, units;
                entry_work<false>(a, en, &tiles, &units);
                const uint32_t local = u - off[e], it_in = local / units;
                const int head = (int)it_in / tiles, tile = (int)it_in % tiles;
                const int p0 = (int)(local % units), cnt = (int)min((uint32_t)(units - p0), u1 - u);
                uint32_t q[8][4];
                float qs[2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
                int lim[2];
                load_q(a, en, head, tile * 16, G, q, qs, lim);
                float o[16][4];
#pragma unroll
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
                for (int i = 0; i < cnt; ++i, ++it) {
                    const int st = it % kStages;
                    if (!mbar_wait(&full[st], (it / kStages) & 1, abortp, wait_ns)) break;
                    const uint32_t kb = smem_u32(ring + st * 2 * kTileBytes), vb = kb + kTileBytes;
                    const int key0 = (p0 + i) * kPage + warp * 16;  // this warp's first key
                    if (page_ok[st] && key0 < en.len) {
                        float s[2][4];
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) {
                            const uint32_t rowa = kb + (warp * 16 + nt * 8 + g) * 128;
                            const uint4 k0 = lds128(rowa + (((2 * t) ^ g) << 4)), k1 = lds128(rowa + (((2 * t + 1) ^ g) << 4));
                            const uint32_t w[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) s[nt][j] = 0.f;
#pragma unroll
                            for (int j = 0; j < 8; ++j) mma_f16(s[nt], q[j], e4m3x2_to_f16x2(w[j]), e4m3x2_to_f16x2(w[j] >> 16));
                        }
                        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int r = j >> 1, key = key0 + nt * 8 + 2 * t + (j & 1);
                                s[nt][j] = key < lim[r] ? s[nt][j] * qs[r] : -INFINITY;
                                mx[r] = max_nan(mx[r], s[nt][j]);
                            }
                        float mn[2], alpha[2];
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            mx[r] = max_nan(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                            mx[r] = max_nan(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                            mn[r] = max_nan(m[r], mx[r]);
                            // a row that has seen no key yet keeps max = -inf, and weights of 0
                            alpha[r] = mn[r] == -INFINITY ? 1.f : exp2f(m[r] - mn[r]);
                            m[r] = mn[r];
                            l[r] *= alpha[r];
                        }
                        uint32_t pa[4];
                        float pv[2][4];
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int r = j >> 1;
                                pv[nt][j] = s[nt][j] == -INFINITY ? 0.f : exp2f(s[nt][j] - mn[r] + kPBias);
                                l[r] += pv[nt][j];
                            }
                        pa[0] = pack_f16(pv[0][0], pv[0][1]);
                        pa[1] = pack_f16(pv[0][2], pv[0][3]);
                        pa[2] = pack_f16(pv[1][0], pv[1][1]);
                        pa[3] = pack_f16(pv[1][2], pv[1][3]);
                        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                o[j][0] *= alpha[0]; o[j][1] *= alpha[0];
                                o[j][2] *= alpha[1]; o[j][3] *= alpha[1];
                            }
                        }
                        // V: thread (g, t) takes dims 16 g .. 16 g + 15 of keys 2t, 2t + 1, 2t + 8, 2t + 9; output
                        // column g of product j is dim 16 g + j.  Keys behind the entry's last hold anything, NaN among
                        // it, and 0 x NaN is NaN, so their bytes become zeros.
                        uint32_t vw[4][4];
#pragma unroll
                        for (int i4 = 0; i4 < 4; ++i4) {
                            const int kr = 2 * t + (i4 & 1) + (i4 >> 1) * 8;
                            const uint4 v = lds128(vb + (warp * 16 + kr) * 128 + ((g ^ (kr & 7)) << 4));
                            const bool live = key0 + kr < en.len;
                            vw[i4][0] = live ? v.x : 0u; vw[i4][1] = live ? v.y : 0u; vw[i4][2] = live ? v.z : 0u; vw[i4][3] = live ? v.w : 0u;
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t a01 = __byte_perm(vw[0][j], vw[1][j], 0x5140), a23 = __byte_perm(vw[0][j], vw[1][j], 0x7362);
                            const uint32_t b01 = __byte_perm(vw[2][j], vw[3][j], 0x5140), b23 = __byte_perm(vw[2][j], vw[3][j], 0x7362);
                            mma_f16(o[4 * j], pa, e4m3x2_to_f16x2(a01), e4m3x2_to_f16x2(b01));
                            mma_f16(o[4 * j + 1], pa, e4m3x2_to_f16x2(a01 >> 16), e4m3x2_to_f16x2(b01 >> 16));
                            mma_f16(o[4 * j + 2], pa, e4m3x2_to_f16x2(a23), e4m3x2_to_f16x2(b23));
                            mma_f16(o[4 * j + 3], pa, e4m3x2_to_f16x2(a23 >> 16), e4m3x2_to_f16x2(b23 >> 16));
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&empty[st]);
                }
                // ---- the segment's rows: the four warps' parts, brought to one maximum
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
                    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
                    if (t == 0) {
                        s_m[warp][g + 8 * r] = m[r];
                        s_l[warp][g + 8 * r] = l[r];
                    }
                }
                consumer_sync();
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = g + 8 * r;
                    const float M = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
                    const float f = m[r] == -INFINITY ? 0.f : exp2f(m[r] - M);
                    float* dst = comb + (warp * 16 + row) * kPitch + t * 32;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 16; j += 4)
                            *reinterpret_cast<float4*>(dst + h * 16 + j) = make_float4(o[j][2 * r + h] * f, o[j + 1][2 * r + h] * f, o[j + 2][2 * r + h] * f, o[j + 3][2 * r + h] * f);
                }
                consumer_sync();
                {
                    float* seg = p.s.seg[0] + (size_t)(blockIdx.x + item[e] + it_in) * Shape<false>::kSegFloats;
                    const int rows = min(16, en.ntok * G - tile * 16);
                    if (tid < rows) {
                        const float M = fmaxf(fmaxf(s_m[0][tid], s_m[1][tid]), fmaxf(s_m[2][tid], s_m[3][tid]));
                        float sum = 0.f;
#pragma unroll
                        for (int w = 0; w < kConsumers; ++w) sum += s_m[w][tid] == -INFINITY ? 0.f : s_l[w][tid] * exp2f(s_m[w][tid] - M);
                        seg[tid] = M - kPBias;
                        seg[16 + tid] = sum;
                    }
                    for (int r = 0; r < rows; ++r) {
                        float sum = 0.f;
#pragma unroll
                        for (int w = 0; w < kConsumers; ++w) sum += comb[(w * 16 + r) * kPitch + tid];
                        seg[32 + r * kDim + tid] = sum;
                    }
                }
                consumer_sync();
                u += cnt;
            }
        }
    }
    __syncthreads();
    if (*abortp) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the CTA's memory goes
        if (tid == 0 && !guard_failed(a.guard)) guard_fail(a.guard, MONO_ERR_DEADLINE, kSiteWait);
    }
}

// ------------------------------------------------------------------ merge
// One CTA of four warps per (token, 4 / SPLIT heads): SPLIT warps share a row's segments.  A lane holds four dims.
template <int SPLIT>
__global__ void __launch_bounds__(128) prefix_merge_kernel(const mono_prefix_attn_args a, const Scratch s, int narrow_ctas, int wide_ctas) {
    pdl_prologue();
    __shared__ int s_seq, s_grp;
    __shared__ float4 s_num[4][32];
    __shared__ float s_den[4];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int token = blockIdx.x, head = blockIdx.y * (4 / SPLIT) + warp / SPLIT, part = warp % SPLIT;
    if (tid == 0) { s_seq = INT32_MAX; s_grp = INT32_MAX; }
    __syncthreads();
    for (int e = tid; e < a.groups + a.seqs; e += 128) {
        const Entry n = entry_of(a, e);
        if (token >= n.tok0 && token < n.tok0 + n.ntok) atomicMin(e < a.groups ? &s_grp : &s_seq, e);
    }
    __syncthreads();
    if (s_seq == INT32_MAX) return;  // behind the last sequence: the row stays as it was
    const bool on = head < a.q_heads;
    const int G = a.q_heads / a.kv_heads, E = a.groups + a.seqs;
    // the segments of the row's two items: `count` segments `stride` floats apart
    const float* base[2] = {nullptr, nullptr};
    int count[2] = {0, 0}, stride[2] = {0, 0}, tile_rows[2] = {0, 0}, row_in[2] = {0, 0}, twice[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int e = k ? s_seq : s_grp;
        if (e == INT32_MAX || !on) continue;
        const Entry n = entry_of(a, e);
        const int w = n.ntok * G >= kWideRows;
        const int tr = w ? Shape<true>::kTile : Shape<false>::kTile;
        int tiles, units;
        if (w) entry_work<true>(a, n, &tiles, &units); else entry_work<false>(a, n, &tiles, &units);
        if (units == 0) continue;
        const uint32_t* off = s.off[w];
        const uint32_t U = off[E], ctas = min((uint32_t)(w ? wide_ctas : narrow_ctas), U);
        if (U == 0) continue;  // refused tables
        const int row = (token - n.tok0) * G + head % G, it_in = (head / G) * tiles + row / tr;
        const uint32_t first = off[e] + (uint32_t)it_in * units;
        const uint32_t c0 = owner(U, first, ctas), c1 = owner(U, first + units - 1, ctas);
        stride[k] = w ? Shape<true>::kSegFloats : Shape<false>::kSegFloats;
        base[k] = s.seg[w] + (size_t)(c0 + s.item[w][e] + it_in) * stride[k];
        tile_rows[k] = tr;
        row_in[k] = row % tr;
        twice[k] = w && n.ntok * G - (row / tr) * tr <= kWideHalf;
        count[k] = ((int)(c1 - c0) + 1) << twice[k];
    }
    const int total = count[0] + count[1];
    // part i of the row: where its segment lies, and the row in that segment
    auto part_of = [&](int i, const float** sg, int* rows, int* r) {
        const int k = i >= count[0], j = i - (k ? count[0] : 0);
        *sg = base[k] + (size_t)(j >> twice[k]) * stride[k];
        *rows = tile_rows[k];
        *r = row_in[k] + (twice[k] ? (j & 1) * kWideHalf : 0);
    };
    float M = -INFINITY;
    for (int i = lane; i < total; i += 32) {
        const float* sg;
        int rows, rr;
        part_of(i, &sg, &rows, &rr);
        M = fmaxf(M, __ldcg(sg + rr));
    }
    M = warp_max(M);
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
    constexpr int B = 4;
    for (int i0 = part; i0 < total; i0 += SPLIT * B) {
        float m[B], l[B];
        float4 v[B];
#pragma unroll
        for (int j = 0; j < B; ++j) {  // unconditional loads, all in flight together
            const float* sg;
            int rows, rr;
            part_of(min(i0 + j * SPLIT, total - 1), &sg, &rows, &rr);
            m[j] = __ldcg(sg + rr);
            l[j] = __ldcg(sg + rows + rr);
            v[j] = ld_cg_f4_ordered(sg + 2 * rows + rr * kDim + lane * 4);
        }
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const bool live = i0 + j * SPLIT < total && m[j] != -INFINITY;
            const float w = live ? exp2f(m[j] - M) : 0.f;
            den += live ? l[j] * w : 0.f;
            num.x += live ? v[j].x * w : 0.f; num.y += live ? v[j].y * w : 0.f;
            num.z += live ? v[j].z * w : 0.f; num.w += live ? v[j].w * w : 0.f;
        }
    }
    if (SPLIT > 1) {
        s_num[warp][lane] = num;
        if (lane == 0) s_den[warp] = den;
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int w = 1; w < SPLIT; ++w) {
            const float4 x = s_num[warp + w][lane];
            num.x += x.x; num.y += x.y; num.z += x.z; num.w += x.w;
            den += s_den[warp + w];
        }
    }
    if (!on) return;
    const float f = den == 0.f ? 0.f : a.v_scale / den;  // a row that sees no key gives zeros
    const __nv_bfloat162 lo = __floats2bfloat162_rn(num.x * f, num.y * f), hi = __floats2bfloat162_rn(num.z * f, num.w * f);
    reinterpret_cast<uint2*>(a.out)[((size_t)token * a.q_heads + head) * (kDim / 4) + lane] =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

// ------------------------------------------------------------------ host
static int sm_or_default() {
    const int n = mono_sm_count();
    return n > 0 ? n : 148;
}
static size_t up256(size_t v) { return (v + 255) & ~size_t(255); }
// Segments a launch may leave: one per CTA and one per item.
static size_t narrow_segments(size_t tokens, size_t q_heads, size_t kv_heads, size_t seqs, size_t groups) {
    const size_t tiles = (tokens * (q_heads / kv_heads)) / 16 + 1;
    return 2 * (size_t)sm_or_default() + kv_heads * (2 * tiles + seqs + groups);
}
// The wide kernel's entries have kWideRows rows at least, so there are at most 2 rows / kWideRows of them.
static size_t wide_segments(size_t tokens, size_t q_heads, size_t kv_heads) {
    const size_t rows = tokens * (q_heads / kv_heads);
    if (rows < kWideRows) return 0;
    return (size_t)sm_or_default() + kv_heads * 2 * (rows / Shape<true>::kTile + rows / kWideRows);
}
static size_t narrow_bytes(int tokens, int q_heads, int kv_heads, int seqs, int groups) {
    return up256(narrow_segments(tokens, q_heads, kv_heads, seqs, groups) * Shape<false>::kSegFloats * sizeof(float));
}

}  // namespace prefix_attn

extern "C" size_t mono_prefix_attn_scratch_bytes(int tokens, int q_heads, int kv_heads, int seqs, int groups) {
    using namespace prefix_attn;
    if (tokens < 1 || q_heads < 1 || kv_heads < 1 || seqs < 1 || groups < 0 || q_heads % kv_heads) return 0;
    return 4 * up256((size_t)(seqs + groups + 1) * 4) + narrow_bytes(tokens, q_heads, kv_heads, seqs, groups) +
           wide_segments(tokens, q_heads, kv_heads) * Shape<true>::kSegFloats * sizeof(float);
}

extern "C" int mono_prefix_attn_launch(const mono_prefix_attn_args* a, void* stream) {
    using namespace prefix_attn;
    const char* who = "mono_prefix_attn_launch";
    if (!a || a->tokens < 1 || a->tokens > (1 << 20) || a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads || a->q_heads / a->kv_heads > kMaxGroup ||
        a->kv_heads > 256) {
        mono_set_error("%s: 1..2^20 tokens, 1..256 kv heads and q_heads a multiple of kv_heads, at most %d to one, required", who, kMaxGroup);
        return MONO_E_ARG;
    }
    if (a->seqs < 1 || a->groups < 0 || a->seqs + a->groups > kMaxEntries) {
        mono_set_error("%s: at least one sequence, and at most %d sequences and groups, required", who, kMaxEntries);
        return MONO_E_ARG;
    }
    if (!a->q || !a->k_cache || !a->v_cache || !a->q_start || !a->page_table || !a->lens || a->pt_ld < 1 || !a->out || !a->scratch ||
        (a->groups && (!a->group_start || !a->prefix_table || !a->prefix_lens || a->prefix_ld < 1))) {
        mono_set_error("%s: q, caches, sequence tables, prefix tables (with groups), scratch and out required", who);
        return MONO_E_ARG;
    }
    if (a->q_ld < (long)a->q_heads * kDim || (a->q_ld & 7) || ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 15) ||
        (reinterpret_cast<uintptr_t>(a->scratch) & 255) || !(a->k_scale > 0.f) || !(a->v_scale > 0.f) || !(a->sm_scale > 0.f)) {
        mono_set_error("%s: q rows at least q_heads * 128 values apart (a multiple of 8) on 16-byte addresses, scratch on a 256-byte address and positive scales required", who);
        return MONO_E_ARG;
    }
    if (a->n_pages < 1 || a->n_pages > (1ll << 31) / kPage - 1 || a->pt_ld > (1 << 24) || a->prefix_ld > (1 << 24)) {
        mono_set_error("%s: 1..2^25 - 1 pages and tables of at most 2^24 pages a row required", who);
        return MONO_E_ARG;
    }
    // units are counted in 32 bits: 16-row tiles x pages, for the sequences' own keys and once more for the prefixes
    const double tiles = (double)a->tokens * (a->q_heads / a->kv_heads) / 16 + a->seqs + a->groups;
    if (tiles * a->kv_heads * ((double)a->pt_ld + a->prefix_ld) >= 4.0e9) {
        mono_set_error("%s: too much work for one launch (tiles x kv heads x table width above 4e9): split the tokens", who);
        return MONO_E_ARG;
    }
    const size_t need = mono_prefix_attn_scratch_bytes(a->tokens, a->q_heads, a->kv_heads, a->seqs, a->groups);
    if (a->scratch_bytes < need) {
        mono_set_error("%s: scratch of %zu bytes, needs %zu", who, a->scratch_bytes, need);
        return MONO_E_ARG;
    }
    Params p;
    const uint64_t inner = (uint64_t)a->kv_heads * kDim, rows = (uint64_t)a->n_pages * kPage;
    if (int rc = mono_tmap_encode_box(reinterpret_cast<mono_tmap_t*>(&p.kmap), a->k_cache, inner, rows, 1, inner, inner * rows, kPage)) return rc;
    if (int rc = mono_tmap_encode_box(reinterpret_cast<mono_tmap_t*>(&p.vmap), a->v_cache, inner, rows, 1, inner, inner * rows, kPage)) return rc;
    p.a = *a;
    uint8_t* at = reinterpret_cast<uint8_t*>(a->scratch);
    const size_t words = up256((size_t)(a->seqs + a->groups + 1) * 4);
    for (int w = 0; w < 2; ++w) {
        p.s.off[w] = reinterpret_cast<uint32_t*>(at);
        p.s.item[w] = reinterpret_cast<uint32_t*>(at + words);
        at += 2 * words;
    }
    p.s.seg[0] = reinterpret_cast<float*>(at);
    p.s.seg[1] = reinterpret_cast<float*>(at + narrow_bytes(a->tokens, a->q_heads, a->kv_heads, a->seqs, a->groups));
    const cudaStream_t st = (cudaStream_t)stream;
    const size_t smem = 1024 + kStages * 2 * kTileBytes + kConsumers * 16 * kPitch * sizeof(float) + 2 * (size_t)(a->seqs + a->groups + 1) * 4;
    static std::atomic<uint64_t> attr_once{0};  // bit d: set on device d
    if (attr_needed(attr_once)) {
        const size_t most = 1024 + kStages * 2 * kTileBytes + kConsumers * 16 * kPitch * sizeof(float) + 2 * (size_t)(kMaxEntries + 1) * 4;
        const cudaError_t e = cudaFuncSetAttribute(prefix_narrow_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (e != cudaSuccess) {
            mono_set_error("%s: %s", who, cudaGetErrorString(e));
            return (int)e;
        }
        attr_done(attr_once);
    }
    const int narrow = 2 * sm_or_default();
    const int wide = (long)a->tokens * (a->q_heads / a->kv_heads) >= kWideRows ? sm_or_default() : 0;  // no entry has more rows than the step
    cudaError_t e = wide ? launch_wide(p, wide, st) : cudaSuccess;
    if (e == cudaSuccess) e = launch_k(prefix_narrow_kernel, narrow, kThreads, smem, st, p);
    // Few rows: four warps share a row's segments (a long prefix leaves many of them); many rows: a warp each.
    if (e == cudaSuccess) {
        if ((long)a->tokens * a->q_heads < 2048)
            e = launch_k(prefix_merge_kernel<4>, dim3(a->tokens, a->q_heads), 128, 0, st, *a, p.s, narrow, wide);
        else
            e = launch_k(prefix_merge_kernel<1>, dim3(a->tokens, (a->q_heads + 3) / 4), 128, 0, st, *a, p.s, narrow, wide);
    }
    if (e != cudaSuccess) mono_set_error("%s: %s", who, cudaGetErrorString(e));
    return (int)e;
}
