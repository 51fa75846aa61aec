// Attention of a batch whose sequences share long prefixes, over the paged E4M3 K and V caches: narrow split and merge.
//
//   out[t][h] = softmax over the keys that token t sees (its group's prefix, its sequence's own keys up to itself) of
//               (q[t][h] . k) k_scale sm_scale,  times v v_scale
//
// A prefix is read once for all tokens of its group: the rows of a tile come from every sequence of the group.
// prefix_attn.cuh says how the work is cut.  This file holds the kernel for few rows and the merge; prefix_attn_tc.cu
// the kernel for many.
#include <algorithm>

#include "prefix_attn.cuh"

extern void mono_set_error(const char* fmt, ...);
extern int mono_tmap_encode_box3(mono_tmap_t* out, const void* base, uint64_t inner_bytes, uint64_t rows, uint64_t outer, uint64_t row_stride_bytes,
                                 uint64_t outer_stride_bytes, uint32_t box_rows, uint32_t box_outer);

namespace prefix_attn {
MONO_TL_DECLARE(tl_narrow)

constexpr int kConsumers = 8;                        // warps that compute; one more fetches
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kStages = 5;
constexpr int kTileBytes = 128 * kDim;               // 128 rows of K (or V): 128 / heads keys of each head of the group
constexpr int kPitch = kDim + 4;                     // floats of a joint row: rows two apart start eight banks apart
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
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// a maximum that keeps NaN: a row with a NaN score is a row of NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {  // of a matrix of f16: lane (g, t) has row g, columns 2t, 2t + 1
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}

// The queries of eight rows in the layout of the B fragments of S^T = K Q^T, and their scales.  The contraction's order
// is free as long as both operands share it, so thread (g, t) of a fragment takes dims 32 t .. 32 t + 31 of row g: a key's
// 32 bytes are then two 16-byte shared loads.  A row is scaled by a power of two so that its largest value lies in
// [2^13, 2^14): f16 then holds every bf16 value down to 2^-28 of that exactly.  scale: of rows 2t and 2t + 1.
__device__ __forceinline__ void load_q(const mono_prefix_attn_args& a, const Entry& n, int head, int row0, int G, uint32_t q[8][2], float scale[2]) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3, row = row0 + g;
    const bool live = row < n.ntok * G;
    const int r = live ? row : 0;
    const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)(n.tok0 + r / G) * a.q_ld + (size_t)(head * G + r % G) * kDim + t * 32;
    uint4 raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j] = live ? __ldcg(reinterpret_cast<const uint4*>(src) + j) : make_uint4(0, 0, 0, 0);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[j] << 16)), fabsf(__uint_as_float(w[j] & 0xFFFF0000u))));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // exponent field of the largest value, kept where 2^(13 - e) and its inverse are normal numbers
    const int e = clamp_int((int)(__float_as_uint(amax) >> 23), 30, 254);
    const float up = __uint_as_float((uint32_t)(267 - e) << 23);  // 2^(13 - (e - 127))
    const float back = score_scale(a, __uint_as_float((uint32_t)(e - 13) << 23));
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) q[s][i] = pack_f16(__uint_as_float(w[2 * s + i] << 16) * up, __uint_as_float(w[2 * s + i] & 0xFFFF0000u) * up);
    scale[0] = __shfl_sync(0xffffffffu, back, 8 * t);
    scale[1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
}

// Up to 8 NT rows per tile, of every head of a group.  A unit's 128 rows of K and V arrive by one TMA box each, head after
// head (128-byte swizzle, which makes the 16-byte shared loads below free of bank conflicts); each of the eight warps
// takes 16 keys of one head, with a running maximum and sum of its own.  Where a head has several warps they join their
// parts at the segment's end.  The ninth warp keeps the ring of units full.  K and V stay bytes until a warp has them in
// registers, where they become f16 exactly.
//
// Bound: on all SMs HBM (80 us for 256 sequences of 512 keys, 48 heads on 8: fetching alone took 64); on the share of them
// that it has beside the wide kernel, mma.sync: of 1530 cycles a unit, 330 go to the first product, 200 to the softmax, 430 to
// the second, and 460 to the wait for the unit and the turn's start; a product of 16 x 8 x 16 occupies a quadrant's tensor pipe for 32 cycles,
// which are 1024 a unit.
//
// Both products are formed transposed: S^T[key][row] = K Q^T and O^T[dim][row] += V^T P^T, with keys and dims as the 16
// rows of the fragments and NT times 8 query rows as their columns: one token's heads are at most eight as a rule, and as
// the 16 rows they left most of the work empty.  P^T is turned from result to operand by two 8 x 8 transpositions.
// (Two tiles of eight rows take all 168 registers, and 72 bytes a thread are spilled.)
template <int NT>
__global__ void __launch_bounds__(kThreads, 1) prefix_narrow_kernel(const __grid_constant__ Params p) {
    constexpr int kTile = 8 * NT;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* comb = reinterpret_cast<float*>(ring + kStages * 2 * kTileBytes);  // [4 warps][kNarrowTile rows][kPitch]
    const mono_prefix_attn_args& a = p.a;
    const int E = a.groups + a.seqs;
    uint32_t* off = reinterpret_cast<uint32_t*>(comb + 4 * kNarrowTile * kPitch);
    uint32_t* item = off + E + 1;
    __shared__ uint64_t full[kStages], empty[kStages];
    __shared__ int page_ok[kStages];  // bit i: page i of the unit (a unit of one head has two)
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
    MONO_TL(tl_narrow, 0);
    // Beside the wide kernel, whose CTAs let this one start once all that was launched before them is done: what they
    // leave is not read here, and the wait for them is at the end (the merge waits for this kernel alone).
    pdl_launch_dependents();
    if (p.beside) __threadfence(); else pdl_wait();
    const uint32_t ctas = p.beside ? __ldcg(p.s.share + 1) : gridDim.x;
    MONO_TL(tl_narrow, 1);
    if (tid == 0 && guard_failed(a.guard)) abort_flag = 1;
    const bool used = blockIdx.x < ctas;
    if (used) make_plan<false, kThreads>(a, p.s, off, item, red, ctas);
    MONO_TL(tl_narrow, 2);
    const int G = a.q_heads / a.kv_heads, hg = group_heads(a.kv_heads), keys = unit_keys(a.kv_heads);
    const uint32_t U = used ? off[E] * head_groups(a.kv_heads) : 0, per = part_size(U, ctas), u0 = min(blockIdx.x * per, U), u1 = min(u0 + per, U);
    const uint64_t wait_ns = a.wait_ns ? a.wait_ns : kWaitLimitNs;
    if (u0 < u1) {
        if (warp == kConsumers) {
            // ---- fetch: 32 units' pages at a time are looked up by the lanes, then requested in order
            const int span = min(keys, kPage);  // keys of a box
            const int n_box = keys / span;
            int it = 0;
            bool given_up = false;
            for (uint32_t base = u0; base < u1 && !given_up; base += 32) {
                const uint32_t u = min(base + lane, u1 - 1);
                const Place at = place_of(off, E, u);
                const Entry en = entry_of(a, at.e);
                const Work w = entry_work<false>(a, en);
                const int key = (int)(at.local % (uint32_t)w.units) * keys;
                int row[2];  // of the cache, where the boxes start; -1: no such page
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int k = key + i * span, page = i < n_box && k < en.len ? en.table[k / kPage] : -1;
                    row[i] = page >= 0 && page < a.n_pages ? page * kPage + k % kPage : -1;
                }
                // A lane asks for its unit, a ring's worth of lanes at a time, so that slots that fall free together are filled
                // together.  (One lane for all took 900 to 1900 cycles a unit beside eight computing warps.)
                const int cnt = (int)min(32u, u1 - base), n = it + lane, st = n % kStages, head = at.head * hg;
                const uint32_t parity = (n / kStages - 1) & 1, box = (uint32_t)span * hg * kDim;
                uint8_t* dst = ring + st * 2 * kTileBytes;
                for (int j = 0; j < cnt && !given_up; j += kStages) {
                    bool todo = lane >= j && lane < min(j + kStages, cnt);
                    uint64_t t0 = 0;
                    for (uint32_t tries = 1; __any_sync(0xffffffffu, todo); ++tries) {
                        if (todo && (n < kStages || mbar_test(&empty[st], parity))) {
                            page_ok[st] = (row[0] >= 0 ? 1 : 0) | (row[1] >= 0 ? 2 : 0);
                            mbar_expect_tx(&full[st], ((row[0] >= 0 ? 2 : 0) + (row[1] >= 0 ? 2 : 0)) * box);
                            if (row[0] >= 0) {
                                tma_load_3d(dst, &p.kmap, 0, row[0], head, &full[st]);
                                tma_load_3d(dst + kTileBytes, &p.vmap, 0, row[0], head, &full[st]);
                            }
                            if (row[1] >= 0) {
                                tma_load_3d(dst + box, &p.kmap, 0, row[1], head, &full[st]);
                                tma_load_3d(dst + kTileBytes + box, &p.vmap, 0, row[1], head, &full[st]);
                            }
                            todo = false;
                        }
                        if (tries & 255) continue;
                        const uint64_t now = globaltimer_ns();
                        if (t0 == 0) t0 = now;
                        if (now - t0 > wait_ns) *abortp = 1;
                        given_up = __any_sync(0xffffffffu, *abortp);  // the consumers' waits see the flag
                        if (given_up) break;
                    }
                }
                it += cnt;
                __syncwarp();
            }
        } else {
            const int g = lane >> 2, t = lane & 3;
            const int h = warp & (hg - 1), slot = warp / hg, slots = kConsumers / hg;  // head of the group; which 16 of its keys
            const int rows_at = h * keys + slot * 16;                                  // in a unit's tile
            const int ok_bit = slot * 16 / kPage;
            int it = 0, nth = 0;
            for (uint32_t u = u0; u < u1; ++nth) {
                const Place at = place_of(off, E, u);
                const Entry en = entry_of(a, at.e);
                const Work wk = entry_work<false>(a, en);
                const int head = at.head * hg + h;
                const bool mine = head < a.kv_heads;
                const int tile = (int)(at.local / wk.units);
                const int p0 = (int)(at.local - (uint32_t)tile * wk.units), cnt = (int)min((uint32_t)(wk.units - p0), u1 - u);
                const int rows = en.ntok * G - tile * kTile;
                uint32_t q[NT][8][2];
                float qs[NT][2], m[NT][2], l[NT][2];
                int lim[NT][2], lim_all = en.len;  // keys below lim_all are seen by every row
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    load_q(a, en, mine ? head : 0, tile * kTile + n * 8, G, q[n], qs[n]);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int row = n * 8 + 2 * t + c;
                        lim[n][c] = row < rows ? min(row_limit(en, tile * kTile + row, G), en.len) : en.len;
                        lim_all = min(lim_all, lim[n][c]);
                        m[n][c] = -INFINITY;
                        l[n][c] = 0.f;
                    }
                }
                lim_all = __reduce_min_sync(0xffffffffu, lim_all);
                MONO_TL(tl_narrow, 3 + 4 * nth);  // the first three items
                float o[8][NT][4];  // dims 16 g + 2 j, 16 g + 2 j + 1 of rows 8 n + 2 t, 8 n + 2 t + 1
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[j][n][i] = 0.f;
                // Two units a turn where there are two: a warp's chain of loads, products, shuffles and exponentials is long, and
                // the second unit's runs beside the first's.
                for (int i = 0; i < cnt; i += 2) {
                    const int np = min(2, cnt - i);
                    uint32_t kb[2];
                    bool on[2];
                    int key0[2];  // this warp's first key of each unit
                    const int s0 = it % kStages, s1 = s0 + 1 == kStages ? 0 : s0 + 1;
                    const uint32_t ph0 = (it / kStages) & 1, ph1 = s1 == 0 ? ph0 ^ 1 : ph0;
                    // both asked at once, and waited for only where one is not there
                    const bool h0 = mbar_test(&full[s0], ph0), h1 = np < 2 || mbar_test(&full[s1], ph1);
                    bool have = true;
                    if (!h0) have = mbar_wait(&full[s0], ph0, abortp, wait_ns);
                    if (!h1) have = have && mbar_wait(&full[s1], ph1, abortp, wait_ns);
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const int st = z ? s1 : s0;
                        kb[z] = smem_u32(ring + st * 2 * kTileBytes) + rows_at * 128;
                        key0[z] = (p0 + i + z) * keys + slot * 16;
                        on[z] = z < np && have && mine && (page_ok[st] >> ok_bit & 1) && key0[z] < en.len;
                    }
                    if (!have) break;
                    if (i == 0) MONO_TL(tl_narrow, 4 + 4 * nth);
                    if (on[0] || on[1]) {
                        float s[2][NT][4];  // keys g and g + 8, rows 2t and 2t + 1
#pragma unroll
                        for (int z = 0; z < 2; ++z)
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int j = 0; j < 4; ++j) s[z][n][j] = on[z] ? 0.f : -INFINITY;
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            if (!on[z]) continue;
                            const uint32_t rowa = kb[z] + g * 128, c0 = ((2 * t) ^ g) << 4, c1 = ((2 * t + 1) ^ g) << 4;
                            const uint4 k00 = lds128(rowa + c0), k01 = lds128(rowa + c1), k10 = lds128(rowa + 1024 + c0), k11 = lds128(rowa + 1024 + c1);
                            const uint32_t wa[8] = {k00.x, k00.y, k00.z, k00.w, k01.x, k01.y, k01.z, k01.w};
                            const uint32_t wb[8] = {k10.x, k10.y, k10.z, k10.w, k11.x, k11.y, k11.z, k11.w};
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const uint32_t fa[4] = {e4m3x2_to_f16x2(wa[j]), e4m3x2_to_f16x2(wb[j]), e4m3x2_to_f16x2(wa[j] >> 16), e4m3x2_to_f16x2(wb[j] >> 16)};
#pragma unroll
                                for (int n = 0; n < NT; ++n) mma_f16(s[z][n], fa, q[n][j][0], q[n][j][1]);
                            }
                        }
                        // scores stay in the units of the product: qs > 0, so their maximum is the scaled scores'
#pragma unroll
                        for (int z = 0; z < 2; ++z)
                            if (on[z] && key0[z] + 16 > lim_all) {
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int j = 0; j < 4; ++j)
                                        if (key0[z] + g + 8 * (j >> 1) >= lim[n][j & 1]) s[z][n][j] = -INFINITY;
                            }
                        bool moved = false;
                        float alpha[NT][2];
                        uint32_t pb[2][NT][2];
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float base[2];
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                float mx = max_nan(max_nan(s[0][n][c], s[0][n][c + 2]), max_nan(s[1][n][c], s[1][n][c + 2]));
#pragma unroll
                                for (int x = 4; x < 32; x *= 2) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                                const float mn = max_nan(m[n][c], mx * qs[n][c]), zero = mn == -INFINITY ? 0.f : mn;
                                // a row that has seen no key yet keeps max = -inf, and weights of 0
                                alpha[n][c] = ex2(m[n][c] - zero);
                                moved = moved || alpha[n][c] != 1.f;
                                m[n][c] = mn;
                                l[n][c] *= alpha[n][c];
                                base[c] = kPBias - zero;
                            }
#pragma unroll
                            for (int z = 0; z < 2; ++z) {
                                float pv[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    pv[j] = ex2(fmaf(s[z][n][j], qs[n][j & 1], base[j & 1]));
                                    l[n][j & 1] += pv[j];
                                }
                                pb[z][n][0] = transpose8x8(pack_f16(pv[0], pv[1]));
                                pb[z][n][1] = transpose8x8(pack_f16(pv[2], pv[3]));
                            }
                        }
                        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int i = 0; i < 4; ++i) o[j][n][i] *= alpha[n][i & 1];
                        }
                        // V: thread (g, t) takes dims 16 g .. 16 g + 15 of keys 2t, 2t + 1, 2t + 8, 2t + 9; rows g and g + 8 of
                        // product j are dims 16 g + 2 j and 16 g + 2 j + 1.  Keys behind the entry's last hold anything, NaN
                        // among it, and 0 x NaN is NaN, so their bytes become zeros.
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            if (!on[z]) continue;
                            const uint32_t vb = kb[z] + kTileBytes;
                            if (lim_all < en.len && key0[z] + 16 > lim_all) {
#pragma unroll 1
                                for (int i4 = 0; i4 < 4; ++i4) {
                                    const int kr = 2 * t + (i4 & 1) + (i4 >> 1) * 8, key = key0[z] + kr;
                                    if (key >= lim_all && key < en.len) drop_nan(vb + kr * 128 + ((g ^ (kr & 7)) << 4), p.s.share + 2);
                                }
                                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next unit comes here
                            }
                            uint32_t vw[4][4];
#pragma unroll
                            for (int i4 = 0; i4 < 4; ++i4) {
                                const int kr = 2 * t + (i4 & 1) + (i4 >> 1) * 8;
                                const uint4 v = lds128(vb + kr * 128 + ((g ^ (kr & 7)) << 4));
                                vw[i4][0] = v.x; vw[i4][1] = v.y; vw[i4][2] = v.z; vw[i4][3] = v.w;
                            }
                            if (key0[z] + 16 > en.len) {
#pragma unroll
                                for (int i4 = 0; i4 < 4; ++i4)
                                    if (key0[z] + 2 * t + (i4 & 1) + (i4 >> 1) * 8 >= en.len) vw[i4][0] = vw[i4][1] = vw[i4][2] = vw[i4][3] = 0;
                            }
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const uint32_t a01 = __byte_perm(vw[0][j], vw[1][j], 0x5140), a23 = __byte_perm(vw[0][j], vw[1][j], 0x7362);
                                const uint32_t b01 = __byte_perm(vw[2][j], vw[3][j], 0x5140), b23 = __byte_perm(vw[2][j], vw[3][j], 0x7362);
                                const uint32_t f01[4] = {e4m3x2_to_f16x2(a01), e4m3x2_to_f16x2(a01 >> 16), e4m3x2_to_f16x2(b01), e4m3x2_to_f16x2(b01 >> 16)};
                                const uint32_t f23[4] = {e4m3x2_to_f16x2(a23), e4m3x2_to_f16x2(a23 >> 16), e4m3x2_to_f16x2(b23), e4m3x2_to_f16x2(b23 >> 16)};
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    mma_f16(o[2 * j][n], f01, pb[z][n][0], pb[z][n][1]);
                                    mma_f16(o[2 * j + 1][n], f23, pb[z][n][0], pb[z][n][1]);
                                }
                            }
                        }
                    }
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&empty[s0]);
                        if (np == 2) mbar_arrive(&empty[s1]);
                    }
                    it += np;
                }
                MONO_TL(tl_narrow, 5 + 4 * nth);
                // ---- the segment's rows of this head
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int x = 4; x < 32; x *= 2) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], x);
                if (slots > 1) {  // the head's warps bring their parts to one maximum and add them up in halves
                    if (g == 0) {
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                s_m[warp][n * 8 + 2 * t + c] = m[n][c];
                                s_l[warp][n * 8 + 2 * t + c] = l[n][c];
                            }
                    }
                    consumer_sync();
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float f[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int row = n * 8 + 2 * t + c;
                            float top = -INFINITY, sum = 0.f;
                            for (int k = 0; k < slots; ++k) top = fmaxf(top, s_m[k * hg + h][row]);
                            for (int k = 0; k < slots; ++k) {
                                const float mk = s_m[k * hg + h][row];
                                sum += mk == -INFINITY ? 0.f : s_l[k * hg + h][row] * ex2(mk - top);
                            }
                            f[c] = m[n][c] == -INFINITY ? 0.f : ex2(m[n][c] - top);
                            m[n][c] = top;
                            l[n][c] = sum;
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[j][n][i] *= f[i & 1];
                    }
                    for (int half = slots / 2; half >= 1; half /= 2) {
                        float* at4 = comb + ((slot & (half - 1)) * hg + h) * kTile * kPitch + g * 16;
                        if (slot >= half && slot < 2 * half) {
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int c = 0; c < 2; ++c)
#pragma unroll
                                    for (int j = 0; j < 8; j += 2)
                                        *reinterpret_cast<float4*>(at4 + (n * 8 + 2 * t + c) * kPitch + 2 * j) = make_float4(o[j][n][c], o[j][n][c + 2], o[j + 1][n][c], o[j + 1][n][c + 2]);
                        }
                        consumer_sync();
                        if (slot < half) {
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int c = 0; c < 2; ++c)
#pragma unroll
                                    for (int j = 0; j < 8; j += 2) {
                                        const float4 v = *reinterpret_cast<const float4*>(at4 + (n * 8 + 2 * t + c) * kPitch + 2 * j);
                                        o[j][n][c] += v.x; o[j][n][c + 2] += v.y; o[j + 1][n][c] += v.z; o[j + 1][n][c + 2] += v.w;
                                    }
                        }
                        consumer_sync();
                    }
                }
                if (slot == 0 && mine) {
                    float* seg = p.s.seg[0] + ((size_t)(blockIdx.x + at.head * item[E] + item[at.e] + tile) * hg + h) * seg_floats(kTile);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int row = n * 8 + 2 * t + c;
                            if (row >= rows) continue;
                            if (g == 0) {
                                seg[row] = l[n][c] != l[n][c] ? l[n][c] : m[n][c] - kPBias;  // a row of NaN stays one
                                seg[kTile + row] = l[n][c];
                            }
#pragma unroll
                            for (int j = 0; j < 8; j += 2)
                                *reinterpret_cast<float4*>(seg + 2 * kTile + row * kDim + g * 16 + 2 * j) = make_float4(o[j][n][c], o[j][n][c + 2], o[j + 1][n][c], o[j + 1][n][c + 2]);
                        }
                }
                MONO_TL(tl_narrow, 6 + 4 * nth);
                u += cnt;
            }
        }
    }
    __syncthreads();
    MONO_TL(tl_narrow, 15);
    if (p.beside) pdl_wait();
    if (*abortp) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the CTA's memory goes
        if (tid == 0 && !guard_failed(a.guard)) guard_fail(a.guard, MONO_ERR_DEADLINE, kSiteWait);
    }
}

// ------------------------------------------------------------------ merge
// The parts of one row that one kernel left for one entry: `count` segments `stride` floats apart.
struct Parts {
    const float *m, *v;  // the first part's maximum (its sum lies `rows` floats behind) and the first of this lane's values
    int rows, count, step;  // step: floats from the lane's first four values to the next four
    size_t stride;
};
__device__ __forceinline__ uint32_t over(uint32_t x, uint32_t per, uint32_t inverse) {  // x / per
    uint32_t c = __umulhi(x, inverse);
    if (c * per > x) --c;
    if (x - c * per >= per) ++c;
    return c;
}
__device__ __forceinline__ Parts parts_of(const mono_prefix_attn_args& a, const Scratch& s, const Record& n, int token, int kh, int in_group, int G, int sub) {
    Parts r = {nullptr, nullptr, 0, 0, 0, 0};
    const int wide = n.wide;
    const uint4 tot = *reinterpret_cast<const uint4*>(s.total[wide]);  // units and items of a list, units of a part, inverse
    if (n.tiles == 0 || tot.x == 0) return r;  // no keys, or refused tables
    const int row = (token - n.tok0) * G + in_group;
    const int shift = wide ? 8 : narrow_tile(a) == 8 ? 3 : 4;  // rows of a tile
    r.rows = 1 << shift;
    const int tile = row >> shift, at = row & (r.rows - 1);
    const int hg = wide ? 1 : group_heads(a.kv_heads), list = wide ? kh : kh / hg;
    const uint32_t first = list * tot.x + n.off + (uint32_t)tile * n.units;
    const uint32_t c0 = over(first, tot.z, tot.w), c1 = over(first + (tile == n.tiles - 1 ? n.last : n.units) - 1, tot.z, tot.w);
    r.stride = hg * seg_floats(r.rows);
    const float* seg = s.seg[wide] + (size_t)(c0 + list * tot.y + n.item + tile) * r.stride + (kh - list * hg) * seg_floats(r.rows);
    r.m = seg + at;
    // narrow: rows of 128 values; wide: four dims of all rows, then the next four (as a thread per row writes them)
    r.v = seg + 2 * r.rows + (wide ? (sub * 2 * kWideTile + at) * 4 : at * kDim + sub * 8);
    r.step = wide ? kWideTile * 4 : 4;
    r.count = (int)(c1 - c0) + 1;
    return r;
}

// NaN for those of this lane's eight dims that are NaN in a key which the token sees and the first row of its tile does not
// (prefix_attn.cuh).  Apart from the kernel's body, which it would take registers from.
static __device__ __noinline__ void mark_nan(const mono_prefix_attn_args& a, int e, int token, int head, int tile_rows) {
    const Entry n = entry_of(a, e);
    const int G = a.q_heads / a.kv_heads, kh = head / G, row = (token - n.tok0) * G + head - kh * G, dim = (threadIdx.x & 15) * 8;
    const int end = min(row_limit(n, row, G), n.len);
    for (int key = max(row_limit(n, row & ~(tile_rows - 1), G), 0); key < end; ++key) {
        const int page = n.table[key / kPage];
        if (page < 0 || page >= a.n_pages) continue;
        const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v_cache) + (((size_t)page * kPage + key % kPage) * a.kv_heads + kh) * kDim + dim);
        const uint32_t nan[2] = {nan_bytes(v.x), nan_bytes(v.y)};
        if (!(nan[0] | nan[1])) continue;
        for (int q = 0; q < 8; ++q)
            if (nan[q >> 2] >> (8 * (q & 3) + 7) & 1) reinterpret_cast<uint16_t*>(a.out)[((size_t)token * a.q_heads + head) * kDim + dim + q] = 0x7FC0;
    }
}

// Half a warp per (token, head): a lane holds eight dims, and the rows of neighbouring heads, which lie side by side in a
// wide segment, are read together.  SPLIT warps of a CTA share a pair of heads' parts; a batch of parts is requested at
// once and added to a running maximum, so a row of few parts costs one round trip.  Bound: latency, of tables, then parts
// (7 us for 48 rows, 11 us for 192 rows of 74 parts, 15 us for 12288 rows of 7 to 10).
template <int SPLIT>
__global__ void __launch_bounds__(128) prefix_merge_kernel(const __grid_constant__ mono_prefix_attn_args a, const __grid_constant__ Scratch s) {
    pdl_prologue();
    __shared__ float s_num[4][8][32], s_m[4][2], s_den[4][2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, half = lane >> 4, sub = lane & 15;
    const int token = blockIdx.x, head = (blockIdx.y * (4 / SPLIT) + warp / SPLIT) * 2 + half, part = warp % SPLIT;
    // The token's group and sequence.  Nobody clears the list between launches: what it says counts if the entry has the
    // token.
    const int E = a.groups + a.seqs;
    const int e[2] = {a.groups ? s.entry[0][token] : -1, s.entry[1][token]};
    Record rec[2];
    bool in[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        in[k] = k ? e[k] >= a.groups && e[k] < E : e[k] >= 0 && e[k] < a.groups;
        if (in[k]) rec[k] = s.rec[e[k]];
        in[k] = in[k] && token >= rec[k].tok0 && token < rec[k].tok0 + rec[k].ntok;
    }
    if (!in[1]) return;  // a token of no sequence: the row stays as it was
    // keys with NaN that this row may see and others of its tile do not: steps without the kernel for many rows have few of
    // them, and look without having been told to
    const bool look = rec[1].ntok > 1 && (!wide_step(a.tokens, a.q_heads / a.kv_heads) || s.share[2]);
    const int G = a.q_heads / a.kv_heads, kh = head / G;
    float M = -INFINITY, den = 0.f, num[8] = {};
    if (head < a.q_heads) {
        const Parts both[2] = {in[0] ? parts_of(a, s, rec[0], token, kh, head - kh * G, G, sub) : Parts{nullptr, nullptr, 0, 0, 0, 0},
                               parts_of(a, s, rec[1], token, kh, head - kh * G, G, sub)};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const Parts ps = both[k];
            constexpr int B = 4;
#pragma unroll 1
            for (int i0 = part; i0 < ps.count; i0 += SPLIT * B) {
                float m[B], l[B], top = M;
                float4 v[B][2];
#pragma unroll
                for (int j = 0; j < B; ++j) {  // all in flight together
                    m[j] = -INFINITY;
                    l[j] = 0.f;
                    v[j][0] = v[j][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (i0 + j * SPLIT < ps.count) {
                        const size_t o = (size_t)(i0 + j * SPLIT) * ps.stride;
                        m[j] = ps.m[o];
                        l[j] = ps.m[ps.rows + o];
                        v[j][0] = *reinterpret_cast<const float4*>(ps.v + o);
                        v[j][1] = *reinterpret_cast<const float4*>(ps.v + ps.step + o);
                    }
                }
#pragma unroll
                for (int j = 0; j < B; ++j) top = fmaxf(top, m[j]);
                // A part without keys (m = -inf) has sums of zeros, and so has its weight; without any, all stay zero.
                const float base = top == -INFINITY ? 0.f : top, old = exp2f(M - base);
                den *= old;
#pragma unroll
                for (int q = 0; q < 8; ++q) num[q] *= old;
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    const float w = exp2f(m[j] - base);  // NaN for a row of NaN
                    const float vv[8] = {v[j][0].x, v[j][0].y, v[j][0].z, v[j][0].w, v[j][1].x, v[j][1].y, v[j][1].z, v[j][1].w};
                    den = fmaf(l[j], w, den);
#pragma unroll
                    for (int q = 0; q < 8; ++q) num[q] = fmaf(vv[q], w, num[q]);
                }
                M = top;
            }
        }
    }
    if (SPLIT > 1) {
#pragma unroll
        for (int q = 0; q < 8; ++q) s_num[warp][q][lane] = num[q];
        if (sub == 0) { s_m[warp][half] = M; s_den[warp][half] = den; }
        __syncthreads();
        if (part != 0) return;
        float top = M;
#pragma unroll
        for (int w = 1; w < SPLIT; ++w) top = fmaxf(top, s_m[warp + w][half]);
        den = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) num[q] = 0.f;
#pragma unroll
        for (int w = 0; w < SPLIT; ++w) {
            const float d = s_den[warp + w][half], mw = s_m[warp + w][half];
            // (a part of NaN alone has no maximum, and NaN sums)
            const float f = mw != -INFINITY ? exp2f(mw - top) : d != d ? 1.f : 0.f;
            den += d * f;
#pragma unroll
            for (int q = 0; q < 8; ++q) num[q] += s_num[warp + w][q][lane] * f;
        }
    }
    if (head >= a.q_heads) return;
    const float f = den == 0.f ? 0.f : a.v_scale / den;  // a row that sees no key gives zeros
    uint32_t o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(num[2 * q] * f, num[2 * q + 1] * f);
        o[q] = *reinterpret_cast<const uint32_t*>(&b);
    }
    reinterpret_cast<uint4*>(a.out)[((size_t)token * a.q_heads + head) * (kDim / 8) + sub] = make_uint4(o[0], o[1], o[2], o[3]);
    if (look) mark_nan(a, s.entry[1][token], token, head, s.rec[s.entry[1][token]].wide ? kWideTile : narrow_tile(a));
}

// ------------------------------------------------------------------ host
static int sm_or_default() {
    const int n = mono_sm_count();
    return n > 0 ? n : 148;
}
static size_t up256(size_t v) { return (v + 255) & ~size_t(255); }
// Segments a launch may leave: one per CTA and one per item, for each head of a group.  Tiles of 16 rows: an entry that the
// narrow kernel has in a step of kWideStep rows or more fits one (two of half the size, if they have 8 rows); smaller steps
// have at most kWideStep - 1 rows of sequences and as many of groups, so two full tiles of each beside one per entry.
static size_t narrow_segments(size_t kv_heads, size_t seqs, size_t groups) {
    static_assert(kWideRows <= kNarrowTile + 1 && 17 <= kNarrowTile + 1 && kWideStep - 1 <= 2 * kNarrowTile, "what the count says");
    return group_heads((int)kv_heads) * ((size_t)sm_or_default() + head_groups((int)kv_heads) * (4 + seqs + groups));
}
// A token's rows lie in a sequence and, with groups, in a group.  The wide kernel's entries have kWideRows rows at least,
// which bounds their number.
static size_t wide_segments(size_t tokens, size_t q_heads, size_t kv_heads, size_t seqs, size_t groups) {
    const size_t rows = tokens * (q_heads / kv_heads), kinds = groups ? 2 : 1;
    if (!wide_step((int)tokens, (int)(q_heads / kv_heads))) return 0;
    return (size_t)sm_or_default() + kv_heads * (kinds * (rows / kWideTile) + std::min(kinds * (rows / kWideRows), seqs + groups));
}
// The wide kernel's queries (two planes of 128 bytes a row) and their scales; none where no entry can have so many rows.
static size_t image_bytes(size_t tokens, size_t q_heads, size_t kv_heads) {
    return !wide_step((int)tokens, (int)(q_heads / kv_heads)) ? 0 : up256(tokens * q_heads * 256) + up256(tokens * q_heads * 4);
}
static size_t narrow_bytes(int kv_heads, int seqs, int groups) {
    return up256(narrow_segments(kv_heads, seqs, groups) * seg_floats(kNarrowTile) * sizeof(float));
}

}  // namespace prefix_attn

extern "C" size_t mono_prefix_attn_scratch_bytes(int tokens, int q_heads, int kv_heads, int seqs, int groups) {
    using namespace prefix_attn;
    if (tokens < 1 || q_heads < 1 || kv_heads < 1 || seqs < 1 || groups < 0 || q_heads % kv_heads) return 0;
    return up256((size_t)(seqs + groups) * sizeof(Record)) + 256 + 2 * up256((size_t)tokens * 4) + image_bytes(tokens, q_heads, kv_heads) + narrow_bytes(kv_heads, seqs, groups) +
           wide_segments(tokens, q_heads, kv_heads, seqs, groups) * seg_floats(kWideTile) * sizeof(float);
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
        (reinterpret_cast<uintptr_t>(a->scratch) & 255) || !mono::scale_ok(a->k_scale) || !mono::scale_ok(a->v_scale) || !mono::scale_ok(a->sm_scale)) {
        mono_set_error("%s: q rows at least q_heads * 128 values apart (a multiple of 8) on 16-byte addresses, scratch on a 256-byte address and scales of 2^-100 .. 2^100 required", who);
        return MONO_E_ARG;
    }
    if (a->k_scale * a->sm_scale > 0x1p100f) {
        mono_set_error("%s: k_scale sm_scale of at most 2^100 required", who);
        return MONO_E_ARG;
    }
    if (a->n_pages < 1 || a->n_pages > (1ll << 31) / kPage - 1 || a->pt_ld > (1 << 24) || a->prefix_ld > (1 << 24)) {
        mono_set_error("%s: 1..2^25 - 1 pages and tables of at most 2^24 pages a row required", who);
        return MONO_E_ARG;
    }
    // units are counted in 32 bits: 16-row tiles x pages, for the sequences' own keys and once more for the prefixes
    const double tiles = (double)a->tokens * (a->q_heads / a->kv_heads) / 16 + a->seqs + a->groups;
    if (tiles * (a->kv_heads + 3) * ((double)a->pt_ld + a->prefix_ld) >= 4.0e9) {
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
    const int wide = wide_step(a->tokens, a->q_heads / a->kv_heads) ? sm_or_default() : 0;
    const int hg = group_heads(a->kv_heads), span = unit_keys(a->kv_heads) < kPage ? unit_keys(a->kv_heads) : kPage;
    for (int v = 0; v < 2; ++v) {  // boxes of the narrow kernel (the group's heads) and of the wide one (a head of a page)
        const uint8_t* cache = v ? a->v_cache : a->k_cache;
        if (int rc = mono_tmap_encode_box3(reinterpret_cast<mono_tmap_t*>(v ? &p.vmap : &p.kmap), cache, kDim, rows, a->kv_heads, inner, kDim, span, hg)) return rc;
        if (wide)
            if (int rc = mono_tmap_encode_box3(reinterpret_cast<mono_tmap_t*>(v ? &p.vmap1 : &p.kmap1), cache, kDim, rows, a->kv_heads, inner, kDim, kPage, 1)) return rc;
    }
    p.a = *a;
    uint8_t* at = reinterpret_cast<uint8_t*>(a->scratch);
    p.s.rec = reinterpret_cast<Record*>(at);
    at += up256((size_t)(a->seqs + a->groups) * sizeof(Record));
    for (int w = 0; w < 2; ++w) p.s.total[w] = reinterpret_cast<uint32_t*>(at) + 4 * w;
    p.s.share = reinterpret_cast<uint32_t*>(at) + 8;
    p.beside = wide > 0;
    at += 256;
    for (int w = 0; w < 2; ++w) {
        p.s.entry[w] = reinterpret_cast<int*>(at);
        at += up256((size_t)a->tokens * 4);
    }
    p.s.q_image = at;
    p.s.q_scale = reinterpret_cast<float*>(at + up256((size_t)a->tokens * a->q_heads * 256));
    at += image_bytes(a->tokens, a->q_heads, a->kv_heads);
    p.s.seg[0] = reinterpret_cast<float*>(at);
    p.s.seg[1] = reinterpret_cast<float*>(at + narrow_bytes(a->kv_heads, a->seqs, a->groups));
    const cudaStream_t st = (cudaStream_t)stream;
    constexpr size_t fixed = 1024 + kStages * 2 * kTileBytes + 4 * kNarrowTile * kPitch * sizeof(float);
    const size_t smem = fixed + 2 * (size_t)(a->seqs + a->groups + 1) * 4;
    static std::atomic<uint64_t> attr_once{0};  // bit d: set on device d
    if (attr_needed(attr_once)) {
        const size_t most = fixed + 2 * (size_t)(kMaxEntries + 1) * 4;
        cudaError_t e = cudaFuncSetAttribute(prefix_narrow_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(prefix_narrow_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (e != cudaSuccess) {
            mono_set_error("%s: %s", who, cudaGetErrorString(e));
            return (int)e;
        }
        attr_done(attr_once);
    }
    const int narrow = sm_or_default();
    const uint64_t q_rows = (uint64_t)a->tokens * a->q_heads;
    if (wide)
        if (int rc = mono_tmap_encode_box(reinterpret_cast<mono_tmap_t*>(&p.qmap), p.s.q_image, 128, q_rows, 2, 128, q_rows * 128, 128)) return rc;
    cudaError_t e = wide ? launch_wide(p, wide, st) : cudaSuccess;
    if (e == cudaSuccess) e = launch_k(narrow_tile(*a) == 8 ? prefix_narrow_kernel<1> : prefix_narrow_kernel<2>, narrow, kThreads, smem, st, p);
    // Few rows: four warps share two heads' segments (a long prefix leaves many of them); many rows: a warp each.  (64 tokens
    // of 48 heads: 103 us the whole step with four, 117 with one; 256 tokens: 184 with four, 176 with two, 175 with one.)
    if (e == cudaSuccess) {
        if ((long)a->tokens * a->q_heads < 8192)
            e = launch_k(prefix_merge_kernel<4>, dim3(a->tokens, (a->q_heads + 1) / 2), 128, 0, st, *a, p.s);
        else
            e = launch_k(prefix_merge_kernel<1>, dim3(a->tokens, (a->q_heads + 7) / 8), 128, 0, st, *a, p.s);
    }
    if (e != cudaSuccess) mono_set_error("%s: %s", who, cudaGetErrorString(e));
    return (int)e;
}

#ifdef MONO_TIMELINE
// Copies the narrow kernel's stamps of the last launch to `out` (MONO_TL_CTAS x MONO_TL_POINTS); blocks the host.
extern "C" int mono_timeline_read_prefix_narrow(unsigned long long* out, int* ctas, int* points) {
    *ctas = MONO_TL_CTAS;
    *points = MONO_TL_POINTS;
    return (int)cudaMemcpyFromSymbol(out, prefix_attn::tl_narrow, sizeof(unsigned long long) * MONO_TL_CTAS * MONO_TL_POINTS);
}
#endif
