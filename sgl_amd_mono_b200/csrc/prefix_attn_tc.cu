// Shared-prefix attention for many rows on 5th-generation tensor cores (prefix_attn.cuh: how the work is cut).
//
// A unit is 128 keys of one kv head for up to 256 rows, which two streams of 128 rows (the TMEM lanes) work on:
//   S[row][key] = sum_d Q[row][d] K[key][d]   kind::f8f6f4, M 128, N 128, K 128, twice: the bf16 queries as two E4M3 planes
//   O[row][dim] += sum_k P[row][k] V[k][dim]  kind::f16, M 128, N 128, K 128, P in tensor memory
// K is used as the bytes that lie in the cache: a query row, scaled by a power of two, is split into hi + lo E4M3 values,
// exactly for values within 2^12 of the row's largest.  P is f16 (11 bits, and with the bias below weights down to 2^-31 of
// the largest: two E4M3 planes would drop weights below 2^-18, which a long tail of small weights adds up), so four
// warps widen V to f16 in shared memory, which is exact.  Each stream has a warpgroup of softmax threads, one row each,
// and while it works on its scores the tensor core works for the other stream.  An item of at most 128 rows gives both
// streams the same rows and alternate units.
//
// The running maximum is lazy: values are scaled to a reference that is raised (and O rescaled in tensor memory) only
// when a score passes it by 2^8, which f16 P has room for.
//
// Bound: the two products are 4 x 128 x 128 x 128 multiply-adds a unit and stream pair, 2048 tensor cycles, against 2048
// cycles of exponentials (16 a cycle); from HBM a unit is 32 KB, read once for all 256 rows.
#include "prefix_attn.cuh"

namespace prefix_attn {
namespace {

constexpr int kKeys = 128;
constexpr int kSoftmaxThreads = 256;  // warps 0..3: stream 0, 4..7: stream 1
constexpr int kConvWarp0 = 8, kTmaWarp = 12, kMmaWarp = 13;
constexpr int kThreadsWide = 14 * 32;
constexpr int kKStages = 3, kVStages = 2, kWStages = 2;  // K bytes, V bytes, widened V
constexpr int kQPlane = 128 * 128;                       // [128 rows][128 B]
constexpr int kKTile = kKeys * 128, kVTile = kKeys * 128, kWTile = 2 * kKeys * 128;
constexpr int kOkRing = 8;  // page flags outlive their K stage until the softmax of their unit
constexpr int kSmemFixed = 1024 + 2 * 2 * kQPlane + kKStages * kKTile + kVStages * kVTile + kWStages * kWTile;
constexpr int kTmemCols = 512;  // S of stream 0 and 1 (P over their first half), O of stream 0 and 1
constexpr float kBias = 7.f, kLazy = 8.f;

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// A from tensor memory: lane = row, one 32-bit column = two f16 of the contraction
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
#define PA_REGS32(r) "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
// 32 columns of this thread's lane, requested; wait_ld() before they are used
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t r[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : PA_REGS32(r) : "r"(taddr) : "memory");
}
#undef PA_REGS32
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t r[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// Shared-memory matrix descriptors, 128-byte swizzle (sm_100 version 1).  K-major: rows of 128 bytes, groups of eight
// rows `sbo` apart.  MN-major: atoms of 128 contiguous bytes x 8 contraction rows, `sbo` apart along the contraction
// and `lbo` apart along the other dimension.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((saddr & 0x3FFFF) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
constexpr uint32_t kIdescS = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);               // E4M3 x E4M3 -> f32, both K-major
constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);  // f16 x f16 -> f32, B MN-major

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t widen2(uint32_t lo16) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(lo16 & 0xFFFFu), __NV_E4M3);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The CTA's current item, as every role walks it.
struct Item {
    Entry en;
    int head, row0, rows;  // first row, rows of the item (at most 256)
    int p0, units;         // first unit, units to compute (those no row sees are left out)
    bool split;            // both streams have the same rows and take alternate units
    uint32_t seg, span;    // segment number; units of the list that this covers
    // stream st takes units first(st), first(st) + step, ...
    __device__ __forceinline__ int first(int st) const { return split ? st : 0; }
    __device__ __forceinline__ int step() const { return split ? 2 : 1; }
    __device__ __forceinline__ int count(int st) const { return split ? (units - st + 1) / 2 : units; }
};
__device__ __forceinline__ Item item_at(const mono_prefix_attn_args& a, const uint32_t* off, const uint32_t* item, uint32_t u, uint32_t u1, int* e) {
    Item it;
    const int E = a.groups + a.seqs, G = a.q_heads / a.kv_heads;
    if (*e < 0) *e = find_entry(off, E, u);
    while (off[*e + 1] <= u) ++*e;
    it.en = entry_of(a, *e);
    int tiles, units;
    entry_work<true>(a, it.en, &tiles, &units);
    const uint32_t local = u - off[*e], in = local / units;
    it.head = (int)in / tiles;
    it.row0 = ((int)in % tiles) * Shape<true>::kTile;
    it.rows = min(Shape<true>::kTile, it.en.ntok * G - it.row0);
    it.split = it.rows <= kWideHalf;
    it.p0 = (int)(local % units);
    it.span = min((uint32_t)(units - it.p0), u1 - u);
    const int seen = max(row_limit(it.en, it.row0 + it.rows - 1, G), 0);
    it.units = max(0, min((int)it.span, (seen + kKeys - 1) / kKeys - it.p0));
    it.seg = blockIdx.x + item[*e] + in;
    return it;
}

// A unit's scores: weights into P, their sum into l.  `vis`: how many of the unit's keys this row sees; `ok`: which of
// its two pages exist.
template <bool MASK>
__device__ __forceinline__ float unit_max(uint32_t s_addr, int vis, int ok) {
    float mx = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        uint32_t r[32];
        tmem_ld32(s_addr + c * 32, r);
        wait_ld();
        const bool page = ok >> (c >> 1) & 1;
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float v = __uint_as_float(r[i]);
            if (MASK) v = page && c * 32 + i < vis ? v : -INFINITY;
            m4[i & 3] = fmaxf(m4[i & 3], v);
        }
        mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
    }
    return mx;
}
template <bool MASK>
__device__ __forceinline__ float unit_weights(uint32_t s_addr, int vis, int ok, float scale, float shift) {
    float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        uint32_t r[32], w[16];
        tmem_ld32(s_addr + c * 32, r);
        wait_ld();
        const bool page = ok >> (c >> 1) & 1;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float x0 = fmaf(__uint_as_float(r[i]), scale, shift), x1 = fmaf(__uint_as_float(r[i + 1]), scale, shift);
            if (MASK) {
                x0 = page && c * 32 + i < vis ? x0 : -INFINITY;
                x1 = page && c * 32 + i + 1 < vis ? x1 : -INFINITY;
            }
            const float p0 = ex2(x0), p1 = ex2(x1);
            l4[i & 2] += p0;
            l4[(i & 2) + 1] += p1;
            w[i >> 1] = pack_half(p0, p1);
        }
        tmem_st16(s_addr + c * 16, w);  // over columns of S that have been read
    }
    return (l4[0] + l4[1]) + (l4[2] + l4[3]);
}

__global__ void __launch_bounds__(kThreadsWide, 1) prefix_wide_kernel(const __grid_constant__ Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* qbuf = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));  // [stream][plane][128][128 B]
    uint8_t* kbuf = qbuf + 2 * 2 * kQPlane;
    uint8_t* vbuf = kbuf + kKStages * kKTile;
    uint8_t* wbuf = vbuf + kVStages * kVTile;  // [stage][dims 0-63 | 64-127][128 keys][128 B]
    const mono_prefix_attn_args& a = p.a;
    const int E = a.groups + a.seqs, G = a.q_heads / a.kv_heads;
    uint32_t* off = reinterpret_cast<uint32_t*>(wbuf + kWStages * kWTile);
    uint32_t* item = off + E + 1;
    __shared__ uint64_t k_full[kKStages], k_empty[kKStages], v_full[kVStages], v_empty[kVStages], w_full[kWStages], w_empty[kWStages];
    __shared__ uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
    __shared__ int page_ok[kOkRing];
    __shared__ uint32_t red[64], tmem_base_s;
    __shared__ int abort_flag;
    volatile int* abortp = &abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i < kKStages; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
        for (int i = 0; i < kVStages; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 4); }
        for (int i = 0; i < kWStages; ++i) { mbar_init(&w_full[i], 128); mbar_init(&w_empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 128); mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 128); mbar_init(&o_full[i], 1); }
        mbar_fence_init();
        prefetch_tmap(&p.kmap);
        prefetch_tmap(&p.vmap);
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base_s;
    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0 && guard_failed(a.guard)) abort_flag = 1;
    make_plan<true, kThreadsWide>(a, off, item, red);
    if (blockIdx.x == 0) {  // the merge reads it
        for (int e = tid; e <= E; e += kThreadsWide) {
            p.s.off[1][e] = off[e];
            p.s.item[1][e] = item[e];
        }
    }
    const uint32_t U = off[E], n = min(gridDim.x, U);
    const uint64_t wait_ns = a.wait_ns ? a.wait_ns : kWaitLimitNs;
    if (blockIdx.x < n) {
        const uint32_t u0 = cut(U, blockIdx.x, n), u1 = cut(U, blockIdx.x + 1, n);
        int e = -1;
        if (warp == kTmaWarp) {
            // ---- fetch: lane l looks up the two pages of a batch's unit l; lane 0 requests them in order
            int it = 0;
            for (uint32_t u = u0; u < u1 && !*abortp;) {
                const Item x = item_at(a, off, item, u, u1, &e);
                const int pages = (x.en.len + kPage - 1) / kPage;
                for (int b = 0; b < x.units && !*abortp; b += 32) {
                    int pg[2] = {-1, -1};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int at = (x.p0 + min(b + lane, x.units - 1)) * 2 + h;
                        if (at < pages) pg[h] = x.en.table[at];
                        if (pg[h] >= a.n_pages) pg[h] = -1;
                    }
                    const int cnt = min(32, x.units - b);
                    for (int j = 0; j < cnt; ++j, ++it) {
                        const int g0 = __shfl_sync(0xffffffffu, pg[0], j), g1 = __shfl_sync(0xffffffffu, pg[1], j);
                        if (lane == 0 && !*abortp) {
                            const int ks = it % kKStages, vs = it % kVStages;
                            const uint32_t bytes = (g0 >= 0 ? kPage * 128 : 0) + (g1 >= 0 ? kPage * 128 : 0);
                            if (it < kKStages || mbar_wait(&k_empty[ks], ((it / kKStages) - 1) & 1, abortp, wait_ns)) {
                                page_ok[it % kOkRing] = (g0 >= 0 ? 1 : 0) | (g1 >= 0 ? 2 : 0);
                                mbar_expect_tx(&k_full[ks], bytes);
                                if (g0 >= 0) tma_load_3d(kbuf + ks * kKTile, &p.kmap, x.head * kDim, g0 * kPage, 0, &k_full[ks]);
                                if (g1 >= 0) tma_load_3d(kbuf + ks * kKTile + kPage * 128, &p.kmap, x.head * kDim, g1 * kPage, 0, &k_full[ks]);
                                if (it < kVStages || mbar_wait(&v_empty[vs], ((it / kVStages) - 1) & 1, abortp, wait_ns)) {
                                    mbar_expect_tx(&v_full[vs], bytes);
                                    if (g0 >= 0) tma_load_3d(vbuf + vs * kVTile, &p.vmap, x.head * kDim, g0 * kPage, 0, &v_full[vs]);
                                    if (g1 >= 0) tma_load_3d(vbuf + vs * kVTile + kPage * 128, &p.vmap, x.head * kDim, g1 * kPage, 0, &v_full[vs]);
                                }
                            }
                        }
                        __syncwarp();
                    }
                }
                u += x.span;
            }
        } else if (warp == kMmaWarp) {
            // ---- the products: one thread issues; per stream S, (softmax), O, in the order that lets the streams alternate
            if (lane == 0) {
                int it0 = 0;                                    // units before this item, over the CTA's life
                uint32_t qph[2] = {0, 0}, pph[2] = {0, 0};
                bool live = true;
                for (uint32_t u = u0; u < u1 && live;) {
                    const Item x = item_at(a, off, item, u, u1, &e);
                    auto scores = [&](int st, int t) -> bool {  // S of the stream's t-th unit
                        const int i = it0 + x.first(st) + t * x.step(), ks = i % kKStages;
                        if (t == 0) {
                            if (!mbar_wait(&q_full[st], qph[st], abortp, wait_ns)) return false;
                            qph[st] ^= 1;
                        }
                        if (!mbar_wait(&k_full[ks], (i / kKStages) & 1, abortp, wait_ns)) return false;
                        fence_after();
                        const uint32_t q = smem_u32(qbuf + st * 2 * kQPlane), k = smem_u32(kbuf + ks * kKTile);
                        const uint64_t kd = desc_sw128(k, 0, 1024);
#pragma unroll
                        for (int pl = 0; pl < 2; ++pl) {
                            const uint64_t qd = desc_sw128(q + pl * kQPlane, 0, 1024);
#pragma unroll
                            for (int s = 0; s < 4; ++s) mma_f8(tmem + st * 128, qd + 2 * s, kd + 2 * s, kIdescS, pl + s > 0);
                        }
                        mma_commit(&s_full[st]);
                        if (x.split || st == 1) mma_commit(&k_empty[ks]);
                        return true;
                    };
                    auto values = [&](int st, int t) -> bool {  // O += P V of the stream's t-th unit
                        const int i = it0 + x.first(st) + t * x.step(), ws = i % kWStages;
                        if (!mbar_wait(&w_full[ws], (i / kWStages) & 1, abortp, wait_ns)) return false;
                        if (!mbar_wait(&p_full[st], pph[st], abortp, wait_ns)) return false;
                        pph[st] ^= 1;
                        fence_after();
                        const uint32_t w = smem_u32(wbuf + ws * kWTile);
#pragma unroll
                        for (int s = 0; s < 8; ++s)
                            mma_f16_ts(tmem + 256 + st * 128, tmem + st * 128 + s * 8, desc_sw128(w + s * 16 * 128, kKeys * 128, 1024), kIdescO, t > 0 || s > 0);
                        if (x.split || st == 1) mma_commit(&w_empty[ws]);
                        if (t == x.count(st) - 1) mma_commit(&o_full[st]);
                        return true;
                    };
                    for (int st = 0; st < 2 && live; ++st)
                        if (x.count(st) > 0) live = scores(st, 0);
                    for (int t = 0; t < x.count(0) && live; ++t)
                        for (int st = 0; st < 2 && live; ++st) {
                            if (t >= x.count(st)) continue;
                            live = values(st, t);
                            if (live && t + 1 < x.count(st)) live = scores(st, t + 1);
                        }
                    it0 += x.units;
                    u += x.span;
                }
            }
            __syncwarp();
        } else if (warp >= kConvWarp0) {
            // ---- widen V: bytes [key][dim], as TMA left them, to f16 in the layout of an MN-major operand.  Keys behind
            // the entry's last and pages that do not exist become zeros: 0 x NaN would be NaN.
            const int ct = tid - kConvWarp0 * 32;
            int it = 0;
            bool live = true;
            for (uint32_t u = u0; u < u1 && live;) {
                const Item x = item_at(a, off, item, u, u1, &e);
                for (int i = 0; i < x.units && live; ++i, ++it) {
                    const int vs = it % kVStages, ws = it % kWStages;
                    live = mbar_wait(&v_full[vs], (it / kVStages) & 1, abortp, wait_ns) &&
                           (it < kWStages || mbar_wait(&w_empty[ws], ((it / kWStages) - 1) & 1, abortp, wait_ns));
                    if (!live) break;
                    const uint32_t src = smem_u32(vbuf + vs * kVTile), dst = smem_u32(wbuf + ws * kWTile);
                    const int have = x.en.len - (x.p0 + i) * kKeys, ok = page_ok[it % kOkRing];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int key = (ct & 7) + 8 * j + 64 * (ct >> 6), c16 = (ct >> 3) & 7;  // eight lanes: eight keys, no bank twice
                        uint4 v = lds128(src + key * 128 + ((c16 ^ (key & 7)) << 4));
                        if (key >= have || !(ok >> (key >> 6) & 1)) v = make_uint4(0, 0, 0, 0);
                        const uint32_t at = dst + (c16 >> 2) * (kKeys * 128) + key * 128, c = (c16 & 3) * 2;
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at + ((c ^ (key & 7)) << 4)), "r"(widen2(v.x)), "r"(widen2(v.x >> 16)), "r"(widen2(v.y)), "r"(widen2(v.y >> 16)) : "memory");
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at + (((c + 1) ^ (key & 7)) << 4)), "r"(widen2(v.z)), "r"(widen2(v.z >> 16)), "r"(widen2(v.w)), "r"(widen2(v.w >> 16)) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(&w_full[ws]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_empty[vs]);
                }
                u += x.span;
            }
        } else {
            // ---- softmax: thread = row
            const int st = warp >> 2, row_in = tid & 127;
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t s_addr = tmem + lanes + st * 128, o_addr = tmem + lanes + 256 + st * 128;
            int it0 = 0;
            uint32_t sph = 0, oph = 0;
            bool live = true;
            for (uint32_t u = u0; u < u1 && live;) {
                const Item x = item_at(a, off, item, u, u1, &e);
                const int row = x.row0 + (x.split ? row_in : st * 128 + row_in);
                const bool mine = row < x.row0 + x.rows;
                const int count = x.count(st);
                float m = -INFINITY, l = 0.f;
                if (count > 0) {
                    // ---- the row's query, as two planes of E4M3 in the layout of a K-major operand
                    float qs;
                    {
                        const int r = mine ? row : x.row0;
                        const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)(x.en.tok0 + r / G) * a.q_ld + (size_t)(x.head * G + r % G) * kDim;
                        float amax = 0.f;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + j);
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int q = 0; q < 4; ++q) amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[q] << 16)), fabsf(__uint_as_float(w[q] & 0xFFFF0000u))));
                        }
                        // the power of two that brings the largest value into [128, 256): E4M3 ends at 448
                        const int ex = clamp_int((int)(__float_as_uint(amax) >> 23), 30, 254);
                        const float up = mine ? __uint_as_float((uint32_t)(261 - ex) << 23) : 0.f;  // 2^(134 - ex)
                        qs = __uint_as_float((uint32_t)(ex - 7) << 23) * (a.sm_scale * a.k_scale * 1.4426950408889634f);
                        uint8_t* dst = qbuf + st * 2 * kQPlane + row_in * 128;
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + 2 * c + h);
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    const float f0 = __uint_as_float(w[q] << 16) * up, f1 = __uint_as_float(w[q] & 0xFFFF0000u) * up;
                                    const __nv_fp8x2_storage_t hb = __nv_cvt_float2_to_fp8x2(make_float2(f0, f1), __NV_SATFINITE, __NV_E4M3);
                                    const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(hb, __NV_E4M3);
                                    const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&hr));
                                    const __nv_fp8x2_storage_t lb = __nv_cvt_float2_to_fp8x2(make_float2(f0 - hf.x, f1 - hf.y), __NV_SATFINITE, __NV_E4M3);
                                    hi[h * 2 + (q >> 1)] |= (uint32_t)hb << (16 * (q & 1));
                                    lo[h * 2 + (q >> 1)] |= (uint32_t)lb << (16 * (q & 1));
                                }
                            }
                            uint8_t* d = dst + ((c ^ (row_in & 7)) << 4);
                            *reinterpret_cast<uint4*>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                            *reinterpret_cast<uint4*>(d + kQPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        }
                        if (!(amax <= 3.0e38f)) qs = __uint_as_float(0x7FC00000u);  // a query of infinities or NaN: a row of NaN
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        mbar_arrive(&q_full[st]);
                    }
                    const int lim = mine ? row_limit(x.en, row, G) : 0;
                    for (int t = 0; t < count; ++t) {
                        const int i = x.first(st) + t * x.step();
                        live = mbar_wait(&s_full[st], sph, abortp, wait_ns);
                        if (!live) break;
                        sph ^= 1;
                        fence_after();
                        const int vis = lim - (x.p0 + i) * kKeys, ok = page_ok[(it0 + i) % kOkRing];
                        const bool plain = __all_sync(0xffffffffu, vis >= kKeys) && ok == 3;
                        const float mx = (plain ? unit_max<false>(s_addr, vis, ok) : unit_max<true>(s_addr, vis, ok)) * qs;
                        // raise the reference where it must be, and O with it
                        float up = 1.f;
                        if (mx > m + kLazy || (m == -INFINITY && mx > m)) {
                            up = m == -INFINITY ? 0.f : ex2(m - mx);
                            m = mx;
                        }
                        if (t > 0 && __any_sync(0xffffffffu, up != 1.f)) {
                            l *= up;
#pragma unroll 1
                            for (int c = 0; c < 4; ++c) {
                                uint32_t r[32];
                                tmem_ld32(o_addr + c * 32, r);
                                wait_ld();
#pragma unroll
                                for (int q = 0; q < 32; ++q) r[q] = __float_as_uint(__uint_as_float(r[q]) * up);
                                tmem_st16(o_addr + c * 32, r);
                                tmem_st16(o_addr + c * 32 + 16, r + 16);
                            }
                        }
                        const float shift = kBias - (m == -INFINITY ? 0.f : m);
                        l += plain ? unit_weights<false>(s_addr, vis, ok, qs, shift) : unit_weights<true>(s_addr, vis, ok, qs, shift);
                        wait_st();
                        fence_before();
                        mbar_arrive(&p_full[st]);
                    }
                    if (!live) break;
                    live = mbar_wait(&o_full[st], oph, abortp, wait_ns);
                    if (!live) break;
                    oph ^= 1;
                    fence_after();
                }
                // ---- the segment's row; a stream without units leaves an empty part
                float* seg = p.s.seg[1] + (size_t)x.seg * Shape<true>::kSegFloats;
                const int at = st * 128 + row_in;
                if (mine) {
                    seg[at] = l != l ? l : m - kBias;
                    seg[Shape<true>::kTile + at] = l;
                }
                if (count > 0) {
                    float* dst = seg + 2 * Shape<true>::kTile + at * kDim;
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t r[32];
                        tmem_ld32(o_addr + c * 32, r);
                        wait_ld();
                        if (mine) {
#pragma unroll
                            for (int q = 0; q < 32; q += 4)
                                *reinterpret_cast<uint4*>(dst + c * 32 + q) = make_uint4(r[q], r[q + 1], r[q + 2], r[q + 3]);
                        }
                    }
                    fence_before();
                } else if (mine) {
                    for (int q = 0; q < kDim; q += 4) *reinterpret_cast<uint4*>(seg + 2 * Shape<true>::kTile + at * kDim + q) = make_uint4(0, 0, 0, 0);
                }
                it0 += x.units;
                u += x.span;
            }
        }
    }
    fence_before();
    __syncthreads();
    if (*abortp) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies and products in flight end before the CTA's memory goes
        if (tid == 0 && !guard_failed(a.guard)) guard_fail(a.guard, MONO_ERR_DEADLINE, kSiteWait);
    }
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

}  // namespace

cudaError_t launch_wide(const Params& p, int ctas, cudaStream_t st) {
    static std::atomic<uint64_t> attr_once{0};  // bit d: set on device d
    if (attr_needed(attr_once)) {
        const cudaError_t e = cudaFuncSetAttribute(prefix_wide_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemFixed + 2 * (kMaxEntries + 1) * 4);
        if (e != cudaSuccess) return e;
        attr_done(attr_once);
    }
    return launch_k(prefix_wide_kernel, ctas, kThreadsWide, kSmemFixed + 2 * (size_t)(p.a.seqs + p.a.groups + 1) * 4, st, p);
}

}  // namespace prefix_attn
