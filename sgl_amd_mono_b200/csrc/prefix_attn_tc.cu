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
MONO_TL_DECLARE(tl_wide)

constexpr int kKeys = 128;
// warps 0..3: softmax of stream 0, 4..7: of stream 1
constexpr int kConvWarp0 = 8, kTmaWarp = 12, kMmaWarp = 13;
constexpr int kThreadsWide = 16 * 32;  // warps 14 and 15 only fill the fetching warps' warpgroup
// Registers per thread: 128 at launch, moved from the warpgroups that need few to the two softmax ones, which hold a
// X.
constexpr int kRegsSoftmax = 168, kRegsConv = 72, kRegsFetch = 104;
constexpr int kKStages = 3, kVStages = 2, kWStages = 2;  // K bytes, V bytes, widened V
constexpr int kQPlane = 128 * 128;                       // [128 rows][128 B]
constexpr int kKTile = kKeys * 128, kVTile = kKeys * 128, kWTile = 2 * kKeys * 128;
constexpr int kOkRing = 8;  // page flags outlive their K stage until the softmax of their unit
constexpr int kSmemFixed = 1024 + 2 * 2 * kQPlane + kKStages * kKTile + kVStages * kVTile + kWStages * kWTile;
constexpr int kTmemCols = 512;  // S of stream 0 and 1 (P over their first half), O of stream 0 and 1
constexpr float kBias = 7.f, kLazy = 8.f;

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// The roles share the instruction caches, and the issuing warp pays for every line the others push out (it took 0.5 us
// to issue eight products beside softmax loops unrolled over a whole block): waits are short code, and the loops below are
// rolled over quarters of a block.
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t limit_ns) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
    while (!mbar_try_wait(bar, parity)) {  // (each try sleeps for a while)
        if (*abort_flag) return false;
        if (globaltimer_ns() - t0 > limit_ns) {
            *abort_flag = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t r[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
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

// A block's scores, in two passes over tensor memory (a quarter is requested while the one before is worked on): their
// maximum, then the weights into P, over columns of S that have been read, and the weights' sum.  `vis`: how many of the
// block's keys this row sees; `ok`: which of its two pages exist.
template <bool MASK>
__device__ __forceinline__ float quarter_max(const uint32_t r[32], int c, int vis, int ok, float mx) {
    const int n = MASK ? (ok >> (c >> 1) & 1 ? vis - c * 32 : 0) : 32;
    float m4[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 32; ++i) m4[i & 3] = fmaxf(m4[i & 3], !MASK || i < n ? __uint_as_float(r[i]) : -INFINITY);
    return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
}
template <bool MASK>
__device__ __forceinline__ float block_max(uint32_t s_addr, int vis, int ok) {
    uint32_t a[32], b[32];
    float mx = -INFINITY;
    tmem_ld32(s_addr, a);
    wait_ld();
#pragma unroll 1
    for (int c = 0; c < 4; c += 2) {
        tmem_ld32(s_addr + (c + 1) * 32, b);
        mx = quarter_max<MASK>(a, c, vis, ok, mx);
        wait_ld();
        tmem_ld32(s_addr + ((c + 2) & 3) * 32, a);
        mx = quarter_max<MASK>(b, c + 1, vis, ok, mx);
        wait_ld();
    }
    return mx;
}
template <bool MASK>
__device__ __forceinline__ void quarter_weights(const uint32_t r[32], uint32_t s_addr, int c, int vis, int ok, float scale, float shift, float l4[4]) {
    const int n = MASK ? (ok >> (c >> 1) & 1 ? vis - c * 32 : 0) : 32;
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        float p0 = ex2(fmaf(__uint_as_float(r[i]), scale, shift)), p1 = ex2(fmaf(__uint_as_float(r[i + 1]), scale, shift));
        if (MASK) {
            p0 = i < n ? p0 : 0.f;
            p1 = i + 1 < n ? p1 : 0.f;
        }
        l4[i & 2] += p0;
        l4[(i & 2) + 1] += p1;
        w[i >> 1] = pack_half(p0, p1);
    }
    tmem_st16(s_addr + c * 16, w);
}
template <bool MASK>
__device__ __forceinline__ float block_weights(uint32_t s_addr, int vis, int ok, float scale, float shift) {
    uint32_t a[32], b[32];
    float l4[4] = {0.f, 0.f, 0.f, 0.f};
    tmem_ld32(s_addr, a);
    wait_ld();
#pragma unroll 1
    for (int c = 0; c < 4; c += 2) {
        tmem_ld32(s_addr + (c + 1) * 32, b);
        quarter_weights<MASK>(a, s_addr, c, vis, ok, scale, shift, l4);
        wait_ld();
        if (c == 0) tmem_ld32(s_addr + 64, a);
        quarter_weights<MASK>(b, s_addr, c + 1, vis, ok, scale, shift, l4);
        wait_ld();
    }
    return (l4[0] + l4[1]) + (l4[2] + l4[3]);
}

// The queries of a warp's 32 rows (row0 ..; those from `rows` on are zeros) as two planes of E4M3 in the layout of a
// K-major operand at `dst` (rows of 128 bytes, 16-byte pieces swizzled by the row's low three bits), each row scaled by
// the power of two that brings its largest value into [128, 256) (E4M3 ends at 448).  Half a warp loads a row (lines are
// read whole: many CTAs want the same queries at the same time).  Returns what undoes the scale of row0 + lane.
__device__ __forceinline__ float write_queries(const mono_prefix_attn_args& a, const Entry& en, int head, int G, int row0, int rows, uint8_t* dst) {
    const int lane = threadIdx.x & 31, half = lane >> 4, sub = lane & 15;
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)en.tok0 * a.q_ld + (size_t)head * G * kDim + sub * 8;
    float mine = 1.f;
    constexpr int B = 8;
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 2 * B) {
        uint4 v[B];
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const int row = row0 + r0 + 2 * j + half, r = row < rows ? row : 0, tok = r / G;
            v[j] = __ldg(reinterpret_cast<const uint4*>(q + (size_t)tok * a.q_ld + (size_t)(r - tok * G) * kDim));
        }
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const int at = r0 + 2 * j + half;
            const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
            uint32_t top = 0;  // the exponent of the largest |value|: NaN and infinity have the largest
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, max((w[i] << 16) & 0x7F800000u, w[i] & 0x7F800000u));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int ex = clamp_int((int)(top >> 23), 30, 254);
            const float up = row0 + at < rows ? __uint_as_float((uint32_t)(261 - ex) << 23) : 0.f;  // 2^(134 - ex)
            uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f0 = __uint_as_float(w[i] << 16) * up, f1 = __uint_as_float(w[i] & 0xFFFF0000u) * up;
                const __nv_fp8x2_storage_t hb = __nv_cvt_float2_to_fp8x2(make_float2(f0, f1), __NV_SATFINITE, __NV_E4M3);
                const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(hb, __NV_E4M3);
                const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&hr));
                const __nv_fp8x2_storage_t lb = __nv_cvt_float2_to_fp8x2(make_float2(f0 - hf.x, f1 - hf.y), __NV_SATFINITE, __NV_E4M3);
                hi[i >> 1] |= (uint32_t)hb << (16 * (i & 1));
                lo[i >> 1] |= (uint32_t)lb << (16 * (i & 1));
            }
            uint8_t* d = dst + at * 128 + (((sub >> 1) ^ (at & 7)) << 4) + (sub & 1) * 8;
            *reinterpret_cast<uint2*>(d) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(d + kQPlane) = make_uint2(lo[0], lo[1]);
            // infinite or NaN: saturation would hide it; a row of NaN
            float back = top == 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)(ex - 7) << 23);
            back = __shfl_sync(0xffffffffu, back, (lane & 1) * 16);
            if (lane >> 1 == (r0 >> 1) + j) mine = back;
        }
    }
    return mine;
}

// The CTA's current item, as every role walks it.
struct Item {
    Entry en;
    int head, row0, rows;  // first row, rows of the item (at most 256)
    int b0, blocks;        // first block of 128 keys, blocks to compute (those no row sees are left out)
    bool split;            // both streams have the same rows and take alternate blocks
    uint32_t seg, span;    // segment number; units of the list that this covers
    // stream st takes blocks first(st), first(st) + step, ...
    __device__ __forceinline__ int first(int st) const { return split ? st : 0; }
    __device__ __forceinline__ int step() const { return split ? 2 : 1; }
    __device__ __forceinline__ int count(int st) const { return split ? (blocks - st + 1) / 2 : blocks; }
};
__device__ __forceinline__ Item item_at(const mono_prefix_attn_args& a, const uint32_t* off, const uint32_t* item, uint32_t u, uint32_t u1) {
    Item it;
    const int E = a.groups + a.seqs, G = a.q_heads / a.kv_heads;
    const Place at = place_of(off, E, u);
    it.en = entry_of(a, at.e);
    it.head = at.head;
    const Work w = entry_work<true>(a, it.en);
    const int tile = min((int)at.local / w.units, w.tiles - 1), unit = (int)at.local - tile * w.units;
    it.row0 = tile * Shape<true>::kTile;
    it.rows = min(Shape<true>::kTile, it.en.ntok * G - it.row0);
    it.split = it.rows <= kWideHalf;
    it.span = min((uint32_t)((tile == w.tiles - 1 ? w.last : w.units) - unit), u1 - u);
    it.b0 = it.split ? 2 * unit : unit;
    const int seen = max(row_limit(it.en, it.row0 + it.rows - 1, G), 0);
    it.blocks = max(0, min((int)it.span * it.step(), (seen + kKeys - 1) / kKeys - it.b0));
    it.seg = blockIdx.x + it.head * item[E] + item[at.e] + tile;
    return it;
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
    __shared__ uint64_t q_full[2], s_full[2], p_full[2], o_full[2], j_free, j_full, j_done;
    __shared__ float s_join[2][128];  // stream 1's maxima and sums
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
        mbar_init(&j_free, 128);
        mbar_init(&j_full, 128);
        mbar_init(&j_done, 128);
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
    MONO_TL(tl_wide, 0);
    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0 && guard_failed(a.guard)) abort_flag = 1;
    MONO_TL(tl_wide, 1);
    make_plan<true, kThreadsWide>(a, p.s, off, item, red);
    MONO_TL(tl_wide, 2);
    const uint32_t U = off[E] * a.kv_heads, per = part_size(U, gridDim.x), u0 = min(blockIdx.x * per, U), u1 = min(u0 + per, U);
    const uint64_t wait_ns = a.wait_ns ? a.wait_ns : kWaitLimitNs;
    if (warp >= kTmaWarp) {
        regs_down<kRegsFetch>();
        if (u0 < u1 && warp == kTmaWarp) {
            // ---- fetch: lane l looks up the two pages of a batch's block l; lane 0 requests them in order
            int it = 0;
            for (uint32_t u = u0; u < u1 && !*abortp;) {
                const Item x = item_at(a, off, item, u, u1);
                const int pages = (x.en.len + kPage - 1) / kPage;
                for (int b = 0; b < x.blocks && !*abortp; b += 32) {
                    int pg[2] = {-1, -1};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int at = (x.b0 + min(b + lane, x.blocks - 1)) * 2 + h;
                        if (at < pages) pg[h] = x.en.table[at];
                        if (pg[h] >= a.n_pages) pg[h] = -1;
                    }
                    const int cnt = min(32, x.blocks - b);
                    for (int j = 0; j < cnt; ++j, ++it) {
                        const int g0 = __shfl_sync(0xffffffffu, pg[0], j), g1 = __shfl_sync(0xffffffffu, pg[1], j);
                        if (lane == 0 && !*abortp) {
                            const int ks = it % kKStages, vs = it % kVStages;
                            const uint32_t bytes = (g0 >= 0 ? kPage * 128 : 0) + (g1 >= 0 ? kPage * 128 : 0);
                            if (it < kKStages || wait_on(&k_empty[ks], ((it / kKStages) - 1) & 1, abortp, wait_ns)) {
                                page_ok[it % kOkRing] = (g0 >= 0 ? 1 : 0) | (g1 >= 0 ? 2 : 0);
                                mbar_expect_tx(&k_full[ks], bytes);
                                if (g0 >= 0) tma_load_3d(kbuf + ks * kKTile, &p.kmap, x.head * kDim, g0 * kPage, 0, &k_full[ks]);
                                if (g1 >= 0) tma_load_3d(kbuf + ks * kKTile + kPage * 128, &p.kmap, x.head * kDim, g1 * kPage, 0, &k_full[ks]);
                                if (it < kVStages || wait_on(&v_empty[vs], ((it / kVStages) - 1) & 1, abortp, wait_ns)) {
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
        } else if (u0 < u1 && warp == kMmaWarp) {
            // ---- the products: per stream S, (softmax), O, in the order that lets the streams alternate.  The warp walks
            // together and one elected lane issues, so that descriptors stay in uniform registers.
            {
                int it0 = 0;  // blocks before this item, over the CTA's life
                uint32_t qph[2] = {0, 0}, pph[2] = {0, 0};
                bool live = true;
                for (uint32_t u = u0; u < u1 && live;) {
                    const Item x = item_at(a, off, item, u, u1);
                    auto scores = [&](int st, int t) -> bool {  // S of the stream's t-th unit
                        const int i = it0 + x.first(st) + t * x.step(), ks = i % kKStages;
                        if (t == 0) {
                            if (!wait_on(&q_full[st], qph[st], abortp, wait_ns)) return false;
                            qph[st] ^= 1;
                        }
                        if (!wait_on(&k_full[ks], (i / kKStages) & 1, abortp, wait_ns)) return false;
                        fence_after();
                        const uint32_t q = smem_u32(qbuf + st * 2 * kQPlane), k = smem_u32(kbuf + ks * kKTile);
                        const uint64_t kd = desc_sw128(k, 0, 1024), qd = desc_sw128(q, 0, 1024);
                        if (elect_one()) {
#pragma unroll
                            for (int s = 0; s < 8; ++s) mma_f8(tmem + st * 128, qd + (s >> 2) * (kQPlane / 16) + 2 * (s & 3), kd + 2 * (s & 3), kIdescS, s > 0);
                            mma_commit(&s_full[st]);
                            if (x.split || st == 1) mma_commit(&k_empty[ks]);
                        }
                        __syncwarp();
                        return true;
                    };
                    auto values = [&](int st, int t) -> bool {  // O += P V of the stream's t-th unit
                        const int i = it0 + x.first(st) + t * x.step(), ws = i % kWStages;
                        if (!wait_on(&w_full[ws], (i / kWStages) & 1, abortp, wait_ns)) return false;
                        if (!wait_on(&p_full[st], pph[st], abortp, wait_ns)) return false;
                        pph[st] ^= 1;
                        fence_after();
                        const uint64_t wd = desc_sw128(smem_u32(wbuf + ws * kWTile), kKeys * 128, 1024);
                        if (elect_one()) {
#pragma unroll
                            for (int s = 0; s < 8; ++s)
                                mma_f16_ts(tmem + 256 + st * 128, tmem + st * 128 + s * 8, wd + s * (16 * 128 / 16), kIdescO, s > 0 || t > 0);
                            if (x.split || st == 1) mma_commit(&w_empty[ws]);
                            if (t == x.count(st) - 1) mma_commit(&o_full[st]);
                        }
                        __syncwarp();
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
                    it0 += x.blocks;
                    u += x.span;
                }
            }
        }
    } else if (warp >= kConvWarp0) {
        regs_down<kRegsConv>();
        if (u0 < u1) {
            // ---- widen V: bytes [key][dim], as TMA left them, to f16 in the layout of an MN-major operand.  Keys behind
            // the entry's last and pages that do not exist become zeros: 0 x NaN would be NaN.
            const int ct = tid - kConvWarp0 * 32;
            int it = 0;
            bool live = true;
            for (uint32_t u = u0; u < u1 && live;) {
                const Item x = item_at(a, off, item, u, u1);
                for (int i = 0; i < x.blocks && live; ++i, ++it) {
                    const int vs = it % kVStages, ws = it % kWStages;
                    live = wait_on(&v_full[vs], (it / kVStages) & 1, abortp, wait_ns) &&
                           (it < kWStages || wait_on(&w_empty[ws], ((it / kWStages) - 1) & 1, abortp, wait_ns));
                    if (!live) break;
                    const uint32_t src = smem_u32(vbuf + vs * kVTile), dst = smem_u32(wbuf + ws * kWTile);
                    const int have = x.en.len - (x.b0 + i) * kKeys, ok = page_ok[it % kOkRing];
#pragma unroll 2
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
        }
    } else {
        regs_up<kRegsSoftmax>();
        if (u0 < u1) {
            // ---- softmax: thread = row
            const int st = warp >> 2, row_in = tid & 127;
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t s_addr = tmem + lanes + st * 128, o_addr = tmem + lanes + 256 + st * 128;
            float* joint = reinterpret_cast<float*>(qbuf);  // [32 x 4 dims][128 rows] of stream 1, once a split item's queries are done with
            int it0 = 0;
            uint32_t sph = 0, oph = 0, jph = 0;
            bool live = true;
            for (uint32_t u = u0; u < u1 && live;) {
                const Item x = item_at(a, off, item, u, u1);
                const int row = x.row0 + (x.split ? row_in : st * 128 + row_in);
                const bool mine = row < x.row0 + x.rows;
                const int count = x.count(st);
                const bool join = x.split && x.count(1) > 0;  // stream 0 takes stream 1's part into its own
                float m = -INFINITY, l = 0.f;
                if (count > 0) {
                    const int w0 = (warp & 3) * 32;  // this warp's rows
                    const float qs = write_queries(a, x.en, x.head, G, x.row0 + (x.split ? 0 : st * 128) + w0, x.row0 + x.rows, qbuf + st * 2 * kQPlane + w0 * 128) *
                                     (a.sm_scale * a.k_scale * 1.4426950408889634f);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(&q_full[st]);
                    MONO_TL(tl_wide, 3);
                    const int lim = mine ? row_limit(x.en, row, G) : 0;
                    for (int t = 0; t < count; ++t) {
                        const int i = x.first(st) + t * x.step();
                        live = wait_on(&s_full[st], sph, abortp, wait_ns);
                        if (!live) break;
                        sph ^= 1;
                        fence_after();
                        MONO_TL(tl_wide, 4 + 3 * t);  // the first three blocks
                        // keys of the block that this row sees, of the pages that exist
                        const int vis = lim - (x.b0 + i) * kKeys, ok = page_ok[(it0 + i) % kOkRing];
                        const bool masked = !__all_sync(0xffffffffu, vis >= kKeys) || ok != 3;
                        const float mx = (masked ? block_max<true>(s_addr, vis, ok) : block_max<false>(s_addr, vis, ok)) * qs;
                        MONO_TL(tl_wide, 5 + 3 * t);
                        // raise the reference where it must be, and O with it
                        float up = 1.f;
                        if (mx > m + kLazy || (m == -INFINITY && mx > m)) {
                            up = m == -INFINITY ? 0.f : ex2(m - mx);
                            m = mx;
                        }
                        if (t > 0 && __any_sync(0xffffffffu, up != 1.f)) {
                            l *= up;
#pragma unroll 1
                            for (int c = 0; c < 8; ++c) {
                                uint32_t r16[16];
                                tmem_ld16(o_addr + c * 16, r16);
                                wait_ld();
#pragma unroll
                                for (int q = 0; q < 16; ++q) r16[q] = __float_as_uint(__uint_as_float(r16[q]) * up);
                                tmem_st16(o_addr + c * 16, r16);
                            }
                        }
                        const float shift = kBias - (m == -INFINITY ? 0.f : m);
                        l += masked ? block_weights<true>(s_addr, vis, ok, qs, shift) : block_weights<false>(s_addr, vis, ok, qs, shift);
                        wait_st();
                        fence_before();
                        mbar_arrive(&p_full[st]);
                        MONO_TL(tl_wide, 6 + 3 * t);
                    }
                    if (!live) break;
                    live = wait_on(&o_full[st], oph, abortp, wait_ns);
                    MONO_TL(tl_wide, 13);
                    if (!live) break;
                    oph ^= 1;
                    fence_after();
                }
                // ---- the segment's row; an item without blocks leaves an empty part
                float f0 = 1.f, f1 = 0.f;
                if (join) {
                    if (st == 1) {
                        // the other stream's queries are done with too: its last scores come before its part is asked for
                        live = wait_on(&j_free, jph, abortp, wait_ns);
                        if (!live) break;
                        s_join[0][row_in] = m;
                        s_join[1][row_in] = l;
#pragma unroll 1
                        for (int c = 0; c < 8; ++c) {
                            uint32_t r16[16];
                            tmem_ld16(o_addr + c * 16, r16);
                            wait_ld();
#pragma unroll
                            for (int q = 0; q < 16; q += 4)
                                *reinterpret_cast<uint4*>(joint + ((c * 4 + q / 4) * 128 + row_in) * 4) = make_uint4(r16[q], r16[q + 1], r16[q + 2], r16[q + 3]);
                        }
                        mbar_arrive(&j_full);
                    } else {
                        mbar_arrive(&j_free);
                        live = wait_on(&j_full, jph, abortp, wait_ns);
                        if (!live) break;
                        const float m1 = s_join[0][row_in], l1 = s_join[1][row_in], top = fmaxf(m, m1);
                        f0 = m == -INFINITY ? 0.f : ex2(m - top);
                        f1 = m1 == -INFINITY ? 0.f : ex2(m1 - top);
                        l = (l != l || l1 != l1) ? __uint_as_float(0x7FC00000u) : l * f0 + l1 * f1;
                        m = top;
                    }
                }
                if (!(x.split && st == 1)) {
                    float* seg = p.s.seg[1] + (size_t)x.seg * Shape<true>::kSegFloats;
                    const int at = st * 128 + row_in;
                    if (mine) {
                        seg[at] = l != l ? l : m - kBias;
                        seg[Shape<true>::kTile + at] = l;
                    }
                    float* dst = seg + 2 * Shape<true>::kTile + at * 4;  // [32 x 4 dims][256 rows][4]
#pragma unroll 1
                    for (int c = 0; c < 8; ++c) {
                        uint32_t r16[16];
                        if (count > 0) {
                            tmem_ld16(o_addr + c * 16, r16);
                            wait_ld();
                        } else {
#pragma unroll
                            for (int q = 0; q < 16; ++q) r16[q] = 0;
                        }
                        if (join) {
#pragma unroll
                            for (int q = 0; q < 16; q += 4) {
                                const float4 o = *reinterpret_cast<const float4*>(joint + ((c * 4 + q / 4) * 128 + row_in) * 4);
                                const float ov[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                                for (int k = 0; k < 4; ++k) r16[q + k] = __float_as_uint(__uint_as_float(r16[q + k]) * f0 + ov[k] * f1);
                            }
                        }
                        if (mine) {
#pragma unroll
                            for (int q = 0; q < 16; q += 4)
                                *reinterpret_cast<uint4*>(dst + (c * 4 + q / 4) * (Shape<true>::kTile * 4)) = make_uint4(r16[q], r16[q + 1], r16[q + 2], r16[q + 3]);
                        }
                    }
                }
                fence_before();
                if (join) {  // the next item's queries overwrite what stream 0 reads here
                    if (st == 0) mbar_arrive(&j_done);
                    live = wait_on(&j_done, jph, abortp, wait_ns);
                    jph ^= 1;
                }
                MONO_TL(tl_wide, 14);
                it0 += x.blocks;
                u += x.span;
            }
        }
    }
    fence_before();
    __syncthreads();
    MONO_TL(tl_wide, 15);
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

#ifdef MONO_TIMELINE
// Copies the wide kernel's stamps of the last launch to `out` (MONO_TL_CTAS x MONO_TL_POINTS); blocks the host.
extern "C" int mono_timeline_read_prefix_wide(unsigned long long* out, int* ctas, int* points) {
    *ctas = MONO_TL_CTAS;
    *points = MONO_TL_POINTS;
    return (int)cudaMemcpyFromSymbol(out, prefix_attn::tl_wide, sizeof(unsigned long long) * MONO_TL_CTAS * MONO_TL_POINTS);
}
#endif
