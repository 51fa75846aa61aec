// Shared-prefix attention for many rows on 5th-generation tensor cores (prefix_attn.cuh: how the work is cut).
//
// A block is one page (64 keys) of one kv head for up to 256 rows, which two streams of 128 rows (the TMEM lanes) work on:
//   S[row][key] = sum_d Q[row][d] K[key][d]   kind::f8f6f4, M 128, N 64, K 128, twice: the bf16 queries as two planes
//   O[row][dim] += sum_k P[row][k] V[k][dim]  kind::f16, M 128, N 128, K 64, P in tensor memory
// K is used as the bytes that lie in the cache: a query row, scaled by a power of two, is split into hi (E5M2) + lo (E4M3),
// exactly for values within 2^13 of the row's largest, and to 2^-21 of the largest below that.  P is f16 (11 bits, and with the bias below weights down to 2^-31 of
// the largest: two E4M3 planes would drop weights below 2^-18, which a long tail of small weights adds up), so four
// warps widen V to f16 in shared memory, which is exact.  Each stream has a warpgroup of softmax threads, one row each.
// The softmax takes a block's scores to registers at once, so the next block's are made while it works; P has two buffers,
// so it waits for the second product of two blocks before, which is long done.  An item of at most 128 rows gives both streams
// the same rows and alternate pages, and their two parts are joined in shared memory at its end.
//
// The running maximum is lazy: values are scaled to a reference that is raised (and O rescaled in tensor memory) only
// when a score passes it by 2^8, which f16 P has room for.
//
// Bound: per block and stream pair shared memory moves 168 KB (the queries are read again for every block: 6 KB for 32
// tensor cycles of the first product), 1312 cycles, the products take 1024 cycles and the exponentials 1024 (16 a cycle).
// Measured: 1.1 us (2100 cycles) a pair of blocks, 41 % of the tensor pipe: a stream's way from scores to weights is one
// dependent chain that two streams do not quite fill.  1442 rows of prompt chunks x 12 heads over 4100 + 1500 keys: 70 us, 590 TFLOP/s.
#include "prefix_attn.cuh"

namespace prefix_attn {
namespace {
MONO_TL_DECLARE(tl_wide)

// warps 0..3: softmax of stream 0, 4..7: of stream 1
constexpr int kConvWarp0 = 8, kTmaWarp = 12, kMmaWarp = 13;  // 13 and 14: the products of stream 0 and 1
constexpr int kThreadsWide = 16 * 32;                         // (warp 15 only fills the warpgroup)
// Registers per thread: 128 at launch, moved from the warpgroups that need few to the two softmax ones, which hold a
// block's 64 scores: 2 x 152 + 104 + 104 = 4 x 128.
constexpr int kRegsSoftmax = 152, kRegsConv = 104, kRegsFetch = 104;
constexpr int kKStages = 6, kVStages = 4, kWStages = 4;  // K bytes, V bytes, widened V
constexpr int kQPlane = 128 * 128;                       // [128 rows][128 B]
constexpr int kKTile = kPage * 128, kVTile = kPage * 128, kWTile = 2 * kPage * 128;
constexpr int kOkRing = 16;  // page flags outlive their K stage until the softmax of their block (eleven blocks at most)
constexpr int kSmemFixed = 1024 + 2 * 2 * kQPlane + kKStages * kKTile + kVStages * kVTile + kWStages * kWTile;
constexpr int kTmemCols = 512;  // per stream S (64 columns) and two buffers of P (32 each), then O of stream 0 and 1
constexpr float kBias = 7.f, kLazy = 8.f;

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// The roles share the instruction caches, and the issuing warp pays for every line the others push out (it took 0.5 us
// to issue eight products beside softmax loops unrolled over a whole block): waits are short code, and the loops below are
// rolled over quarters of a block.
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t limit_ns) {
    if (mbar_try_wait(bar, parity)) return true;
    uint64_t t0 = 0;
#pragma unroll 1
    for (uint32_t i = 1; !mbar_try_wait(bar, parity); ++i) {  // (each try sleeps for a while)
        if (i & 31) continue;  // the global timer is slow to read: only once a wait is clearly long
        const uint64_t now = globaltimer_ns();
        if (t0 == 0) t0 = now;
        if (*abort_flag) return false;
        if (now - t0 > limit_ns) {
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
constexpr uint32_t kIdescLo = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24);              // E4M3 x E4M3 -> f32, both K-major
constexpr uint32_t kIdescHi = kIdescLo | (1u << 7);                                               // E5M2 x E4M3
constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);  // f16 x f16 -> f32, B MN-major

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
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

// ------------------------------------------------------------------ queries
// Every query row as two planes of bytes, scaled by the power of two that brings its largest value into [2^11, 2^12), and
// what undoes the scale.  hi is the value's first three bits (E5M2, down to 2^-16); the rest has at most four more bits, is at
// most 2^8 (E4M3 ends at 448) and ends at 2^-9 in E4M3: values of 2^-2 and more are exact, smaller ones off by 2^-10 at most.
// (hi in E4M3 takes a largest value of 2^7 and is exact for 2^9 below it: scores of a row with one value of 1024 among
// values of 1 were off by 0.026.)  Image: [plane][kv head][token][head of the kv head][128 bytes].  Half a warp per row.
// (The rows are wanted by every CTA that has a part of their prefix: made by each of them, on its own rows, at its start, they
// cost 4 to 7 us of it.)
__global__ void __launch_bounds__(256) prefix_split_kernel(const mono_prefix_attn_args a, uint8_t* image, float* back_scale, uint32_t* share, int ctas) {
    pdl_prologue();
    if (blockIdx.x == 0) {
        make_share(a, share, (uint32_t)ctas);
        return;
    }
    const int lane = threadIdx.x & 31, sub = lane & 15;
    const unsigned G = a.q_heads / a.kv_heads, rows = (unsigned)a.tokens * a.q_heads;
    const unsigned r = ((blockIdx.x - 1) * 8 + (threadIdx.x >> 5)) * 2 + (lane >> 4);  // row of the image
    const unsigned k = min(r, rows - 1), per = (unsigned)a.tokens * G, kh = k / per, tok = (k - kh * per) / G, g = k - kh * per - tok * G;
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)tok * a.q_ld + (size_t)(kh * G + g) * kDim) + sub);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t top = 0;  // the exponent of the largest |value|: NaN and infinity have the largest
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, max((w[i] << 16) & 0x7F800000u, w[i] & 0x7F800000u));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int ex = clamp_int((int)(top >> 23), 30, 254);
    const float up = __uint_as_float((uint32_t)(265 - ex) << 23);  // 2^(11 - (ex - 127))
    uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float f0 = __uint_as_float(w[i] << 16) * up, f1 = __uint_as_float(w[i] & 0xFFFF0000u) * up;
        const __nv_fp8x2_storage_t hb = __nv_cvt_float2_to_fp8x2(make_float2(f0, f1), __NV_SATFINITE, __NV_E5M2);
        const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(hb, __NV_E5M2);
        const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&hr));
        const __nv_fp8x2_storage_t lb = __nv_cvt_float2_to_fp8x2(make_float2(f0 - hf.x, f1 - hf.y), __NV_SATFINITE, __NV_E4M3);
        hi[i >> 1] |= (uint32_t)hb << (16 * (i & 1));
        lo[i >> 1] |= (uint32_t)lb << (16 * (i & 1));
    }
    if (r >= rows) return;
    *reinterpret_cast<uint2*>(image + (size_t)r * 128 + sub * 8) = make_uint2(hi[0], hi[1]);
    *reinterpret_cast<uint2*>(image + ((size_t)rows + r) * 128 + sub * 8) = make_uint2(lo[0], lo[1]);
    // infinite or NaN: saturation would hide it; a row of NaN
    if (sub == 0) back_scale[r] = top == 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)(ex - 11) << 23);
}

// ------------------------------------------------------------------ attention
// f16 weights 2^(s scale + shift) of a block's scores, pairwise, their f32 sum and the scores' maximum.
__device__ __forceinline__ float weights(const uint32_t s[64], float scale, float shift, uint32_t w[32], float* mx) {
    float l4[4] = {0.f, 0.f, 0.f, 0.f}, m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int k = 0; k < 64; k += 2) {
        const float a = __uint_as_float(s[k]), b = __uint_as_float(s[k + 1]);
        const float p0 = ex2(fmaf(a, scale, shift)), p1 = ex2(fmaf(b, scale, shift));
        m2[(k >> 1) & 1] = max3(m2[(k >> 1) & 1], a, b);
        l4[k & 2] += p0;
        l4[(k & 2) + 1] += p1;
        w[k >> 1] = pack_half(p0, p1);
    }
    *mx = fmaxf(m2[0], m2[1]);
    return (l4[0] + l4[1]) + (l4[2] + l4[3]);
}

// The CTA's current item, as every role walks it.
struct Item {
    Entry en;
    int head, row0, rows;  // first row, rows of the item (at most 256)
    int b0, blocks;        // first page, pages to compute (those no row sees are left out)
    bool split;            // both streams have the same rows and take alternate pages
    uint32_t seg, span;    // segment number; units of the list that this covers
    int image;             // its first row in the query image
    // stream st takes blocks first(st), first(st) + step, ...
    __device__ __forceinline__ int first(int st) const { return split ? st : 0; }
    __device__ __forceinline__ int step() const { return split ? 2 : 1; }
    __device__ __forceinline__ int count(int st) const { return split ? (blocks - st + 1) / 2 : blocks; }
    __device__ __forceinline__ bool join() const { return split && blocks > 1; }  // both streams have a part of the same rows
};
__device__ __forceinline__ Item item_at(const mono_prefix_attn_args& a, const uint32_t* off, const uint32_t* item, uint32_t u, uint32_t u1) {
    Item it;
    const int E = a.groups + a.seqs, G = a.q_heads / a.kv_heads;
    const Place at = place_of(off, E, u);
    it.en = entry_of(a, at.e);
    it.head = at.head;
    const Work w = entry_work<true>(a, it.en);
    const int tile = min((int)at.local / w.units, w.tiles - 1), unit = (int)at.local - tile * w.units;
    it.row0 = tile * kWideTile;
    it.rows = min(kWideTile, it.en.ntok * G - it.row0);
    it.split = it.rows <= kWideHalf;
    it.span = min((uint32_t)((tile == w.tiles - 1 ? w.last : w.units) - unit), u1 - u);
    it.b0 = it.split ? 2 * unit : unit;
    const int seen = max(row_limit(it.en, it.row0 + it.rows - 1, G), 0);
    it.blocks = max(0, min((int)it.span * it.step(), (seen + kPage - 1) / kPage - it.b0));
    it.seg = blockIdx.x + it.head * item[E] + item[at.e] + tile;
    it.image = (it.head * a.tokens + it.en.tok0) * G + it.row0;
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
    __shared__ uint64_t q_full[2], q_free[2], s_full[2], s_free[2], p_full[2][2], o_done[2][2], j_free, j_full, j_done;
    __shared__ float s_join[2][128];  // stream 1's maxima and sums
    __shared__ int page_ok[kOkRing];
    __shared__ uint32_t red[64], tmem_base_s;
    __shared__ int abort_flag;
    volatile int* abortp = &abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i < kKStages; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 2); }
        for (int i = 0; i < kVStages; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 4); }
        for (int i = 0; i < kWStages; ++i) { mbar_init(&w_full[i], 128); mbar_init(&w_empty[i], 2); }
        for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_free[i], 1); mbar_init(&s_full[i], 1); mbar_init(&s_free[i], 4); mbar_init(&p_full[0][i], 4); mbar_init(&p_full[1][i], 4); mbar_init(&o_done[0][i], 1); mbar_init(&o_done[1][i], 1); }
        mbar_init(&j_free, 128);
        mbar_init(&j_full, 128);
        mbar_init(&j_done, 128);
        mbar_fence_init();
        prefetch_tmap(&p.kmap1);
        prefetch_tmap(&p.vmap1);
        prefetch_tmap(&p.qmap);
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
    pdl_wait();
    pdl_launch_dependents();  // only now: the narrow kernel starts on what the wait above waited for
    const uint32_t ctas = p.s.share[0];
    if (tid == 0 && guard_failed(a.guard)) abort_flag = 1;
    MONO_TL(tl_wide, 1);
    const bool used = blockIdx.x < ctas;
    if (used) make_plan<true, kThreadsWide>(a, p.s, off, item, red, ctas);
    MONO_TL(tl_wide, 2);
    const uint32_t U = used ? off[E] * a.kv_heads : 0, per = part_size(U, ctas), u0 = min(blockIdx.x * per, U), u1 = min(u0 + per, U);
    const uint64_t wait_ns = a.wait_ns ? a.wait_ns : kWaitLimitNs;
    if (warp >= kTmaWarp) {
        regs_down<kRegsFetch>();
        if (u0 < u1 && warp == kTmaWarp) {
            // ---- fetch: lane l looks up the page of a batch's block l; lane 0 requests them in order
            int it = 0;
            uint32_t fph[2] = {0, 0}, jph = 0;
            bool joined = false, used[2] = {false, false};  // how the item before used the query buffers
            for (uint32_t u = u0; u < u1 && !*abortp;) {
                const Item x = item_at(a, off, item, u, u1);
                if (lane == 0) {
                    // the streams' queries, once the last item's scores are made, or its parts joined in the same place
                    if (joined) {
                        wait_on(&j_done, jph, abortp, wait_ns);
                        jph ^= 1;
                    }
                    for (int st = 0; st < 2; ++st) {
                        if (used[st]) {
                            wait_on(&q_free[st], fph[st], abortp, wait_ns);
                            fph[st] ^= 1;
                        }
                        used[st] = x.count(st) > 0;
                        if (!used[st] || *abortp) continue;
                        mbar_expect_tx(&q_full[st], 2 * kQPlane);
                        for (int pl = 0; pl < 2; ++pl)
                            tma_load_3d(qbuf + (st * 2 + pl) * kQPlane, &p.qmap, 0, x.image + (x.split ? 0 : st * 128), pl, &q_full[st]);
                    }
                    joined = x.join();
                }
                __syncwarp();
                for (int b = 0; b < x.blocks && !*abortp; b += 32) {
                    int page = x.en.table[x.b0 + min(b + lane, x.blocks - 1)];
                    if (page >= a.n_pages) page = -1;
                    const int cnt = min(32, x.blocks - b);
                    for (int j = 0; j < cnt; ++j, ++it) {
                        const int g = __shfl_sync(0xffffffffu, page, j);
                        if (lane == 0 && !*abortp) {
                            const int ks = it % kKStages, vs = it % kVStages;
                            const uint32_t bytes = g >= 0 ? kPage * 128 : 0;
                            if (it < kKStages || wait_on(&k_empty[ks], ((it / kKStages) - 1) & 1, abortp, wait_ns)) {
                                page_ok[it % kOkRing] = g >= 0;
                                mbar_expect_tx(&k_full[ks], bytes);
                                if (g >= 0) tma_load_3d(kbuf + ks * kKTile, &p.kmap1, 0, g * kPage, x.head, &k_full[ks]);
                                if (it < kVStages || wait_on(&v_empty[vs], ((it / kVStages) - 1) & 1, abortp, wait_ns)) {
                                    mbar_expect_tx(&v_full[vs], bytes);
                                    if (g >= 0) tma_load_3d(vbuf + vs * kVTile, &p.vmap1, 0, g * kPage, x.head, &v_full[vs]);
                                }
                            }
                        }
                        __syncwarp();
                    }
                }
                u += x.span;
            }
        } else if (u0 < u1 && warp < kMmaWarp + 2) {
            // ---- the products of one stream.  The warp walks together and one elected lane issues, so that descriptors
            // stay in uniform registers.  (Waits, commits and issue cost a warp some 0.6 us a block: one warp for both streams
            // needed 1.5 us where the tensor core needs 0.7.)
            const int st = warp - kMmaWarp;
            int it0 = 0, g0 = 0;  // blocks before this item over the CTA's life, and of them this stream's
            uint32_t qph = 0;
            bool live = true;
            const uint64_t qd = desc_sw128(smem_u32(qbuf + st * 2 * kQPlane), 0, 1024);
            const uint32_t s_at = tmem + st * 128, o_at = tmem + 256 + st * 128;
            for (uint32_t u = u0; u < u1 && live;) {
                const Item x = item_at(a, off, item, u, u1);
                const int count = x.count(st), step = x.step();
                // A block's scores are asked for as soon as the softmax has the scores before in registers, ahead of that
                // block's values.  (The two products are of different kinds and end in no certain order: that P of block t is
                // used, and that O holds it, is asked of o_done, a barrier for even blocks and one for odd ones.)
                for (int t = -1; t < count && live; ++t) {
                    if (t + 1 < count) {  // S = Q K^T of block t + 1
                        const int i = it0 + x.first(st) + (t + 1) * step, ks = i % kKStages, g = g0 + t + 1;
                        if (t < 0) {
                            live = wait_on(&q_full[st], qph, abortp, wait_ns);
                            qph ^= 1;
                        }
                        live = live && wait_on(&k_full[ks], (i / kKStages) & 1, abortp, wait_ns) && (g == 0 || wait_on(&s_free[st], (g - 1) & 1, abortp, wait_ns));
                        if (!live) break;
                        fence_after();
                        const uint64_t kd = desc_sw128(smem_u32(kbuf + ks * kKTile), 0, 1024);
                        if (elect_one()) {
#pragma unroll
                            for (int s = 0; s < 8; ++s) mma_f8(s_at, qd + (s >> 2) * (kQPlane / 16) + 2 * (s & 3), kd + 2 * (s & 3), s < 4 ? kIdescHi : kIdescLo, s > 0);
                            mma_commit(&s_full[st]);
                            mma_commit(&k_empty[ks]);  // two arrivals free a stage: one per stream, or both from the only stream that uses it
                            if (x.split) mma_commit(&k_empty[ks]);
                            if (t + 1 == count - 1) mma_commit(&q_free[st]);
                        }
                        __syncwarp();
                    }
                    if (t >= 0) {  // O += P V of block t
                        const int i = it0 + x.first(st) + t * step, ws = i % kWStages, g = g0 + t;
                        live = wait_on(&w_full[ws], (i / kWStages) & 1, abortp, wait_ns) && wait_on(&p_full[st][g & 1], (g >> 1) & 1, abortp, wait_ns);
                        if (!live) break;
                        fence_after();
                        const uint64_t wd = desc_sw128(smem_u32(wbuf + ws * kWTile), kPage * 128, 1024);
                        if (elect_one()) {
#pragma unroll
                            for (int s = 0; s < 4; ++s) mma_f16_ts(o_at, s_at + 64 + (g & 1) * 32 + s * 8, wd + s * (16 * 128 / 16), kIdescO, s > 0 || t > 0);
                            mma_commit(&o_done[st][g & 1]);
                            mma_commit(&w_empty[ws]);
                            if (x.split) mma_commit(&w_empty[ws]);
                        }
                        __syncwarp();
                    }
                }
                g0 += count;
                it0 += x.blocks;
                u += x.span;
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
                const int every = row_limit(x.en, x.row0, G);  // keys below this are seen by all rows
                for (int i = 0; i < x.blocks && live; ++i, ++it) {
                    const int vs = it % kVStages, ws = it % kWStages;
                    live = wait_on(&v_full[vs], (it / kVStages) & 1, abortp, wait_ns) &&
                           (it < kWStages || wait_on(&w_empty[ws], ((it / kWStages) - 1) & 1, abortp, wait_ns));
                    if (!live) break;
                    const uint32_t src = smem_u32(vbuf + vs * kVTile), dst = smem_u32(wbuf + ws * kWTile);
                    const int have = page_ok[it % kOkRing] ? x.en.len - (x.b0 + i) * kPage : 0;
                    const int all = every - (x.b0 + i) * kPage;
                    if (all < min(have, kPage)) {
#pragma unroll 1
                        for (int j = 0; j < 4; ++j) {
                            const int key = (ct & 7) + 8 * j + 32 * (ct >> 6), c16 = (ct >> 3) & 7;
                            if (key >= all && key < have) drop_nan(src + key * 128 + ((c16 ^ (key & 7)) << 4), p.s.share + 2);
                        }
                    }
                    uint4 v[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {  // eight lanes: eight keys, no bank twice
                        const int key = (ct & 7) + 8 * j + 32 * (ct >> 6), c16 = (ct >> 3) & 7;
                        v[j] = lds128(src + key * 128 + ((c16 ^ (key & 7)) << 4));
                    }
                    if (have < kPage) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if ((ct & 7) + 8 * j + 32 * (ct >> 6) >= have) v[j] = make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int key = (ct & 7) + 8 * j + 32 * (ct >> 6), c16 = (ct >> 3) & 7;
                        const uint32_t at = dst + (c16 >> 2) * (kPage * 128) + key * 128, c = (c16 & 3) * 2;
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at + ((c ^ (key & 7)) << 4)), "r"(widen2(v[j].x)), "r"(widen2(v[j].x >> 16)), "r"(widen2(v[j].y)), "r"(widen2(v[j].y >> 16)) : "memory");
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at + (((c + 1) ^ (key & 7)) << 4)), "r"(widen2(v[j].z)), "r"(widen2(v[j].z >> 16)), "r"(widen2(v[j].w)), "r"(widen2(v[j].w >> 16)) : "memory");
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
            int it0 = 0, g0 = 0;  // blocks before this item over the CTA's life, and of them this stream's
            uint32_t jph = 0;
            bool live = true;
            for (uint32_t u = u0; u < u1 && live;) {
                const Item x = item_at(a, off, item, u, u1);
                const int row = x.row0 + (x.split ? row_in : st * 128 + row_in);
                const bool mine = row < x.row0 + x.rows;
                const int count = x.count(st);
                const bool join = x.join();  // stream 0 takes stream 1's part into its own
                float m = -INFINITY, l = 0.f;
                if (count > 0) {
                    const float qs = mine ? score_scale(a, __ldg(p.s.q_scale + x.image + row - x.row0)) : 1.f;
                    const int lim = mine ? row_limit(x.en, row, G) : 0;
                    for (int t = 0; t < count; ++t) {
                        const int i = x.first(st) + t * x.step(), g = g0 + t;
                        live = wait_on(&s_full[st], g & 1, abortp, wait_ns);
                        if (!live) break;
                        fence_after();
                        MONO_TL(tl_wide, 4 + 3 * t);  // the first three blocks
                        // how many of the block's keys this row sees
                        const int vis = page_ok[(it0 + i) % kOkRing] ? lim - (x.b0 + i) * kPage : 0;
                        uint32_t s[64];
                        tmem_ld32(s_addr, s);
                        tmem_ld32(s_addr + 32, s + 32);
                        wait_ld();
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&s_free[st]);
                        if (!__all_sync(0xffffffffu, vis >= kPage)) {
#pragma unroll
                            for (int k = 0; k < 64; ++k)
                                if (k >= vis) s[k] = 0xFF800000u;
                        }
                        // Weights by the reference as it is, and beside them the block's maximum (which so costs no time of
                        // its own); where it passes the reference too far, the reference is raised, O with it, and the
                        // weights are made again.
                        uint32_t w[32];
                        float mx, sum = weights(s, qs, kBias - (m == -INFINITY ? 0.f : m), w, &mx);
                        mx *= qs;
                        float up = 1.f;
                        if (mx > m + kLazy || (m == -INFINITY && mx > m)) {
                            up = m == -INFINITY ? 0.f : ex2(m - mx);
                            m = mx;
                        }
                        MONO_TL(tl_wide, 5 + 3 * t);
                        if (__any_sync(0xffffffffu, up != 1.f)) {
                            l *= up;
                            if (t > 0) {
                                live = wait_on(&o_done[st][(g - 1) & 1], ((g - 1) >> 1) & 1, abortp, wait_ns);  // the block before is in O
                                if (!live) break;
                                fence_after();
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
                            sum = weights(s, qs, kBias - (m == -INFINITY ? 0.f : m), w, &mx);
                        }
                        if (t > 1) {  // the place of these weights has been read
                            live = wait_on(&o_done[st][g & 1], ((g >> 1) - 1) & 1, abortp, wait_ns);
                            if (!live) break;
                            fence_after();
                        }
                        tmem_st16(s_addr + 64 + (g & 1) * 32, w);
                        tmem_st16(s_addr + 64 + (g & 1) * 32 + 16, w + 16);
                        l += sum;
                        wait_st();
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_full[st][g & 1]);
                        MONO_TL(tl_wide, 6 + 3 * t);
                    }
                    if (!live) break;
                    g0 += count;
                    live = wait_on(&o_done[st][(g0 - 1) & 1], ((g0 - 1) >> 1) & 1, abortp, wait_ns);
                    MONO_TL(tl_wide, 13);
                    if (!live) break;
                    fence_after();
                }
                // ---- the segment's row; an item without blocks leaves an empty part
                float f0 = 1.f, f1 = 0.f;
                if (join) {
                    if (st == 1) {
                        // the other stream's queries are done with too, and no thread of it still reads the item before's
                        live = wait_on(&j_free, jph, abortp, wait_ns);
                        if (!live) break;
                        s_join[0][row_in] = m;
                        s_join[1][row_in] = l;
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            uint32_t r32[32];
                            tmem_ld32(o_addr + c * 32, r32);
                            wait_ld();
#pragma unroll
                            for (int q = 0; q < 32; q += 4)
                                *reinterpret_cast<uint4*>(joint + ((c * 8 + q / 4) * 128 + row_in) * 4) = make_uint4(r32[q], r32[q + 1], r32[q + 2], r32[q + 3]);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // queries come here again
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
                    float* seg = p.s.seg[1] + (size_t)x.seg * seg_floats(kWideTile);
                    const int at = st * 128 + row_in;
                    if (mine) {
                        seg[at] = l != l ? l : m - kBias;
                        seg[kWideTile + at] = l;
                    }
                    float* dst = seg + 2 * kWideTile + at * 4;  // [32 x 4 dims][256 rows][4]
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t r32[32];
                        if (count > 0) {
                            tmem_ld32(o_addr + c * 32, r32);
                            wait_ld();
                        } else {
#pragma unroll
                            for (int q = 0; q < 32; ++q) r32[q] = 0;
                        }
                        if (join) {
#pragma unroll
                            for (int q = 0; q < 32; q += 4) {
                                const float4 o = *reinterpret_cast<const float4*>(joint + ((c * 8 + q / 4) * 128 + row_in) * 4);
                                const float ov[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                                for (int k = 0; k < 4; ++k) r32[q + k] = __float_as_uint(__uint_as_float(r32[q + k]) * f0 + ov[k] * f1);
                            }
                        }
                        if (mine) {
#pragma unroll
                            for (int q = 0; q < 32; q += 4)
                                *reinterpret_cast<uint4*>(dst + (c * 8 + q / 4) * (kWideTile * 4)) = make_uint4(r32[q], r32[q + 1], r32[q + 2], r32[q + 3]);
                        }
                    }
                }
                fence_before();
                if (join) {  // the next item's queries overwrite what stream 0 has read here
                    if (st == 0) mbar_arrive(&j_done);
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
    const unsigned rows = (unsigned)p.a.tokens * p.a.q_heads;
    const cudaError_t e = launch_k(prefix_split_kernel, 1 + (rows + 15) / 16, 256, 0, st, p.a, p.s.q_image, p.s.q_scale, p.s.share, ctas);
    if (e != cudaSuccess) return e;
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
