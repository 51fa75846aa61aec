// What the kernels of the shared-prefix attention have in common: the entries of a step, the split of their work over
// the CTAs, and where a partial result lies.
//
// An entry is a set of query tokens with the one table of keys they all read: group g's tokens with the group's shared
// prefix (entries 0 .. groups-1), or sequence b's tokens with the sequence's own pages (entries groups ..).  For each
// kv head an entry's rows are its tokens x the q heads of that kv head, token-major, cut into tiles of kTile rows; an
// item is (entry, kv head, tile), and its units are the blocks of keys that the tile walks.  The units of all items,
// in order, are one list that is cut into equal parts, one per CTA, whatever the lengths are: a long prefix is split
// over many CTAs, and a CTA takes many short sequences.  The part of an item that one CTA computes is a segment; it
// leaves (max, sum, unnormalised values) per row, and a merge adds the segments of a row's two items.  Lengths are
// device data, so every CTA makes this plan itself, by one scan over the entries.
#pragma once
#include "mono_common.cuh"

namespace prefix_attn {
using namespace mono;

constexpr int kDim = 128;
constexpr int kMaxGroup = 16;      // q heads per kv head
constexpr int kMaxEntries = 2048;  // sequences + groups
constexpr int kSiteWait = 103, kSiteTables = 104;  // guard sites: a wait that ran out, starts that contradict themselves

struct Entry {
    int tok0, ntok, len, causal;
    const int32_t* table;
};

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Entry e's tokens and keys.  Tables that contradict themselves give some in-range answer.
__device__ __forceinline__ Entry entry_of(const mono_prefix_attn_args& a, int e) {
    Entry r;
    int s0, s1;
    if (e < a.groups) {
        s0 = clamp_int(a.group_start[e], 0, a.seqs);
        s1 = clamp_int(a.group_start[e + 1], s0, a.seqs);
        r.len = clamp_int(a.prefix_lens[e], 0, a.prefix_ld * kPage);
        r.table = a.prefix_table + (size_t)e * a.prefix_ld;
        r.causal = 0;
    } else {
        s0 = e - a.groups;
        s1 = s0 + 1;
        r.len = clamp_int(a.lens[s0], 0, a.pt_ld * kPage);
        r.table = a.page_table + (size_t)s0 * a.pt_ld;
        r.causal = 1;
    }
    r.tok0 = clamp_int(a.q_start[s0], 0, a.tokens);
    r.ntok = clamp_int(a.q_start[s1], r.tok0, a.tokens) - r.tok0;
    return r;
}
// Keys that row r (of the entry's rows) sees: all, or for a sequence's own keys all up to its own.
__device__ __forceinline__ int row_limit(const Entry& n, int row, int G) {
    return n.causal ? n.len - n.ntok + 1 + row / G : n.len;
}

// What a product of a scaled query row is multiplied by to be a score in powers of two; `back` undoes the row's scale.  Not
// 0, which would make NaN of the -inf of masked keys: products end at 2^30, so below 2^-126 every score is next to 0 anyway.
__device__ __forceinline__ float score_scale(const mono_prefix_attn_args& a, float back) {
    const float f = back * (a.sm_scale * a.k_scale * 1.4426950408889634f);
    return f < 0x1p-126f ? 0x1p-126f : f;  // (NaN, of a row of NaN, stays)
}

// E4M3 bytes of NaN, as bit 7 of each.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
// A weight of zero does not hide a NaN value from a matrix product.  So values of keys that not all rows of a tile see go to the
// product without their NaN bytes (taken out of the 16 bytes at `at` in shared memory before they are read, out of the way
// of the blocks without such keys), and the merge gives their NaN to the rows that do see them.
__device__ __forceinline__ void drop_nan(uint32_t at, uint32_t* found) {
    uint32_t w[4];
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    const uint32_t nan[4] = {nan_bytes(w[0]), nan_bytes(w[1]), nan_bytes(w[2]), nan_bytes(w[3])};
    if (!(nan[0] | nan[1] | nan[2] | nan[3])) return;
    *found = 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] &= ~((nan[i] >> 7) * 0xFFu);
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}

// A kernel's view of the work: narrow (8- or 16-row tiles, for a group of up to 8 kv heads at once) or wide (256-row tiles, one kv
// head).  A narrow unit is 128 rows of K and V, (keys x heads of the group): a token's heads lie side by side in the
// cache, and read together they come from HBM at its full rate, which they do not head by head.  A wide unit is one page;
// a wide item of at most kWideHalf rows gives its CTA's two halves the same rows and alternate pages, so that its units
// are two pages and cost what the others' do.
constexpr int kWideTile = 256, kNarrowTile = 16;
__host__ __device__ constexpr int seg_floats(int tile) { return 2 * tile + tile * kDim; }  // max, sum, values
// Rows of a narrow tile.  With eight the products are as wide as the rows of one token of up to eight q heads; steps of
// several tokens a sequence (or more heads) take sixteen, so as not to read their keys twice.
__host__ __device__ __forceinline__ int narrow_tile(const mono_prefix_attn_args& a) { return a.q_heads / a.kv_heads <= 8 && a.tokens <= a.seqs ? 8 : kNarrowTile; }
constexpr int kWideHalf = 128;
// kv heads of a narrow group (the last group of a step may have fewer): a power of two
__host__ __device__ __forceinline__ int group_heads(int kv_heads) { return kv_heads >= 8 ? 8 : kv_heads >= 4 ? 4 : kv_heads >= 2 ? 2 : 1; }
__host__ __device__ __forceinline__ int head_groups(int kv_heads) { return (kv_heads + group_heads(kv_heads) - 1) / group_heads(kv_heads); }
__host__ __device__ __forceinline__ int unit_keys(int kv_heads) { return 128 / group_heads(kv_heads); }
// Rows of an entry from which the wide kernel takes it.  An entry of a few tiles reads its keys once per tile, the wide
// kernel once: that wins from three tiles of 8 rows (256 samples of prompts with 17 to 48 rows: 149 us wide, 158 narrow; 10
// rows of a prefix of 11312 keys: 49 wide, 41 narrow) and from one of 16 that is more than half full (14 rows, 30499 keys:
// 77 wide, 112 narrow).  A step of fewer rows than kWideStep in all stays narrow: the wide kernel's launch and start cost it
// more (24 rows: 21 us wide, 16 narrow).
constexpr int kWideRows = 9, kWideStep = 33;
__host__ __device__ __forceinline__ bool wide_step(int tokens, int G) { return (long)tokens * G >= kWideStep; }
__device__ __forceinline__ bool is_wide(const mono_prefix_attn_args& a, int rows) {
    return rows >= (narrow_tile(a) == 8 ? 17 : kWideRows) && wide_step(a.tokens, a.q_heads / a.kv_heads);
}

struct Work {
    int tiles, units, last;  // row tiles; units of a tile, and of the last one
    __device__ __forceinline__ int per_head() const { return (tiles - 1) * units + last; }
};
template <bool WIDE>
__device__ __forceinline__ Work entry_work(const mono_prefix_attn_args& a, const Entry& n) {
    const int rows = n.ntok * (a.q_heads / a.kv_heads);
    Work w = {0, 0, 0};
    if (is_wide(a, rows) != WIDE || rows <= 0 || n.len <= 0) return w;
    const int tile = WIDE ? kWideTile : narrow_tile(a);
    w.tiles = (rows + tile - 1) / tile;
    const int keys = WIDE ? kPage : unit_keys(a.kv_heads);
    w.units = w.last = (n.len + keys - 1) / keys;
    if (WIDE && rows - (w.tiles - 1) * kWideTile <= kWideHalf) w.last = (w.units + 1) / 2;
    return w;
}

// How the SMs are shared between the two kernels, which run side by side: a start, a plan and an end cost each of them some
// 8 us, and what one leaves of HBM or of the SMs the other uses (one after the other 64 samples of a long prompt took 103
// us, side by side 80, and 83 since the wide kernel waits for a block's values by a barrier of its own).  In proportion to their work, a wide unit taken as kWideCost and a narrow one as kNarrowCost for
// every eight rows of its tile (64 samples: 84, 84, 94 and 107 us at ratios of 5, 6, 4 and 3 to 9; 24 samples in tiles of
// 16 rows: 47 to 53 at 6 to 13 to 9, 62 at 4).  Each has at least one CTA, which leaves the merge's records.
constexpr int kWideCost = 3, kNarrowCost = 2;
__device__ __forceinline__ void make_share(const mono_prefix_attn_args& a, uint32_t* share, uint32_t ctas) {
    __shared__ float s_wide[32], s_narrow[32];
    float wide = 0.f, narrow = 0.f;
    for (int e = threadIdx.x; e < a.groups + a.seqs; e += blockDim.x) {
        const Entry n = entry_of(a, e);
        const Work w = entry_work<true>(a, n), x = entry_work<false>(a, n);
        if (w.tiles) wide += (float)w.per_head();
        if (x.tiles) narrow += (float)x.per_head();
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        wide += __shfl_down_sync(0xffffffffu, wide, o);
        narrow += __shfl_down_sync(0xffffffffu, narrow, o);
    }
    if ((threadIdx.x & 31) == 0) { s_wide[threadIdx.x >> 5] = wide; s_narrow[threadIdx.x >> 5] = narrow; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < (int)blockDim.x / 32; ++w) { wide += s_wide[w]; narrow += s_narrow[w]; }
        wide *= (float)(a.kv_heads * kWideCost);
        narrow *= (float)(head_groups(a.kv_heads) * kNarrowCost * narrow_tile(a) / 8);
        const int n = clamp_int((int)((float)ctas * (wide / fmaxf(wide + narrow, 1.f)) + 0.5f), 1, max((int)ctas - 1, 1));
        share[0] = (uint32_t)n;
        share[1] = max(ctas - (uint32_t)n, 1u);
        share[2] = 0;
    }
}

// Every CTA takes `part_size` units, the last of them what is left: no part in use is empty.
__device__ __forceinline__ uint32_t part_size(uint32_t U, uint32_t ctas) { return max((U + ctas - 1) / ctas, 1u); }

// What the merge has to know of an entry, from the kernel that has the entry.
struct alignas(16) Record {
    int tok0, ntok;
    uint32_t off, item;  // the entry's first unit and item of kv head (narrow: head group) 0
    int tiles, units, last, wide;
};
// Where things lie in the scratch.  CTA c's segment of item i is number c + i: both grow along the list of units, so no
// two segments share a number.  `entry`: per token its group (or what an earlier launch left) and its sequence.
struct Scratch {
    Record* rec;           // [entries]
    uint32_t* total[2];    // units and items of one kv head (narrow: head group), units of a CTA's part and 2^32 over that
    uint32_t* share;       // how many of its CTAs the wide and the narrow kernel use, where both run; whether one took NaN bytes out
    int* entry[2];         // [tokens]
    float* seg[2];
    uint8_t* q_image;      // the wide kernel's queries: [2][kv heads][tokens][q heads per kv head][128], and per row
    float* q_scale;        // what undoes their scale
};

// off[0..E]: units of one kv head (narrow: head group) before entry e (off[E]: all of them); item[0..E]: items likewise.  The
// list of units runs through all entries for kv head 0, then for kv head 1, ...  Called by all threads of a block; the
// blocks together (`ctas` of them) leave the merge's records.
template <bool WIDE, int THREADS>
__device__ __forceinline__ void make_plan(const mono_prefix_attn_args& a, const Scratch& s, uint32_t* off, uint32_t* item, uint32_t* red /* [2 * 32] */, uint32_t ctas) {
    const int E = a.groups + a.seqs, per = (E + THREADS - 1) / THREADS;
    const int e0 = min((int)threadIdx.x * per, E), e1 = min(e0 + per, E);
    uint32_t su = 0, si = 0;
    // With starts that never fall and stay in range no token belongs to two sequences or groups, which is what bounds
    // the number of items (and so the scratch): anything else is refused as a whole.
    int bad = 0;
    for (int e = e0; e < e1; ++e) {
        const int32_t* st = e < a.groups ? a.group_start + e : a.q_start + (e - a.groups);
        bad |= st[0] < 0 || st[1] < st[0] || st[1] > (e < a.groups ? a.seqs : a.tokens);
        const Entry n = entry_of(a, e);
        const Work w = entry_work<WIDE>(a, n);
        off[e] = su;
        item[e] = si;
        if (w.tiles) su += (uint32_t)w.per_head();
        si += (uint32_t)w.tiles;
        if (!WIDE) {  // this block's share of the tokens
            int t = n.tok0 + (int)((blockIdx.x + ctas - (uint32_t)n.tok0 % ctas) % ctas);
            for (; t < n.tok0 + n.ntok; t += ctas) s.entry[e >= a.groups][t] = e;
        }
    }
    // the sums of the threads before this one
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t pu = su, pi = si;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, pu, o), i = __shfl_up_sync(0xffffffffu, pi, o);
        if (lane >= o) { pu += u; pi += i; }
    }
    if (lane == 31) { red[warp] = pu; red[32 + warp] = pi; }
    bad = __syncthreads_or(bad);
    uint32_t bu = 0, bi = 0;
    for (int w = 0; w < warp; ++w) { bu += red[w]; bi += red[32 + w]; }
    bu += pu - su;
    bi += pi - si;
    for (int e = e0; e < e1; ++e) { off[e] += bu; item[e] += bi; }
    if (threadIdx.x == THREADS - 1) {
        off[E] = bad ? 0 : bu + su;  // refused: nobody has work
        item[E] = bi + si;
        if (blockIdx.x == 0) {
            const uint32_t per = part_size(off[E] * (WIDE ? a.kv_heads : head_groups(a.kv_heads)), ctas);
            s.total[WIDE][0] = off[E];
            s.total[WIDE][1] = item[E];
            s.total[WIDE][2] = per;
            s.total[WIDE][3] = per == 1 ? 0xFFFFFFFFu : 0xFFFFFFFFu / per + 1;
            if (bad) guard_fail(a.guard, MONO_ERR_ARG, kSiteTables);
        }
    }
    if (blockIdx.x == 0) {
        for (int e = e0; e < e1; ++e) {
            const Entry n = entry_of(a, e);
            const bool wide = is_wide(a, n.ntok * (a.q_heads / a.kv_heads));
            if (wide != WIDE) continue;
            const Work w = entry_work<WIDE>(a, n);
            s.rec[e] = Record{n.tok0, n.ntok, off[e], item[e], w.tiles, w.units, w.last, wide};
        }
    }
    __syncthreads();
}
// A place in the list: kv head (narrow: head group), entry, unit of the entry.
struct Place {
    int head, e;
    uint32_t local;
};
__device__ __forceinline__ Place place_of(const uint32_t* off, int E, uint32_t u) {
    Place p;
    p.head = (int)(u / off[E]);
    u -= (uint32_t)p.head * off[E];
    int lo = 0, hi = E - 1;  // the last entry that starts at or before u (entries without units share a start with the next)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (off[mid] <= u) lo = mid; else hi = mid - 1;
    }
    p.e = lo;
    p.local = u - off[lo];
    return p;
}
struct alignas(64) Params {
    CUtensorMap kmap, vmap, kmap1, vmap1, qmap;  // boxes of a head group, of one head's page, of 128 query rows
    mono_prefix_attn_args a;
    Scratch s;
    int beside;  // the narrow kernel runs beside the wide one
};

// Makes the query image and runs the wide kernel on `ctas` CTAs (prefix_attn_tc.cu).
cudaError_t launch_wide(const Params& p, int ctas, cudaStream_t st);

}  // namespace prefix_attn
