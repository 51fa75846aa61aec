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

// A kernel's view of the work: narrow (16-row tiles, 64-key units) or wide (256-row tiles, 128-key units).
template <bool WIDE>
struct Shape {
    static constexpr int kTile = WIDE ? 256 : 16;
    static constexpr int kKeys = WIDE ? 128 : 64;
    static constexpr int kSegFloats = 2 * kTile + kTile * kDim;  // max, sum, values
};
// rows of an entry from which the wide kernel takes it
constexpr int kWideRows = 48;
// A wide item of at most this many rows is computed twice over alternate units, by the two halves of its CTA: its
// segments then hold two parts per row, at tile rows r and r + 128.
constexpr int kWideHalf = 128;

template <bool WIDE>
__device__ __forceinline__ void entry_work(const mono_prefix_attn_args& a, const Entry& n, int* tiles, int* units) {
    const int rows = n.ntok * (a.q_heads / a.kv_heads);
    const bool mine = (rows >= kWideRows) == WIDE && rows > 0 && n.len > 0;
    *tiles = mine ? (rows + Shape<WIDE>::kTile - 1) / Shape<WIDE>::kTile : 0;
    *units = mine ? (n.len + Shape<WIDE>::kKeys - 1) / Shape<WIDE>::kKeys : 0;
}

// off[0..E]: units before entry e (off[E]: all); item[0..E]: items before entry e.  Called by all threads of a block.
template <bool WIDE, int THREADS>
__device__ __forceinline__ void make_plan(const mono_prefix_attn_args& a, uint32_t* off, uint32_t* item, uint32_t* red /* [2 * 32] */) {
    const int E = a.groups + a.seqs, per = (E + THREADS - 1) / THREADS;
    const int e0 = min((int)threadIdx.x * per, E), e1 = min(e0 + per, E);
    uint32_t su = 0, si = 0;
    // With starts that never fall and stay in range no token belongs to two sequences or groups, which is what bounds
    // the number of items (and so the scratch): anything else is refused as a whole.
    int bad = 0;
    for (int e = e0; e < e1; ++e) {
        const int32_t* st = e < a.groups ? a.group_start + e : a.q_start + (e - a.groups);
        bad |= st[0] < 0 || st[1] < st[0] || st[1] > (e < a.groups ? a.seqs : a.tokens);
        int tiles, units;
        entry_work<WIDE>(a, entry_of(a, e), &tiles, &units);
        off[e] = su;
        item[e] = si;
        su += (uint32_t)tiles * a.kv_heads * units;
        si += (uint32_t)tiles * a.kv_heads;
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
    __syncthreads();
    uint32_t bu = 0, bi = 0;
    for (int w = 0; w < warp; ++w) { bu += red[w]; bi += red[32 + w]; }
    bu += pu - su;
    bi += pi - si;
    for (int e = e0; e < e1; ++e) { off[e] += bu; item[e] += bi; }
    if (threadIdx.x == THREADS - 1) { off[E] = bu + su; item[E] = bi + si; }
    bad = __syncthreads_or(bad);
    if (bad && threadIdx.x == 0) {
        off[E] = 0;  // nobody has work
        if (blockIdx.x == 0) guard_fail(a.guard, MONO_ERR_ARG, kSiteTables);
    }
    __syncthreads();
}
// the entry that holds unit u: the last e with off[e] <= u (entries without units share an offset with the next)
__device__ __forceinline__ int find_entry(const uint32_t* off, int E, uint32_t u) {
    int lo = 0, hi = E - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (off[mid] <= u) lo = mid; else hi = mid - 1;
    }
    return lo;
}
// CTA c of n takes units [cut(c), cut(c + 1)) of U; n is at most U, so nobody's part is empty.
__device__ __forceinline__ uint32_t cut(uint32_t U, uint32_t c, uint32_t n) { return (uint32_t)((uint64_t)U * c / n); }
__device__ __forceinline__ uint32_t owner(uint32_t U, uint32_t u, uint32_t n) { return (uint32_t)((((uint64_t)u + 1) * n - 1) / U); }

// Where things lie in the scratch: per kernel its plan (off, item: E + 1 words each) and its segments.  CTA c's segment
// of item i is number c + i: both grow along the list of units, so no two segments share a number.
struct Scratch {
    uint32_t *off[2], *item[2];
    float* seg[2];
};

struct alignas(64) Params {
    CUtensorMap kmap, vmap;
    mono_prefix_attn_args a;
    Scratch s;
};

// Runs the wide kernel (prefix_attn_tc.cu) on `ctas` CTAs.
cudaError_t launch_wide(const Params& p, int ctas, cudaStream_t st);

}  // namespace prefix_attn
