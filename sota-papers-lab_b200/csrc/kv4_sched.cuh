// How attention over the paged cache is shared out.
//
// A tile is `COLS` consecutive query rows of one (sequence, KV head): row
// n = token * group + query head of the group, counted within the sequence's
// queries.  A tile reads one range of keys, cut into units of UNIT keys.  All
// units of the call, in the order sequence, KV head, tile, unit, are divided
// evenly among the CTAs: CTA i takes units [i U / G, (i + 1) U / G).  So a
// batch of any lengths is balanced, one long sequence is split over the whole
// GPU, and the division follows from the lengths alone (the result does not
// depend on which CTA runs first).  A tile that one CTA holds whole is written
// out by it; the pieces of a split one go to the CTA's two scratch slots
// (slot 1: the tile begins in the CTA, slot 0: it began before) and are joined
// by a second kernel.
//
// Lengths are read from device memory, so every index is checked here: what
// is out of range is clamped and flagged in the error word.
#pragma once

#include "kv4.h"
#include "rotary.cuh"

namespace sp {

struct Seq {
    int row0;    // its first row in q
    int qn;      // its query tokens
    int kv;      // its keys, the queries' own among them
    int tiles;   // of COLS rows
};

struct KeyRange {
    int first;   // the first key any row of the tile sees
    int lo, hi;  // the keys read: [lo, hi), lo = first rounded down to a multiple of 32
    int units;
};

// `flag`: report what is out of range (one caller does, not all).
template <int COLS>
__device__ __forceinline__ Seq seq_at(const Kv4Attend& a, int b, bool flag = false) {
    Seq s;
    bool ok = true;
    if (a.q_start) {
        const int s0 = a.q_start[b], s1 = a.q_start[b + 1];
        s.row0 = min(max(s0, 0), a.tokens);
        const int end = min(max(s1, s.row0), a.tokens);
        s.qn = min(end - s.row0, a.max_q);
        ok = s.row0 == s0 && end == s1 && s.qn == end - s.row0;
    } else {
        s.row0 = b;
        s.qn = 1;
    }
    const int n = a.kv_len[b];
    const long long most = (long long)a.max_pages << a.pool.page_shift;
    s.kv = (int)min((long long)max(n, 0), most);
    ok = ok && s.kv == n;
    if (flag && !ok) atomicOr(a.err, ERR_INDEX);
    s.tiles = (s.qn * a.group + COLS - 1) / COLS;
    return s;
}

// Keys that query token i of the sequence sees: [lo, hi).  Query i sits at
// position kv - qn + i.
__device__ __forceinline__ int key_hi(const Kv4Attend& a, const Seq& s, int i) {
    return a.causal ? max(0, s.kv - s.qn + i + 1) : s.kv;
}
__device__ __forceinline__ int key_lo(const Kv4Attend& a, const Seq& s, int i) {
    return a.window ? max(0, s.kv - s.qn + i + 1 - a.window) : 0;
}

template <int COLS, int UNIT>
__device__ __forceinline__ KeyRange keys_of(const Kv4Attend& a, const Seq& s, int tile) {
    KeyRange r;
    const int first = tile * COLS / a.group, last = min(s.qn - 1, (tile * COLS + COLS - 1) / a.group);
    r.hi = key_hi(a, s, last);
    r.first = min(key_lo(a, s, first), r.hi);
    r.lo = r.first & ~31;
    // a tile without a key still has a unit: its rows are written as zeros
    r.units = max(1, (r.hi - r.lo + UNIT - 1) / UNIT);
    return r;
}

template <int COLS, int UNIT>
__device__ __forceinline__ long long seq_units(const Kv4Attend& a, const Seq& s) {
    long long n = 0;
    for (int t = 0; t < s.tiles; t++) n += keys_of<COLS, UNIT>(a, s, t).units;
    return n;
}

// The CTAs that get work: with fewer units than CTAs one unit each.
__device__ __forceinline__ int shares(long long U, int ctas) { return (int)min(U, (long long)ctas); }
// CTA c of G <= U begins at unit c U / G; the CTA that holds unit u.
__device__ __forceinline__ long long first_unit(long long c, long long U, int G) { return c * U / G; }
__device__ __forceinline__ int cta_of(long long u, long long U, int G) { return (int)(((u + 1) * G - 1) / U); }

// One warp's walk over the sequences: the units of all sequences (one KV
// head), and of those before sequence `upto`.
template <int COLS, int UNIT>
__device__ __forceinline__ void count_units(const Kv4Attend& a, int upto, long long& total, long long& before) {
    const int lane = threadIdx.x & 31;
    long long n = 0, m = 0;
    for (int b = lane; b < a.batch; b += 32) {
        const long long x = seq_units<COLS, UNIT>(a, seq_at<COLS>(a, b));
        n += x;
        if (b < upto) m += x;
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) {
        n += __shfl_xor_sync(0xffffffffu, n, i);
        m += __shfl_xor_sync(0xffffffffu, m, i);
    }
    total = n;
    before = m;
}

// Where unit u lies.
struct Place {
    int b, head, tile;
    long long start;  // the tile's first unit
};

// All lanes of a warp call it with the same u < all units.
template <int COLS, int UNIT>
__device__ __forceinline__ Place find_unit(const Kv4Attend& a, long long u) {
    const int lane = threadIdx.x & 31, hkv = a.pool.kv_heads;
    Place p = {0, 0, 0, 0};
    long long base = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
        const int b = b0 + lane;
        const long long x = b < a.batch ? hkv * seq_units<COLS, UNIT>(a, seq_at<COLS>(a, b)) : 0;
        long long incl = x;
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, incl, i);
            if (lane >= i) incl += y;
        }
        const unsigned over = __ballot_sync(0xffffffffu, base + incl > u);
        if (over) {
            const int w = __ffs(over) - 1;
            p.b = b0 + w;
            const long long per = __shfl_sync(0xffffffffu, x, w) / hkv;
            p.start = base + __shfl_sync(0xffffffffu, incl - x, w);
            p.head = (int)((u - p.start) / per);
            p.start += p.head * per;
            break;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
    const Seq s = seq_at<COLS>(a, p.b);
    for (;; p.tile++) {
        const int n = keys_of<COLS, UNIT>(a, s, p.tile).units;
        if (u < p.start + n || p.tile + 1 >= s.tiles) break;
        p.start += n;
    }
    return p;
}

}  // namespace sp
