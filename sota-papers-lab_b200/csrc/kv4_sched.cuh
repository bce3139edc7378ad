// How attention over the paged cache is shared out.
//
// A tile is `COLS` consecutive query rows of one (sequence, KV head): row
// n = token * group + query head of the group, counted within the sequence's
// queries.  A tile reads one range of keys, cut into units of UNIT keys.  All
// units of the call, in the order sequence, KV head, tile, unit, are divided
// evenly among the CTAs, each taking a run of them.  So a batch of any lengths
// is balanced, one long sequence is split over the whole GPU, and the division
// follows from the lengths alone.  A tile that one CTA holds whole is written
// out by it; the pieces of a split one go to scratch, in one of their CTA's two
// slots (1: the tile begins in the CTA, 0: it began before), and the CTA that
// finishes last joins them, in their order (so the result does not depend on
// which CTA that is).  Its count of finished pieces, under the tile's first
// CTA's number, is zero again when it leaves.
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

// n / group, without a division.
__device__ __forceinline__ int by_group(const Kv4Attend& a, int n) {
    return a.group_mul ? (int)(__umulhi((uint32_t)n, a.group_mul) >> a.group_shift) : n;
}

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
    const int first = by_group(a, tile * COLS), last = min(s.qn - 1, by_group(a, tile * COLS + COLS - 1));
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

// U units over `ctas` CTAs: the first U mod G of the G = min(U, ctas) that get
// work have one unit more than the others.
struct Shares {
    long long U, q, r;  // q = U / G, r = U mod G
    int G;
    Shares() = default;
    __device__ __forceinline__ Shares(long long units, int ctas) {
        U = units;
        G = (int)min(U, (long long)ctas);
        if (U < 1ll << 32) {  // a short division
            q = G ? (uint32_t)U / (uint32_t)G : 0;
        } else {
            q = U / G;
        }
        r = U - q * G;
    }
    __device__ __forceinline__ long long first(int c) const { return c * q + min((long long)c, r); }
    __device__ __forceinline__ int holder(long long u) const {  // the CTA of unit u
        const long long wide = r * (q + 1);
        const long long x = u < wide ? u : u - wide, per = u < wide ? q + 1 : q;
        const int base = u < wide ? 0 : (int)r;
        return base + (x < 1ll << 32 ? (int)((uint32_t)x / (uint32_t)per) : (int)(x / per));
    }
};

// Where a unit lies.
struct Place {
    int b, head, tile;
    long long start;  // the tile's first unit
    Seq s;
};

// A warp finds CTA `cta`'s share and the tile it begins in (all lanes get it).
// Lane i holds the lengths of sequence 32 k + i, so up to 32 sequences take one
// round of loads.  Returns false where the CTA has no work.
template <int COLS, int UNIT>
__device__ __forceinline__ bool find_share(const Kv4Attend& a, int cta, int ctas, Shares& sh, Place& p) {
    const int lane = threadIdx.x & 31, hkv = a.pool.kv_heads;
    // sequences b0 + lane, their units, and the units up to and with them (one KV head)
    Seq s;
    long long x, incl;
    auto scan = [&](int b0) {
        const int b = b0 + lane;
        s = b < a.batch ? seq_at<COLS>(a, b) : Seq{0, 0, 0, 0};
        x = incl = seq_units<COLS, UNIT>(a, s);
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, incl, i);
            if (lane >= i) incl += y;
        }
    };
    long long total = 0;
    for (int b0 = (a.batch - 1) & ~31; b0 >= 0; b0 -= 32) {  // the first 32 last: they stay
        scan(b0);
        total += __shfl_sync(0xffffffffu, incl, 31);
    }
    sh = Shares(total * hkv, ctas);
    if (cta >= sh.G) return false;
    const long long u = sh.first(cta);
    long long base = 0;
    for (int b0 = 0;; b0 += 32) {
        if (b0) scan(b0);
        const unsigned over = __ballot_sync(0xffffffffu, base + incl * hkv > u);
        if (over || b0 + 32 >= a.batch) {
            const int w = over ? __ffs(over) - 1 : 0;  // (u < U: there is one)
            p.b = b0 + w;
            const long long per = __shfl_sync(0xffffffffu, x, w);
            p.start = base + __shfl_sync(0xffffffffu, incl - x, w) * hkv;
            p.s.row0 = __shfl_sync(0xffffffffu, s.row0, w);
            p.s.qn = __shfl_sync(0xffffffffu, s.qn, w);
            p.s.kv = __shfl_sync(0xffffffffu, s.kv, w);
            p.s.tiles = __shfl_sync(0xffffffffu, s.tiles, w);
            const long long off = u - p.start;
            p.head = off < per ? 0 : off < 1ll << 32 ? (int)((uint32_t)off / (uint32_t)per) : (int)(off / per);
            p.start += p.head * per;
            break;
        }
        base += __shfl_sync(0xffffffffu, incl, 31) * hkv;
    }
    for (p.tile = 0; p.tile + 1 < p.s.tiles; p.tile++) {
        const int n = keys_of<COLS, UNIT>(a, p.s, p.tile).units;
        if (u < p.start + n) break;
        p.start += n;
    }
    return true;
}

}  // namespace sp
