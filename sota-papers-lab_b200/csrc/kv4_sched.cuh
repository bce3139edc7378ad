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
    if (flag && !ok) atomicOr(a.err + ERR_INDEX_WORD, ERR_INDEX);
    s.tiles = (s.qn * a.group + COLS - 1) / COLS;
    return s;
}

// Keys that query token i of the sequence sees: [lo, hi).  Query i sits at
// position kv - qn + i.
__device__ __forceinline__ int key_hi(const Kv4Attend& a, const Seq& s, int i) {
    return a.causal ? max(0, s.kv - s.qn + i + 1) : s.kv;
}
__device__ __forceinline__ int key_lo(const Kv4Attend& a, const Seq& s, int i) {
    return a.window ? max(0, max(0, s.kv - s.qn + i + 1) - a.window) : 0;
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

// A sequence's units (one KV head); `more`: its tiles, and in the upper half
// the units missing to multiples of LEAST per tile.
template <int COLS, int UNIT, int LEAST>
__device__ __forceinline__ long long seq_units(const Kv4Attend& a, const Seq& s, uint64_t& more) {
    static_assert((LEAST & (LEAST - 1)) == 0, "a power of two");
    long long n = 0;
    more = 0;
    for (int t = 0; t < s.tiles; t++) {
        const int units = keys_of<COLS, UNIT>(a, s, t).units;
        n += units;
        more += 1 + ((uint64_t)(-units & (LEAST - 1)) << 32);
    }
    return n;
}

// All units over `ctas` CTAs.  Where they do not give every CTA `least`, each
// tile is made a multiple of that many, so that no CTA works on two tiles one
// after the other.  Where they do, the first U mod G CTAs have one unit more than
// the others, and a tile counts for `begin` units more, which stand before its
// own: what its rows, first loads and output cost the CTA that starts it (the
// kernels say what either brought).
struct Shares {
    long long U, q, r;  // q = U / G, r = U mod G
    int G;              // CTAs that get work
    int w, pad;         // units that stand before a tile's own; its own are rounded up to a multiple of pad + 1
    Shares() = default;
    __device__ __forceinline__ Shares(long long units, long long missing, long long tiles, int ctas, int least, int begin) {
        const bool few = units + missing <= (long long)least * ctas;
        w = few ? 0 : begin;
        pad = few ? least - 1 : 0;
        U = few ? units + missing : units + w * tiles;
        G = few ? (int)(U / least) : ctas;
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
    __device__ __forceinline__ int of_tile(int units) const { return w + ((units + pad) & ~pad); }
};

// Where a unit lies.
struct Place {
    int b, head, tile;
    long long start;  // the tile's first unit, those before its own among them
    Seq s;
};

// A warp finds CTA `cta`'s share and the tile it begins in (all lanes get it).
// Lane i holds the lengths of sequence 32 k + i, so up to 32 sequences take one
// round of loads.  Returns false where the CTA has no work.
template <int COLS, int UNIT, int LEAST, int BEGIN>
__device__ __forceinline__ bool find_share(const Kv4Attend& a, int cta, int ctas, Shares& sh, Place& p) {
    const int lane = threadIdx.x & 31, hkv = a.pool.kv_heads;
    // sequences b0 + lane, their units, and those up to and with them (one KV head)
    Seq s;
    long long x, incl;
    uint64_t more, more_incl;
    auto scan = [&](int b0) {
        const int b = b0 + lane;
        s = b < a.batch ? seq_at<COLS>(a, b) : Seq{0, 0, 0, 0};
        x = incl = seq_units<COLS, UNIT, LEAST>(a, s, more);
        more_incl = more;
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, incl, i);
            const uint64_t z = __shfl_up_sync(0xffffffffu, more_incl, i);
            if (lane >= i) {
                incl += y;
                more_incl += z;
            }
        }
    };
    long long total = 0, missing = 0, tiles = 0;
    for (int b0 = (a.batch - 1) & ~31; b0 >= 0; b0 -= 32) {  // the first 32 last: they stay
        scan(b0);
        total += __shfl_sync(0xffffffffu, incl, 31);
        const uint64_t m = __shfl_sync(0xffffffffu, more_incl, 31);
        tiles += (uint32_t)m;
        missing += m >> 32;
    }
    sh = Shares(total * hkv, missing * hkv, tiles * hkv, ctas, LEAST, BEGIN);
    if (cta >= sh.G) return false;
    const long long u = sh.first(cta);
    long long base = 0;
    for (int b0 = 0;; b0 += 32) {
        if (b0) scan(b0);
        x += sh.pad ? (long long)(more >> 32) : (long long)sh.w * (uint32_t)more;
        incl += sh.pad ? (long long)(more_incl >> 32) : (long long)sh.w * (uint32_t)more_incl;
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
        const int n = sh.of_tile(keys_of<COLS, UNIT>(a, p.s, p.tile).units);
        if (u < p.start + n) break;
        p.start += n;
    }
    return true;
}

// The part of a tile that a CTA works on: its units unit0 .. unit1 - 1.
struct Piece {
    Place at;
    KeyRange kr;
    int unit0, unit1;
    bool any;  // there is such a piece
};

template <int COLS, int UNIT>
__device__ __forceinline__ void cut_piece(const Kv4Attend& a, const Shares& sh, long long from, Piece& p) {
    p.kr = keys_of<COLS, UNIT>(a, p.at.s, p.at.tile);
    const long long own = p.at.start + sh.w;
    p.unit0 = (int)max(0ll, from - own);
    p.unit1 = (int)min((long long)p.kr.units, sh.first(blockIdx.x + 1) - own);
    p.any = p.unit0 < p.unit1;  // (not where the share ends before the tile's own units)
}

// The CTAs that have a piece's tile between them.
__device__ __forceinline__ int first_holder(const Shares& sh, const Piece& p) {
    return p.unit0 ? sh.holder(p.at.start + sh.w) : blockIdx.x;
}
__device__ __forceinline__ int last_holder(const Shares& sh, const Piece& p) {
    return p.unit1 < p.kr.units ? sh.holder(p.at.start + sh.w + p.kr.units - 1) : blockIdx.x;
}

// The piece after p in the CTA's share.
template <int COLS, int UNIT>
__device__ __forceinline__ void next_piece(const Kv4Attend& a, const Shares& sh, const Piece& p, Piece& n) {
    const long long end = p.at.start + sh.of_tile(p.kr.units);
    n.any = end + sh.w < sh.first(blockIdx.x + 1);
    if (!n.any) return;
    n.at = p.at;
    n.at.start = end;
    if (++n.at.tile >= n.at.s.tiles) {
        n.at.tile = 0;
        if (++n.at.head >= a.pool.kv_heads) {
            n.at.head = 0;
            do n.at.s = seq_at<COLS>(a, ++n.at.b);  // (units are left: there is one)
            while (n.at.s.tiles == 0);
        }
    }
    cut_piece<COLS, UNIT>(a, sh, n.at.start, n);
}

// Four channels of row n of the sequence, from sums relative to 2^ref.  A row
// that saw no key (sum 0) is written as zeros, its lse as -infinity.
template <int D>
__device__ __forceinline__ void put_row(const Kv4Attend& a, const Seq& s, int kv_head, int n, int d, float4 v, float ref,
                                        float sum) {
    const int tok = by_group(a, n), head = kv_head * a.group + n - tok * a.group;
    const float inv = 1.f / sum;
    uint2 r = make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
    if (sum == 0.f) r = make_uint2(0u, 0u);
    *(uint2*)((uint16_t*)a.out.data + (s.row0 + tok) * a.out.st + head * a.out.sh + d) = r;
    if (a.lse && d == 0)
        a.lse[(long long)(s.row0 + tok) * a.heads + head] = (ref + log2f(sum)) * 0.6931471805599453f;
}

// Counts a finished piece of p's tile (the CTA's barrier has ordered its writes
// before); true where it was the last of CTAs c0 .. c1.  One thread calls it.
__device__ __forceinline__ bool last_piece(const Kv4Attend& a, int c0, int c1) {
    // releases the whole CTA's writes, acquires the others'
    uint32_t n;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(n) : "l"(a.done + c0) : "memory");
    const bool last = n == (uint32_t)(c1 - c0);
    if (last) a.done[c0] = 0;
    return last;
}

// Joins the pieces that CTAs c0 .. c1 left of a tile's `cols` columns from row
// n0 on; THREADS threads call it and meet at named barrier 1.  D/4 threads hold a column's channels; where columns are few, the
// pieces of one are shared out among several such teams, which meet in `sm`
// (32 lanes' part every WARP bytes) and `sm_ml` [THREADS / (D/4)].  MEANS: the pieces' outputs are divided by their sums.
template <int D, int COLS, int THREADS, int WARP, bool MEANS = false>
__device__ __forceinline__ void join_tile(const Kv4Attend& a, const Seq& s, int head, int n0, int cols, int c0, int c1,
                                          uint8_t* sm, float2* sm_ml) {
    auto sync = [] { named_bar(1, THREADS); };
    constexpr int LANES = D / 4, TEAMS = THREADS / LANES;
    const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
    if (cols > TEAMS) {
        // many columns (a prompt's tile): NC a team at a time, NP pieces of
        // each in one go, whose loads are all under way together
        constexpr int NC = 4, NP = 3;
        for (int first = team; first < cols; first += NC * TEAMS) {
            float m[NC], sum[NC];
            float4 v[NC];
#pragma unroll
            for (int k = 0; k < NC; k++) {
                m[k] = -INFINITY;
                sum[k] = 0.f;
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            for (int b = c0; b <= c1; b += NP) {
                float2 ml[NC][NP];
                float4 y[NC][NP];
#pragma unroll
                for (int k = 0; k < NC; k++)
#pragma unroll
                    for (int i = 0; i < NP; i++) {
                        const int col = first + k * TEAMS, c = b + i;
                        ml[k][i] = make_float2(-INFINITY, 0.f);
                        y[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (c <= c1 && col < cols) {
                            const long long slot = (long long)(2 * c + (c == c0)) * COLS + col;
                            ml[k][i] = __ldcg(&a.part_ml[slot]);
                            y[k][i] = __ldcg((const float4*)(a.part_o + slot * D + 4 * lane));
                        }
                    }
#pragma unroll
                for (int k = 0; k < NC; k++) {
                    const float old = m[k];
#pragma unroll
                    for (int i = 0; i < NP; i++) m[k] = fmaxf(m[k], ml[k][i].x);
                    const float ref = m[k] == -INFINITY ? 0.f : m[k], f0 = ex2(old - ref);
                    sum[k] *= f0;
                    v[k].x *= f0; v[k].y *= f0; v[k].z *= f0; v[k].w *= f0;
#pragma unroll
                    for (int i = 0; i < NP; i++) {
                        float f = ex2(ml[k][i].x - ref);
                        sum[k] = fmaf(f, ml[k][i].y, sum[k]);
                        if (MEANS) f *= ml[k][i].y;
                        v[k].x = fmaf(f, y[k][i].x, v[k].x); v[k].y = fmaf(f, y[k][i].y, v[k].y);
                        v[k].z = fmaf(f, y[k][i].z, v[k].z); v[k].w = fmaf(f, y[k][i].w, v[k].w);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < NC; k++)
                if (first + k * TEAMS < cols)
                    put_row<D>(a, s, head, n0 + first + k * TEAMS, 4 * lane, v[k], m[k] == -INFINITY ? 0.f : m[k], sum[k]);
        }
        sync();
        return;
    }
    int slices = 1;
    while (2 * slices * cols <= TEAMS) slices *= 2;
    const int per = TEAMS / slices, slice = team / per;  // columns at a time
    auto sm_v = [&](int t) { return (float4*)(sm + t * LANES / 32 * WARP) + t * LANES % 32 + lane; };
    for (int first = 0; first < cols; first += per) {
        const int col = first + team % per;
        float m = -INFINITY, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        // a few pieces at a time, all of their loads under way before the first is used
        constexpr int AHEAD = 8;
        for (int b = c0 + slice; b <= c1; b += slices * AHEAD) {
            float2 ml[AHEAD];
            float4 y[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int c = b + i * slices;
                ml[i] = make_float2(-INFINITY, 0.f);
                y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (c <= c1 && col < cols) {
                    const long long slot = (long long)(2 * c + (c == c0)) * COLS + col;
                    ml[i] = __ldcg(&a.part_ml[slot]);
                    y[i] = __ldcg((const float4*)(a.part_o + slot * D + 4 * lane));
                }
            }
            const float old = m;
#pragma unroll
            for (int i = 0; i < AHEAD; i++) m = fmaxf(m, ml[i].x);
            const float ref = m == -INFINITY ? 0.f : m, f0 = ex2(old - ref);
            sum *= f0;
            v.x *= f0; v.y *= f0; v.z *= f0; v.w *= f0;
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                float f = ex2(ml[i].x - ref);
                sum = fmaf(f, ml[i].y, sum);
                if (MEANS) f *= ml[i].y;
                v.x = fmaf(f, y[i].x, v.x); v.y = fmaf(f, y[i].y, v.y);
                v.z = fmaf(f, y[i].z, v.z); v.w = fmaf(f, y[i].w, v.w);
            }
        }
        *sm_v(team) = v;
        if (lane == 0) sm_ml[team] = make_float2(m, sum);
        sync();
        if (slice == 0 && col < cols) {
            float mm = -INFINITY;
            for (int i = 0; i < slices; i++) mm = fmaxf(mm, sm_ml[team + i * per].x);
            const float ref = mm == -INFINITY ? 0.f : mm;
            sum = 0.f;
            v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < slices; i++) {
                const float2 ml = sm_ml[team + i * per];
                const float4 y = *sm_v(team + i * per);
                const float f = ex2(ml.x - ref);
                sum = fmaf(f, ml.y, sum);
                v.x = fmaf(f, y.x, v.x); v.y = fmaf(f, y.y, v.y);
                v.z = fmaf(f, y.z, v.z); v.w = fmaf(f, y.w, v.w);
            }
            put_row<D>(a, s, head, n0 + col, 4 * lane, v, ref, sum);
        }
        sync();
    }
}

}  // namespace sp
