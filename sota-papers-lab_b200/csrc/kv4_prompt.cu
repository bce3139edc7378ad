// Attention of many query rows over the paged 4-bit KV cache (pieces of
// prompts, drafted tokens): o = softmax(scale q K^T + mask) V on the 5th
// generation tensor cores, K and V = zero + scale * n per 64 channels of a
// token (kv4.h).
//
// 256 query rows (token * group + head of the group) of one KV head share each
// 128-key tile, so that unpacking a key costs a 256th part of a row.  One CTA
// per SM, five warpgroups that share out its registers (setmaxnreg):
//   warps 0-7   softmax: a thread per row, warps 0-3 the first 128 rows (A),
//               4-7 the others (B), 64 of a row's scores in registers at a
//               time.  While A's scores are worked on, the tensor core
//               computes B's, and the other way round.
//   warps 8-15  unpack the next tile into shared memory
//   warp 17     unpacks a tile whose keys' magnitudes are far apart, in turns
//   warp 16     one thread issues tcgen05.mma: S = Q K^T (f16, both operands
//               from shared memory, S in TMEM) and O += P V (f16, P from
//               TMEM, where it takes the place of its S)
// TMEM holds S of A and B (128 columns each; P, packed, in the first 64) and O
// of both (D columns each).
//
// K: scale * (n - 8) has 8 + 3 significant bits, so it is EXACT in f16 when
// scaled by a power of two 2^-E; the rest of the value, c = zero + 8 scale, is
// constant per group of 64 channels and enters through 16 more channels, as two
// f16 terms times two f16 terms of the row's sum over the group (an error below
// 2^-20 of that product, or 2^-19 of the key's largest value times the sum).  So S
// is that of the exact cached values to about f32's rounding, and lse with it,
// where f16 values of K would put a row's lse off by 1e-4 and more.  Each row of
// Q is scaled by a power of two of its own.
// V: zero + scale * n, scaled by a power of two 2^-R, rounded to f16 (2^-11 of
// itself, or 2^-25 of 2^R where that is more); P, times 2^7 and what R differs
// from the R that the row's O refers to, rounded to f16 likewise; sums in f32.
// (bf16 for both, which needs no R, left the output off by 0.0028 of itself
// against 64 bits instead of 0.0017, and unpacked slower.)
// E and R hold for the keys of a tile that share them: see K_WIDE.
//
// The running maximum a row's exponents refer to is only raised when a new one
// is more than 2^8 larger (P and the sums have room for that), so O is hardly
// ever rescaled.
//
// Measured: 2 x 2048 query tokens on up to 8192 cached ones, 32 / 8 heads, D =
// 128 (382 GFLOP), 569 us, 671 TFLOP/s, 0.41 of a large bf16 product's rate.
// No unit bounds it: without the exponentials it took 519 of then 562 us,
// without the products 520, without the unpacking arithmetic 549; the chain
// from S to the P that waits for it does.
//
// Every wait is bounded (sage_dev.cuh): on a timeout all
// roles leave their loops, the MMAs in flight are waited for, TMEM is freed.
#include <atomic>

#include "kv4_sched.cuh"
#include "sage_kernels.h"

namespace sp {

constexpr int PR_ROWS = 256, PR_KEYS = 128;
constexpr int PR_LEAST = 4;  // key tiles a CTA takes at least: a piece's start, end and joining cost as much as several
constexpr uint32_t R_BELOW = 4;  // how far a tile's R may lie below the one that a row's O refers to: P of 2^-28 is not lost
constexpr int PR_BEGIN = 3;  // what a tile's start and end count for when they are shared out (549 us instead of 575, 551 with 6, then)
constexpr int PR_SOFTMAX = 8, PR_UNPACK = 8, PR_MMA_WARP = 16, PR_HELP_WARP = 17, PR_THREADS = 20 * 32;
// Registers a thread: what the block is launched with, and what the
// warpgroups make of them (raising more than there are would wait for ever).
constexpr int PR_REGS = 96, PR_REGS_SOFTMAX = 128, PR_REGS_UNPACK = 88, PR_REGS_MMA = 48;
static_assert(PR_REGS_SOFTMAX >= PR_REGS && PR_REGS_UNPACK <= PR_REGS && PR_REGS_MMA <= PR_REGS &&
                  2 * PR_REGS_SOFTMAX + 2 * PR_REGS_UNPACK + PR_REGS_MMA <= 5 * PR_REGS && PR_THREADS == 5 * 128,
              "the warpgroups share what the block has");

template <int D>
struct PromptCfg {
    static constexpr int NG = D / KV4_GROUP;
    static constexpr int ATOM = 128 * 128;             // 128 rows of 64 16-bit elements, 128-byte swizzle
    static constexpr int Q = NG * ATOM;                // of 128 rows
    static constexpr int K = NG * ATOM;                // of 128 keys
    static constexpr int V = 2 * D * 128;              // V^T: two atoms of D rows and 64 keys
    static constexpr int X = 128 * 32;                 // 16 more channels, 32-byte swizzle
    static constexpr int Q_OFF = 0;
    static constexpr int K_OFF = Q_OFF + 2 * Q;
    static constexpr int V_OFF = K_OFF + 2 * K;
    static constexpr int QX_OFF = V_OFF + 2 * V;
    static constexpr int KX_OFF = QX_OFF + 2 * X;
    static constexpr int N_OFF = KX_OFF + 2 * X;       // u8 [4][2 groups][16]: keys whose V is not finite, a bit each
    static constexpr int END = N_OFF + 4 * 2 * 16;
    static constexpr int DYN = END + 1024;             // room to align to 1024
};

struct PromptBars {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], f_full[4], s_full[2], p_full[2][2], h_full[2], o_full[2], drained;
};

// The MMA and its commit, issued by the one lane for which `lead` is set.  The
// whole warp comes here together, so that the operands are uniform values (a
// branch around them would make each a vector register that is moved over one
// by one, which held the tensor core back by more than half).
__device__ __forceinline__ void umma_ss(uint32_t lead, uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc), "r"(lead));
}
// ... with A in TMEM
__device__ __forceinline__ void umma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc,
                                        uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b_desc), "r"(idesc), "r"(acc), "r"(lead));
}
__device__ __forceinline__ void commit_if(uint32_t lead, uint32_t bar) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar),
        "r"(lead)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 .. 127
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ void sts128(uint32_t p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void sts16(uint32_t p, uint32_t v) {
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(p), "h"((uint16_t)v) : "memory");
}
// Plain loads, not read-only ones (ld.global.nc): the kernel may start while
// the append before it still writes the pool.  As statements that depend on
// their address alone, they can be moved between others as those can be (as C++
// loads they stay behind every barrier: 611 us instead of 583); none can come
// before griddep_wait, since all addresses follow from what is read after it.
__device__ __forceinline__ uint32_t ld_pool(const uint32_t* p) {
    uint32_t v;
    asm("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ int ld_pool(const int* p) { return (int)ld_pool((const uint32_t*)p); }
__device__ __forceinline__ uint4 ld_pool(const uint4* p) {
    uint4 v;
    asm("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Element-wise maxima and sums of two 16-bit halves.
__device__ __forceinline__ uint32_t umax2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t uadd2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// A named barrier that says whether any of its warps came with `x` (a vote of each first: faster than that of all
// threads, 143 -> 136 us for 8 sequences with a window of 8192 and 256 rows).
__device__ __forceinline__ bool named_bar_any(uint32_t id, uint32_t count, bool x) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 q, %3, 0;\n bar.red.or.pred p, %1, %2, q;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(r)
        : "r"(id), "r"(count), "r"((uint32_t)__any_sync(0xffffffffu, x))
        : "memory");
    return r != 0;
}
__device__ __forceinline__ int bexpo(uint32_t bf16_bits) { return (int)(bf16_bits >> 7 & 255) - 127; }
// x as two f16 terms, (hi, lo) in one word
__device__ __forceinline__ uint32_t split_half(float x) {
    const __half hi = __float2half_rn(x);
    return half2_bits(__half2float(hi), x - __half2float(hi));
}

// A turn of a tile: what its K and V were scaled by (2^-E, 2^-R), whether
// another turn of the same tile follows, and whether its keys have been counted
// in the rows' sums by an earlier one.
struct __align__(16) PromptTile {
    int E, R;
    uint32_t more, again;
};

// E and R stay the same from tile to tile as long as all keys' scales fit them:
// K's from 2^-K_WIDE of the largest that f16 holds with E on (its products are
// exact then: 8 bits of scale, 3 of n - 8 above f16's 2^-24), V's from
// 2^-V_WIDE (its values are off by 2^-12 of the largest that the smallest such
// scale can give; with 2^-10 instead, values at that end left the output off by
// 0.0019 of itself instead of 0.0017).  Any other tile goes to the helper, which
// finds E and R for it; where its keys are too far apart for one pair, or their V
// is not finite, it works on the tile in turns, each with the keys whose
// magnitudes go together and all others hidden, so that no key takes precision
// from the rows that do not see it.
constexpr int K_WIDE = 8, V_WIDE = 8;
// E and R for a scale and zero (bf16 bits, zero in the upper half).  K: scales
// below 2^-8, c below 2^6; V: scales below 2^-8, zeros below 2^13.
__device__ __forceinline__ int key_E(uint32_t k) { return min(max(max(bexpo(k) + 9, bexpo(k >> 16) - 4), -100), 136); }
__device__ __forceinline__ int key_R(uint32_t v) { return min(max(max(bexpo(v) + 9, bexpo(v >> 16) - 12), -100), 136); }
__device__ __forceinline__ bool finite2(uint32_t p) { return (p & 0x7f80u) != 0x7f80u && (p & 0x7f800000u) != 0x7f800000u; }
// Where the scales and zeros that fit lie, as bf16 bits: with x added to them
// (half by half), at most y.
__device__ __forceinline__ uint2 fitting(int most_scale, int least_scale, int most_zero) {
    auto bits = [](int e) { return (uint32_t)min(max(e + 127, 1), 255) << 7; };  // of 2^e
    const uint32_t low = bits(least_scale);
    return make_uint2(0x10000u - low, (min(bits(most_zero + 1) - 1, 0x7f7fu) << 16) | (min(bits(most_scale + 1) - 1, 0x7f7fu) - low));
}

// What the unpacking warps and the helper share.
struct FarTile {
    uint4 fit;  // what fits E and R: K's x and y, V's
    int E, R;
    uint32_t kp[2][PR_KEYS], vp[2][PR_KEYS];  // the tile's keys' parameters by group (0: not wanted)
    uint32_t keys[4], values[2][4];           // the turn's keys, a bit each; those of them with V, by group
    int tile0, end;                           // its first key; that behind its last
    uint32_t t, marks;                        // the next turn; K's stages that hold marks of hidden keys, a bit each
    int piece;                                // -1: no more tiles
    bool done, ok;                            // the helper did all of the tile; no wait ran out
};

// Picks the keys of a tile's turn `pass` (a warp calls it): of those that no
// earlier turn took, the ones whose own E is within K_WIDE of the largest, and
// of these the ones with a group of V whose own R is within V_WIDE of the
// largest (so at least one each time), with those groups.  Once all keys have
// had a turn, the same for the groups that are left of them.  A K or V of zero,
// and one that is not finite, fits any.  Returns whether the tile takes more
// than plain unpacking.
__device__ __forceinline__ bool pick_keys(PromptTile& tile, FarTile& far, int groups, int pass) {
    const int lane = threadIdx.x & 31;
    constexpr int ANY = -1000;
    int E[4], R[4][2];
    bool bad = false;
#pragma unroll
    for (int b = 0; b < 4; b++) {
        E[b] = R[b][0] = R[b][1] = ANY;
#pragma unroll
        for (int gr = 0; gr < 2; gr++) {
            if (gr >= groups) break;
            const uint32_t k = far.kp[gr][32 * b + lane] & 0x7fff7fffu, v = far.vp[gr][32 * b + lane] & 0x7fff7fffu;
            if (k && finite2(k)) E[b] = max(E[b], key_E(k));
            if (v && finite2(v)) R[b][gr] = key_R(v);
            bad = bad || !finite2(v);
        }
    }
    // Of the lane's four keys, a bit each: those without a turn so far, those with group 0 or 1 of V left, and the turn's
    uint32_t fresh = 15, left[2] = {15, groups == 2 ? 15u : 0u}, now = 0, with[2] = {0, 0};
    int top_E = 0, top_R = 0;
    bool first = true;
#pragma unroll 1
    for (int i = 0; i <= pass; i++) {
        fresh &= ~now;
        left[0] &= ~with[0];
        left[1] &= ~with[1];
        first = __any_sync(0xffffffffu, fresh);
        const uint32_t open = first ? fresh : left[0] | left[1];
        uint32_t near = 0;
        int top = ANY;
#pragma unroll
        for (int b = 0; b < 4; b++) top = max(top, open >> b & 1 ? E[b] : ANY);
        top_E = __reduce_max_sync(0xffffffffu, top);
        if (top_E == ANY) top_E = far.E;
        if (far.E > top_E && far.E <= top_E + 2) top_E = far.E;  // (no need to go up and down)
        top = ANY;
#pragma unroll
        for (int b = 0; b < 4; b++)
            if ((open >> b & 1) && (E[b] == ANY || E[b] >= top_E - K_WIDE)) {
                near |= 1u << b;
#pragma unroll
                for (int gr = 0; gr < 2; gr++)
                    if (left[gr] >> b & 1) top = max(top, R[b][gr]);
            }
        top_R = __reduce_max_sync(0xffffffffu, top);
        if (top_R == ANY) top_R = far.R;
        if (far.R > top_R && far.R <= top_R + 2) top_R = far.R;
#pragma unroll
        for (int gr = 0; gr < 2; gr++) {
            with[gr] = 0;
#pragma unroll
            for (int b = 0; b < 4; b++)
                if ((near & left[gr]) >> b & 1 && (R[b][gr] == ANY || R[b][gr] >= top_R - V_WIDE)) with[gr] |= 1u << b;
        }
        now = with[0] | with[1];
    }
    const uint32_t behind = (fresh & ~now) | (left[0] & ~with[0]) | (left[1] & ~with[1]);
    const bool more = __any_sync(0xffffffffu, behind);
#pragma unroll
    for (int b = 0; b < 4; b++) {
        const uint32_t word = __ballot_sync(0xffffffffu, now >> b & 1), v0 = __ballot_sync(0xffffffffu, with[0] >> b & 1),
                       v1 = __ballot_sync(0xffffffffu, with[1] >> b & 1);
        if (lane == 0) {
            far.keys[b] = word;
            far.values[0][b] = v0;
            far.values[1][b] = v1;
        }
    }
    if (lane == 0) {
        tile.E = top_E;
        tile.R = top_R;
        tile.more = more;
        tile.again = !first;
    }
    return __any_sync(0xffffffffu, bad || behind || now != 15);
}

// K's values of one key and group, scaled by 2^-E: scale * (n - 8) in f16.
struct K4 {
    uint32_t sl, sh, off;
    __device__ __forceinline__ K4(uint32_t kp, int E) {
        const float s24 = __uint_as_float(kp << 16) * exp2i(24 - E), m8 = s24 * -0x1p-21f;
        sl = half2_bits(s24, s24);
        sh = half2_bits(s24 * 0x1p-4f, s24 * 0x1p-4f);
        off = half2_bits(m8, m8);
    }
    __device__ __forceinline__ void put(uint32_t dst, uint32_t lo) const {  // 8 channels
        const uint32_t hi = lo >> 8;
        sts128(dst, hfma2(lo & 0x000f000fu, sl, off), hfma2(lo & 0x00f000f0u, sh, off), hfma2(hi & 0x000f000fu, sl, off),
               hfma2(hi & 0x00f000f0u, sh, off));
    }
    // c = zero + 8 scale as two terms
    static __device__ __forceinline__ uint32_t extra(uint32_t kp, int E) {
        return split_half(fmaf(8.f, __uint_as_float(kp << 16), __uint_as_float(kp & 0xffff0000u)) * exp2i(24 - E) * 0x1p-16f);
    }
};
// A key's 16 more channels: (hi, hi, lo, lo) of each group, against the row's (hi, lo, hi, lo)
template <int D>
__device__ __forceinline__ void put_extra(uint32_t base, uint32_t st, int kk, const uint32_t (&cw)[2]) {
    using C = PromptCfg<D>;
    sts128(base + C::KX_OFF + st * C::X + kk * 32 + ((kk >> 2 & 1) << 4), __byte_perm(cw[0], 0, 0x1010),
           __byte_perm(cw[0], 0, 0x3232), __byte_perm(cw[1], 0, 0x1010), __byte_perm(cw[1], 0, 0x3232));
}
// A thread's part of K's stage: half of a key's channels (D = 128: a group), and the 16 more.
template <int D>
__device__ __forceinline__ void put_k(uint32_t base, uint32_t st, int kk, int kh, const uint32_t (&kw)[D / 16],
                                      const uint32_t (&kp)[D / KV4_GROUP], int E) {
    using C = PromptCfg<D>;
    constexpr int NG = C::NG, KW = D / 16;
    const K4 k(kh == 0 ? kp[0] : kp[NG - 1], E);
    const uint32_t dst = base + C::K_OFF + st * C::K + (NG == 2 ? kh * C::ATOM : 0) + kk * 128 + ((kk & 7) << 4);
#pragma unroll
    for (int i = 0; i < KW; i++) k.put(dst ^ ((NG == 2 ? i : kh * KW + i) << 4), kw[i]);
    if (kh == 0) {
        uint32_t cw[2] = {0, 0};
#pragma unroll
        for (int gr = 0; gr < NG; gr++) cw[gr] = K4::extra(kp[gr], E);
        put_extra<D>(base, st, kk, cw);
    }
}

// ... and of V's: 8 channels of 8 keys (finite ones), scaled by 2^-R.
template <int D>
__device__ __forceinline__ void put_v(uint32_t base, uint8_t* sm, uint32_t st, uint32_t t, int vk, int vc,
                                      const uint32_t (&vw)[8], const uint32_t (&vp)[8], int R) {
    using C = PromptCfg<D>;
    const float up = exp2i(24 - R);
    uint32_t sl[4], sh_[4], ze[4];  // of two keys: scale * 2^24 and 2^20, zero, times 2^-R
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t p0 = vp[2 * i], p1 = vp[2 * i + 1];
        const float s0 = __uint_as_float(p0 << 16) * up, s1 = __uint_as_float(p1 << 16) * up;
        sl[i] = half2_bits(s0, s1);
        sh_[i] = half2_bits(s0 * 0x1p-4f, s1 * 0x1p-4f);
        ze[i] = half2_bits(__uint_as_float(p0 & 0xffff0000u) * up * 0x1p-24f, __uint_as_float(p1 & 0xffff0000u) * up * 0x1p-24f);
    }
    if ((vc & 7) == 0) sm[C::N_OFF + (t & 3) * 32 + vc / 8 * 16 + vk] = 0;
    const uint32_t dst = base + C::V_OFF + st * C::V + (vk >> 3) * (D * 128) + vc * 1024 + ((vk & 7) << 4);
#pragma unroll
    for (int b = 0; b < 4; b++) {
        const uint32_t sel = b | (b << 4) | ((4 + b) << 8) | ((4 + b) << 12);
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t y = __byte_perm(vw[2 * i], vw[2 * i + 1], sel);
            lo[i] = hfma2(y & 0x000f000fu, sl[i], ze[i]);
            hi[i] = hfma2(y & 0x00f000f0u, sh_[i], ze[i]);
        }
        const int r0 = 2 * b, r1 = 2 * b + 1;  // channels 8 vc + r
        sts128((dst ^ (r0 << 4)) + r0 * 128, lo[0], lo[1], lo[2], lo[3]);
        sts128((dst ^ (r1 << 4)) + r1 * 128, hi[0], hi[1], hi[2], hi[3]);
    }
}

// The largest magnitude of a row of O.
template <int D>
__device__ __forceinline__ float most_of(uint32_t tm_o) {
    float most = 0.f;
#pragma unroll 1
    for (int ch = 0; ch < D / 32; ch++) {
        uint32_t y[32];
        tmem_ld32(tm_o + 32 * ch, y);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i++) most = fmaxf(most, fabsf(__uint_as_float(y[i])));
    }
    return most;
}

template <int D>
__global__ void __launch_bounds__(PR_THREADS, 1) sp_kv4_prompt(const __grid_constant__ Kv4Attend a) {
    using C = PromptCfg<D>;
    constexpr int NG = C::NG, RING = 8;
    constexpr uint32_t IDESC_S = make_idesc(C_F32, 0, 0, 128, 128);  // f16
    constexpr uint32_t IDESC_O = make_idesc(C_F32, 0, 0, 128, D);
    constexpr uint32_t SWZ_32B = 6;
    extern __shared__ uint8_t dyn_smem[];
    __shared__ PromptBars bars;
    __shared__ uint32_t tmem_base_s;
    __shared__ Shares sh;
    // Pieces, made one ahead by the unpacking warps, which are at most two
    // key tiles (so two pieces) ahead of the softmax.
    __shared__ Piece pieces[RING];
    __shared__ int8_t sm_up[PR_ROWS];  // the power of two that each row of Q was scaled by
    __shared__ PromptTile sm_tile[4];
    __shared__ FarTile sm_far;
    __shared__ uint32_t sm_t;  // turns that A has worked on
    __shared__ float2 sm_join[PR_SOFTMAX * 32 / (D / 4)];
    __shared__ bool sm_last;
    __shared__ volatile uint32_t sm_gave_up;  // a wait of this CTA ran out
    // Whether to go on, as one warp of each group decides it ahead of a barrier
    // of the group (each reading sm_gave_up for itself, they could part and
    // wait for one another for good): A, B, unpacking, all of the softmax.
    __shared__ volatile uint32_t sm_go[4][2];
    const uint32_t base = (smem_u32(dyn_smem) + 1023u) & ~1023u;
    uint8_t* const sm = dyn_smem + (base - smem_u32(dyn_smem));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto bar = [&](uint64_t& b) { return smem_u32(&b); };
    griddep_wait();
    if (blockIdx.x == 0)  // what is out of range is reported once
        for (int b = tid; b < a.batch; b += PR_THREADS) seq_at<PR_ROWS>(a, b, true);
    if (warp == 0) {
        Shares share;
        Piece p;
        p.any = find_share<PR_ROWS, PR_KEYS, PR_LEAST, PR_BEGIN>(a, blockIdx.x, gridDim.x, share, p.at);
        if (p.any) cut_piece<PR_ROWS, PR_KEYS>(a, share, share.first(blockIdx.x), p);
        if (lane == 0) {
            sh = share;
            pieces[0] = p;
        }
    } else if (warp == 1 && lane == 0) {
        mbar_init(bar(bars.q_full), PR_SOFTMAX);
        for (int i = 0; i < 2; i++) {
            mbar_init(bar(bars.k_full[i]), PR_UNPACK);
            mbar_init(bar(bars.k_empty[i]), 1);
            mbar_init(bar(bars.v_full[i]), PR_UNPACK);
            mbar_init(bar(bars.v_empty[i]), 1);
            mbar_init(bar(bars.s_full[i]), 1);
            mbar_init(bar(bars.p_full[i][0]), 4);
            mbar_init(bar(bars.p_full[i][1]), 4);
            mbar_init(bar(bars.h_full[i]), 1);
            mbar_init(bar(bars.o_full[i]), 1);
        }
        for (int i = 0; i < 4; i++) mbar_init(bar(bars.f_full[i]), PR_UNPACK);
        mbar_init(bar(bars.drained), 1);
        fence_barrier_init();
    }
    if (tid == 64) {
        sm_gave_up = 0;
        // (a first guess, for K and V of about one: scales up to 2^2 and 1)
        const uint2 k = fitting(1, 1 - K_WIDE, 14), v = fitting(-1, -1 - V_WIDE, 20);
        sm_far.fit = make_uint4(k.x, k.y, v.x, v.y);
        sm_far.E = 10;
        sm_far.R = 8;
    }
    // the second half of the extra channels' rows: Q's first is 1 (against K's, which hides a key with -infinity there),
    // the rest zero
    for (int i = tid; i < 4 * 128; i += PR_THREADS) {
        const int row = i & 127;
        *(uint4*)(sm + C::QX_OFF + (i >> 7) * C::X + row * 32 + ((1 ^ (row >> 2 & 1)) << 4)) = make_uint4(i < 256 ? 0x3c00u : 0u, 0, 0, 0);
    }
    __syncthreads();
    if (!pieces[0].any) return;
    if (warp == PR_MMA_WARP) {
        tmem_alloc(smem_u32(&tmem_base_s), 512);
        tmem_relinquish();
    }
    // (not before TMEM is taken: a kernel that starts early may take it for itself and wait for this one)
    griddep_launch_dependents();
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;

    bool ok = true;
    if (warp < PR_SOFTMAX) {
        // ======== softmax
        regs_up<PR_REGS_SOFTMAX>();
        const int x = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // TMEM lane base in the address
        const uint32_t tm_s = tmem + 128 * x + lanes, tm_o = tmem + 256 + D * x + lanes;
        // Turns of key tiles so far, those that A (B) worked on, pieces it worked on
        uint32_t t = 0, tx = 0, rounds = 0, events = 0;
        for (int turn = 0;; turn++) {
            const Piece& p = pieces[turn % RING];
            const Seq s = p.at.s;
            const int k0 = p.kr.lo + p.unit0 * PR_KEYS, k1 = min(p.kr.hi, p.kr.lo + p.unit1 * PR_KEYS);
            const int n = p.unit1 - p.unit0, n0 = p.at.tile * PR_ROWS, rows = s.qn * a.group;
            const bool two = n0 + 128 < rows;  // B has rows
            const int nr = n0 + x * 128 + row;
            // ---- the rows of Q, each scaled by the power of two that brings
            // its largest magnitude to [2^13, 2^14) (bf16 values down to 2^-28
            // of it stay exact), channels of each 8 in the order 0 4 1 5 2 6
            // 3 7 (that of K's nibbles)
            {
                // D/8 lanes hold a row's 16-byte pieces: 256/D rows of the warp's 32 at a time
                constexpr int PIECES = D / 8, AT_ONCE = 32 / PIECES, TURNS = 32 / AT_ONCE;
                const int piece = lane % PIECES, gr = piece / 8;
                uint4 w[TURNS];
#pragma unroll
                for (int i = 0; i < TURNS; i++) {
                    const int m = nr - lane + i * AT_ONCE + lane / PIECES, tok = by_group(a, min(m, rows - 1));
                    w[i] = make_uint4(0, 0, 0, 0);
                    if (m < rows)
                        w[i] = *((const uint4*)((const uint16_t*)a.q.data + (s.row0 + tok) * a.q.st +
                                                (p.at.head * a.group + m - tok * a.group) * a.q.sh) + piece);
                }
#pragma unroll
                for (int i = 0; i < TURNS; i += 2) {
                    // the largest magnitudes of two turns' rows, as bf16 bits
                    uint32_t top[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint4 v = w[i + j];
                        top[j] = umax2(umax2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), umax2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
                    }
                    uint32_t both = umax2(__byte_perm(top[0], top[1], 0x5410), __byte_perm(top[0], top[1], 0x7632));
#pragma unroll
                    for (int j = 1; j < PIECES; j <<= 1) both = umax2(both, __shfl_xor_sync(0xffffffffu, both, j));
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int m = (warp & 3) * 32 + (i + j) * AT_ONCE + lane / PIECES;
                        const int k = min(max(13 - bexpo(both >> 16 * j), -100), 100);
                        const float up = exp2i(k);
                        float f[8], sum = 0.f;
                        unpack_bf16x8(w[i + j], f);
#pragma unroll
                        for (int n = 0; n < 8; n++) {
                            f[n] *= up;
                            sum += f[n];
                        }
                        sts128(base + C::Q_OFF + x * C::Q + gr * C::ATOM + m * 128 + (((piece & 7) ^ (m & 7)) << 4),
                               half2_bits(f[0], f[4]), half2_bits(f[1], f[5]), half2_bits(f[2], f[6]), half2_bits(f[3], f[7]));
                        // the sum over the group, (hi, lo, hi, lo)
#pragma unroll
                        for (int n = 1; n < 8; n <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, n);
                        const uint32_t twice = split_half(sum * 0x1p-8f);
                        uint8_t* qx = sm + C::QX_OFF + x * C::X + m * 32 + ((m >> 2 & 1) << 4);
                        if ((piece & 7) == 0) *(uint2*)(qx + gr * 8) = make_uint2(twice, twice);
                        if (NG == 1 && piece == 1) *(uint2*)(qx + 8) = make_uint2(0, 0);
                        if (piece == 0) sm_up[x * 128 + m] = (int8_t)k;
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(bars.q_full));
            }
            const int up_row = sm_up[x * 128 + row];  // (of the warp's own rows)
            if (x == 0 || two) {
                float m_ref = -INFINITY, l = 0.f;  // the row's reference, as q k, and sum
                int R_ref = 0;                     // O holds sum(p v) * 2^(7 - R_ref)
                uint32_t poison = 0;               // groups of V that reach the row as NaN
                const int tok = by_group(a, min(nr, rows - 1));
                const int hi = nr < rows ? min(key_hi(a, s, tok), k1) : k1, lo = nr < rows ? key_lo(a, s, tok) : 0;
                const int all_hi = __reduce_min_sync(0xffffffffu, hi), all_lo = __reduce_max_sync(0xffffffffu, lo);
                const bool live = __any_sync(0xffffffffu, nr < rows);
                const bool leader = (warp & 3) == 0;
                bool all_ok = true;  // of the group's four warps
                // V of the last turn (of tile j) that is not finite reaches the rows that see the key.
                auto see_bad = [&](int j) {
                    const uint4* bad = (const uint4*)(sm + C::N_OFF + ((t - 1) & 3) * 32);
#pragma unroll
                    for (int gr = 0; gr < NG; gr++) {
                        const uint4 b = bad[gr];
                        if ((b.x | b.y | b.z | b.w) == 0) continue;
                        const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll 1
                        for (int i = 0; i < 128; i++) {
                            const uint32_t word = i < 32 ? w[0] : i < 64 ? w[1] : i < 96 ? w[2] : w[3];
                            const int key = k0 + j * PR_KEYS + i;
                            if ((word >> (i & 31) & 1) && key < hi && key >= lo) poison |= 1u << gr;
                        }
                    }
                };
                int last = 0;  // the tile of the turn before
                bool first = true;
                for (int j = 0; j < n;) {
                    const uint32_t tj = t;
                    // One warp of the four waits (each poll costs issue slots), the others at a barrier.
                    if (leader)
                        sm_go[x][events & 1] = warp_all_wait(bar(bars.f_full[tj & 3]), tj >> 2 & 1, a.err, 61) &&
                                               warp_all_wait(bar(bars.s_full[x]), tx & 1, a.err, 60) && !sm_gave_up;
                    named_bar(4 + x, PR_SOFTMAX * 16);
                    all_ok = sm_go[x][events++ & 1];
                    if (!all_ok) break;
                    ok = true;
                    if (!first) see_bad(last);
                    tc_fence_after();
                    const int key0 = k0 + j * PR_KEYS;
                    const PromptTile tile = sm_tile[tj & 3];
                    auto hand_over = [&](int h) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar(bars.p_full[x][h]));
                    };
                    if (live) {
                        const bool edge = key0 + PR_KEYS > all_hi || key0 < all_lo;
                        const int R = tile.R;
                        if (first) R_ref = R + 2;
                        bool far_R = (uint32_t)(R_ref - R) > R_BELOW;
                        // (at most 7, so P at most 2^15; below -40 nothing is left of it in f16)
                        int shift = min(max(7 + R - R_ref, -40), 7);
                        // What S is multiplied by: softmax scale times 2^(E - up), in two steps (either may be far from 1).
                        // (At least 2^-87, where f is at least 2^-120 whatever the scale: S is below 2^27, and what is left
                        // of a score there is nothing.  The reference has to be in the same units.)
                        const int e = max(tile.E - up_row, -87);
                        const float f = fminf(a.c * exp2i(e >> 1) * exp2i(e - (e >> 1)), 3e38f);
                        float m_s = m_ref * exp2i(-e >> 1) * exp2i(-e - (-e >> 1));  // the reference in S's units
#pragma unroll 1
                        for (int h = 0; h < 2; h++) {
                            uint32_t r[2][32];
                            tmem_ld32(tm_s + 64 * h, r[0]);
                            tmem_ld32(tm_s + 64 * h + 32, r[1]);
                            tmem_wait_ld();
                            // ---- the row's maximum
                            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                            if (edge) {
#pragma unroll
                                for (int ch = 0; ch < 2; ch++)
#pragma unroll
                                    for (int i = 0; i < 32; i++) {
                                        const int key = key0 + 64 * h + 32 * ch + i;
                                        if (key >= hi || key < lo) r[ch][i] = 0xff800000u;  // -infinity
                                    }
                            }
#pragma unroll
                            for (int ch = 0; ch < 2; ch++)
#pragma unroll
                                for (int i = 0; i < 32; i += 2)
                                    mx[i / 2 & 3] = max3(mx[i / 2 & 3], __uint_as_float(r[ch][i]), __uint_as_float(r[ch][i + 1]));
                            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                            // ---- a new reference, where the maximum has outgrown the last by 2^8; a new R, where a row that
                            // sees keys with it would leave f16's range or lose them there
                            const bool grew = f * (top - m_s) > 8.f;  // (from -infinity: any)
                            const bool move = far_R && top > -INFINITY;
                            if (__any_sync(0xffffffffu, grew || move)) {
                                float fo = grew ? ex2(f * (m_s - top)) : 1.f;
                                if (grew) {
                                    m_s = top;
                                    m_ref = top * exp2i(e >> 1) * exp2i(e - (e >> 1));
                                }
                                l *= fo;
                                if (!first || h > 0) {
                                    // Before the first half this row's O is complete up to the turn before (S came after
                                    // it); before the second, the first half's product may still be adding to it.
                                    if (h > 0) {
                                        ok = warp_all_wait(bar(bars.h_full[x]), tx & 1, a.err, 72);
                                        tc_fence_after();
                                    }
                                    if (__any_sync(0xffffffffu, move)) {
                                        // down only as far as what the row has summed stays within f32
                                        const float most = most_of<D>(tm_o);
                                        if (move) {
                                            const int room = max(100 + 127 - (int)(__float_as_uint(most) >> 23), 0);
                                            const int to = R > R_ref || most == 0.f ? R + 2 : max(R + 2, R_ref - room);
                                            fo = R_ref - to < -126 ? 0.f : fo * exp2i(min(R_ref - to, 126));
                                            R_ref = to;
                                            far_R = false;
                                            shift = min(max(7 + R - R_ref, -40), 7);
                                        }
                                    }
#pragma unroll 1
                                    for (int ch = 0; ch < D / 32; ch++) {
                                        uint32_t y[32];
                                        tmem_ld32(tm_o + 32 * ch, y);
                                        tmem_wait_ld();
#pragma unroll
                                        for (int i = 0; i < 32; i++) y[i] = __float_as_uint(__uint_as_float(y[i]) * fo);
                                        tmem_st32(tm_o + 32 * ch, y);
                                    }
                                }
                            }
                            // ---- P = 2^((S - ref) f + shift), packed over S.  (The difference first: the rounding of ref f
                            // in the exponent of a fused S f - ref f outgrows f32 where scores pass 2^30.)
                            const float less = m_s == -INFINITY ? 0.f : -m_s, up = (float)shift;
                            const uint64_t less2 = pk2(less, less), f2 = pk2(f, f), up2 = pk2(up, up);
                            uint64_t sum2[2] = {0, 0};
#pragma unroll
                            for (int ch = 0; ch < 2; ch++) {
                                uint32_t q[16];
#pragma unroll
                                for (int i = 0; i < 16; i++) {
                                    float u, v;
                                    upk2(fma2(add2(pk2(__uint_as_float(r[ch][2 * i]), __uint_as_float(r[ch][2 * i + 1])), less2), f2, up2), u, v);
                                    u = ex2(u);
                                    v = ex2(v);
                                    sum2[i & 1] = add2(sum2[i & 1], pk2(u, v));
                                    q[i] = half2_bits(u, v);
                                }
                                tmem_st16(tm_s + 32 * h + 16 * ch, q);
                            }
                            float s0, s1;
                            upk2(add2(sum2[0], sum2[1]), s0, s1);
                            if (!tile.again) l = fmaf(s0 + s1, exp2i(-shift), l);
                            tmem_wait_st();
                            if (h == 0) hand_over(0);
                        }
                    } else {
                        hand_over(0);
                    }
                    // The tile's V is waited for before the last of its P is handed over (afterwards its stage may
                    // already hold the next tile but one): see_bad looks at what came with it.
                    if (leader) ok = warp_all_wait(bar(bars.v_full[tj & 1]), tj >> 1 & 1, a.err, 62) && ok;
                    if (ok)
                        hand_over(1);
                    else
                        sm_gave_up = 1;  // (this warp goes on to the next barrier with the others)
                    t++;
                    tx++;
                    first = false;
                    last = j;
                    if (!tile.more) j++;
                }
                // ---- the rows' outputs
                if (all_ok) {
                    if (leader) sm_go[x][events & 1] = warp_all_wait(bar(bars.o_full[x]), rounds & 1, a.err, 70) && !sm_gave_up;
                    named_bar(4 + x, PR_SOFTMAX * 16);
                    ok = sm_go[x][events++ & 1];
                } else {
                    sm_gave_up = 1;
                }
                if (ok && all_ok) {
                    see_bad(last);
                    tc_fence_after();
                    const bool whole = p.unit0 == 0 && p.unit1 == p.kr.units;
                    const long long part_row = (2ll * blockIdx.x + (p.unit0 ? 0 : 1)) * PR_ROWS + x * 128 + row;
                    const int h = p.at.head * a.group + min(nr, rows - 1) - tok * a.group;
                    // O 2^(R_ref - 7) / l, the power of two in two steps (it may be beyond f32's)
                    const float back0 = (l == 0.f ? 0.f : 1.f / l) * exp2i((R_ref - 7) >> 1) * exp2i(R_ref - 7 - ((R_ref - 7) >> 1));
                    // Through shared memory (the warp's part of Q, which nothing reads any more), so that a store
                    // covers whole rows of 128 bytes: 64 channels in bf16, 32 in f32.
                    const uint32_t stage = base + C::Q_OFF + x * C::Q + (warp & 3) * 4096;
#pragma unroll 1
                    for (int ch = 0; ch < D / 32; ch++) {
                        uint32_t r[32];
                        tmem_ld32(tm_o + 32 * ch, r);
                        tmem_wait_ld();
                        const bool nan = poison >> (32 * ch / KV4_GROUP) & 1;
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            r[i] = __float_as_uint(nan ? NAN : l == 0.f ? 0.f : __uint_as_float(r[i]) * back0);
                        }
                        const float* f = (const float*)r;
                        if (whole) {
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                sts128(stage + lane * 128 + (((ch & 1) * 4 + i) ^ (lane & 7)) * 16,
                                       pack_bf16x2(f[8 * i], f[8 * i + 1]), pack_bf16x2(f[8 * i + 2], f[8 * i + 3]),
                                       pack_bf16x2(f[8 * i + 4], f[8 * i + 5]), pack_bf16x2(f[8 * i + 6], f[8 * i + 7]));
                            if ((ch & 1) == 0) continue;
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; i++)
                                sts128(stage + lane * 128 + (i ^ (lane & 7)) * 16, r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int m = 4 * i + (lane >> 3), mr = nr - lane + m;  // row of the warp, of the sequence
                            const uint4 v = *(const uint4*)(sm + (stage - base) + m * 128 + ((lane & 7) ^ (m & 7)) * 16);
                            if (mr >= rows) continue;
                            if (whole) {
                                const int tm = by_group(a, mr), hm = p.at.head * a.group + mr - tm * a.group;
                                *((uint4*)((uint16_t*)a.out.data + (s.row0 + tm) * a.out.st + hm * a.out.sh +
                                           (ch >> 1) * 64) + (lane & 7)) = v;
                            } else {
                                *((uint4*)(a.part_o + (part_row - lane + m) * D + 32 * ch) + (lane & 7)) = v;
                            }
                        }
                        __syncwarp();
                    }
                    if (nr < rows) {
                        if (!whole)
                            a.part_ml[part_row] = make_float2(a.c * m_ref, l);
                        else if (a.lse)
                            a.lse[(long long)(s.row0 + tok) * a.heads + h] =
                                ((m_ref == -INFINITY ? 0.f : a.c * m_ref) + log2f(l)) * 0.6931471805599453f;
                    }
                    tc_fence_before();
                }
                rounds++;
            }
            // (nobody leaves before all eight warps are here)
            if (!ok) sm_gave_up = 1;
            named_bar(1, PR_SOFTMAX * 32);
            if (warp == 0) {
                sm_go[3][0] = !sm_gave_up;
                sm_t = t;
            }
            named_bar(1, PR_SOFTMAX * 32);
            ok = sm_go[3][0];
            t = sm_t;  // (B may have had no rows)
            if (!ok) break;
            if (p.unit0 != 0 || p.unit1 != p.kr.units) {
                // ---- a piece of a split tile: the last to finish joins them
                const int c0 = first_holder(sh, p), c1 = last_holder(sh, p);
                if (tid == 0) sm_last = last_piece(a, c0, c1);
                named_bar(1, PR_SOFTMAX * 32);
                if (sm_last)
                    join_tile<D, PR_ROWS, PR_SOFTMAX * 32, 512, true>(a, s, p.at.head, n0, min(PR_ROWS, rows - n0), c0, c1, sm,
                                                                sm_join);
            }
            if (!pieces[(turn + 1) % RING].any) break;
        }
    } else if (warp < PR_SOFTMAX + PR_UNPACK) {
        // ======== unpack
        regs_down<PR_REGS_UNPACK>();
        const int w = warp - PR_SOFTMAX, P = a.pool.page_tokens, half = P * (D / 2);
        // K: a thread unpacks half of a key's channels (D = 128: a group).
        // V: 8 channels of 8 keys.
        constexpr int KW = D / 16;  // words of 8 channels
        const int kk = (w & 3) * 32 + lane, kh = w >> 2, vk = (w & 3) * 4 + (lane & 3), vc = (w >> 2) * 8 + (lane >> 2);
        const bool v_on = vc < D / 8;
        const int vg = 8 * vc / KV4_GROUP;
        uint32_t t = 0, events = 0, marks = 0;  // (marks: K's stages that hold such, a bit each)
        for (int turn = 0; ok; turn++) {
            const Piece& p = pieces[turn % RING];
            if (w == 0 && lane == 0) next_piece<PR_ROWS, PR_KEYS>(a, sh, p, pieces[(turn + 1) % RING]);
            const int k0 = p.kr.lo + p.unit0 * PR_KEYS, k1 = min(p.kr.hi, p.kr.lo + p.unit1 * PR_KEYS);
            const int n = p.unit1 - p.unit0, first = p.kr.first;
            const uint8_t* head = a.pool.data + (long long)p.at.head * a.pool.block;
            const int* ids = a.pages + (long long)p.at.b * a.max_pages;
            // What is read of a tile goes three tiles deep: page ids are
            // fetched first, a tile later the parameters that they lead to,
            // another tile later the values, so that no load is waited for.
            // (128 is a multiple of every page size: a thread's place in its
            // pages is the same in all tiles.)
            const int kkey = k0 + kk, vkey = k0 + 8 * vk;  // the thread's keys in tile 0
            const int kat = kkey & (P - 1), vat = vkey & (P - 1);
            auto k_on = [&](int j) { return j < n && kkey + j * PR_KEYS < k1 && kkey + j * PR_KEYS >= first; };
            auto v_mask = [&](int j) {  // of the thread's 8 keys (in one page), those wanted
                const int key = vkey + j * PR_KEYS, lo = max(first - key, 0), hi = min(k1 - key, 8);
                return j < n && v_on && lo < hi ? (0xffu >> (8 - hi)) & (0xffu << lo) : 0u;
            };
            auto k_id = [&](int j) { return k_on(j) ? ld_pool(ids + ((kkey + j * PR_KEYS) >> a.pool.page_shift)) : 0; };
            auto v_id = [&](int j) { return v_mask(j) ? ld_pool(ids + ((vkey + j * PR_KEYS) >> a.pool.page_shift)) : 0; };
            // A page's block of the head; page 0's (never used) where nothing is wanted or the id is bad.
            auto block_of = [&](int& id, bool wanted) {
                const bool good = id >= 0 && id < a.pool.pages;
                if (!good) {
                    if (wanted) atomicOr(a.err + ERR_INDEX_WORD, ERR_INDEX);
                    id = -1;
                }
                return head + (long long)(good ? id : 0) * a.pool.page_stride;
            };
            uint32_t kw[KW], kp[NG], kq[NG], vw[8], vp[8], vq[8];  // values and parameters; q: the next tile's
            uint32_t keep, keep_next;                              // keys that count: bits 0-7 V's, 8 K's
            const uint8_t *kb, *vb;                                // the next tile's blocks
            int kid, vid;
            auto find_blocks = [&](int j) {  // of tile j, from kid and vid
                const bool on = k_on(j);
                const uint32_t m = v_mask(j);
                kb = block_of(kid, on);
                vb = block_of(vid, m != 0);
                keep_next = (kid >= 0 && on ? 256u : 0u) | (vid >= 0 ? m : 0u);
            };
            auto load_params = [&] {
                const uint32_t* kpar = (const uint32_t*)(kb + 2 * half) + kat * NG;
                const uint32_t* vpar = (const uint32_t*)(vb + 2 * half + P * NG * 4) + vat * NG + vg;
#pragma unroll
                for (int i = 0; i < NG; i++) kq[i] = ld_pool(kpar + i);
                if (v_on) {
#pragma unroll
                    for (int i = 0; i < 8; i++) vq[i] = ld_pool(vpar + i * NG);
                }
            };
            auto next_params = [&] {
#pragma unroll
                for (int i = 0; i < NG; i++) kp[i] = kq[i];
#pragma unroll
                for (int i = 0; i < 8; i++) vp[i] = v_on ? vq[i] : 0u;
                keep = keep_next;
            };
            auto load_values = [&](const uint8_t* kb, const uint8_t* vb) {
                const uint4* src = (const uint4*)(kb + kat * (D / 2) + kh * (D / 4));
#pragma unroll
                for (int i = 0; i < KW / 4; i++) {
                    const uint4 y = ld_pool(src + i);
                    kw[4 * i] = y.x; kw[4 * i + 1] = y.y; kw[4 * i + 2] = y.z; kw[4 * i + 3] = y.w;
                }
                if (v_on) {
                    const uint32_t* src = (const uint32_t*)(vb + half + vat * (D / 2)) + vc;
#pragma unroll
                    for (int i = 0; i < 8; i++) vw[i] = ld_pool(src + i * (D / 8));
                }
            };
            kid = k_id(0);
            vid = v_id(0);
            find_blocks(0);
            load_params();
            load_values(kb, vb);
            kid = k_id(1);
            vid = v_id(1);
            next_params();
            find_blocks(1);
            load_params();
            kid = k_id(2);
            vid = v_id(2);
            for (int j = 0; j < n; j++) {
                const uint32_t tj = t, st = tj & 1;
                // ---- whether its scales and zeros fit E and R
                const uint4 fit = sm_far.fit;
                if (keep != 0x1ffu) {  // keys that are not wanted: the smallest that fits
#pragma unroll
                    for (int i = 0; i < NG; i++) kp[i] = keep & 256u ? kp[i] : (0u - fit.x) & 0xffffu;
#pragma unroll
                    for (int i = 0; i < 8; i++) vp[i] = keep >> i & 1 ? vp[i] : (0u - fit.z) & 0xffffu;
                }
                uint32_t kx = 0, vx = 0;
#pragma unroll
                for (int i = 0; i < NG; i++) kx = umax2(kx, uadd2(kp[i] & 0x7fff7fffu, fit.x));
#pragma unroll
                for (int i = 0; i < 8; i++) vx = umax2(vx, uadd2(vp[i] & 0x7fff7fffu, fit.z));
                const bool odd = umax2(kx, fit.y) != fit.y || (v_on && umax2(vx, fit.w) != fit.w) || (marks >> st & 1);
                // one warp waits for K's stage, the others for it
                if (w == 0)
                    sm_go[2][events & 1] =
                        (tj < 2 || warp_all_wait(bar(bars.k_empty[st]), ((tj >> 1) - 1) & 1, a.err, 63)) && !sm_gave_up;
                const bool far = named_bar_any(2, PR_UNPACK * 32, odd);
                ok = sm_go[2][events++ & 1];
                if (!ok) break;
                bool done = false;
                if (far) {
                    if (kh == 0) {
#pragma unroll
                        for (int i = 0; i < NG; i++) sm_far.kp[i][kk] = keep & 256u ? kp[i] : 0u;
                    }
                    if (v_on && (vc & 7) == 0) {
#pragma unroll
                        for (int i = 0; i < 8; i++) sm_far.vp[vg][8 * vk + i] = keep >> i & 1 ? vp[i] : 0u;
                    }
                    if (w == 0 && lane == 0) {
                        sm_far.tile0 = k0 + j * PR_KEYS;
                        sm_far.end = k1;
                        sm_far.t = t;
                        sm_far.piece = turn % RING;
                    }
                    named_bar(3, PR_UNPACK * 32 + 32);
                    named_bar(3, PR_UNPACK * 32 + 32);
                    done = sm_far.done;
                    t = sm_far.t;
                    marks = sm_far.marks;
                    if (!(ok = sm_far.ok)) break;
                    // (the smallest that fitted before may be too large for the new R)
#pragma unroll
                    for (int i = 0; i < NG; i++) kp[i] = keep & 256u ? kp[i] : 0u;
#pragma unroll
                    for (int i = 0; i < 8; i++) vp[i] = keep >> i & 1 ? vp[i] : 0u;
                }
                if (!done) {
                    const int E = sm_far.E;
                    // ---- K
                    put_k<D>(base, st, kk, kh, kw, kp, E);
                    if (w == 0 && lane == 0) *(int4*)&sm_tile[tj & 3] = make_int4(E, sm_far.R, 0, 0);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(bar(bars.k_full[st]));
                        mbar_arrive(bar(bars.f_full[tj & 3]));
                    }
                    // ---- V
                    if (tj >= 2) {
                        if (w == 0)
                            sm_go[2][events & 1] =
                                warp_all_wait(bar(bars.v_empty[st]), ((tj >> 1) - 1) & 1, a.err, 65) && !sm_gave_up;
                        named_bar(2, PR_UNPACK * 32);
                        ok = sm_go[2][events++ & 1];
                        if (!ok) break;
                    }
                    if (v_on) put_v<D>(base, sm, st, tj, vk, vc, vw, vp, sm_far.R);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(bars.v_full[st]));
                    t++;
                }
                // Everything that an earlier load brought is taken first, then all new loads are issued together (a
                // load ahead of such a use was waited for with it).
                next_params();
                const uint8_t *kb_now = kb, *vb_now = vb;
                find_blocks(j + 2);
                load_values(kb_now, vb_now);
                load_params();
                kid = k_id(j + 3);
                vid = v_id(j + 3);
            }
            // the next piece was made by this warpgroup's first thread, and its
            // tiles' barrier 2 has ordered that before
            if (!ok || !pieces[(turn + 1) % RING].any) break;
        }
        if (w == 0 && lane == 0) sm_far.piece = -1;
        named_bar(3, PR_UNPACK * 32 + 32);  // (the helper leaves)
    } else {
        regs_down<PR_REGS_MMA>();
        if (warp == PR_HELP_WARP) {
            // ======== tiles whose keys' magnitudes are too far apart, in as
            // many turns as they need.  The unpacking warps wait meanwhile: what
            // such a tile takes stays out of their loop, whose registers are
            // full.  (Rare, so written for few instructions.)
            uint32_t marks = 0;
            for (;;) {
                named_bar(3, PR_UNPACK * 32 + 32);
                if (sm_far.piece < 0) break;
                const Piece& p = pieces[sm_far.piece];
                const int P = a.pool.page_tokens, half = P * (D / 2), tile0 = sm_far.tile0, end = sm_far.end;
                uint32_t t = sm_far.t;
                bool done = false;
                auto words = [&](int key, int v) -> const uint32_t* {  // a key's values, nullptr where it is not wanted
                    if (key < p.kr.first || key >= end) return nullptr;
                    const int id = a.pages[(long long)p.at.b * a.max_pages + (key >> a.pool.page_shift)];
                    if (id < 0 || id >= a.pool.pages) return nullptr;
                    return (const uint32_t*)(a.pool.data + (long long)p.at.head * a.pool.block + (long long)id * a.pool.page_stride +
                                             v * half + (key & (P - 1)) * (D / 2));
                };
                for (int pass = 0;; pass++) {
                    const uint32_t st = t & 1;
                    if (pass && !(ok = warp_all_wait(bar(bars.k_empty[st]), ((t >> 1) - 1) & 1, a.err, 74) && !sm_gave_up)) break;
                    const bool apart = pick_keys(sm_tile[t & 3], sm_far, NG, pass);
                    __syncwarp();
                    const PromptTile tile = sm_tile[t & 3];
                    if (pass == 0) {
                        done = apart || (marks >> st & 1);
                        if (!done) {  // the unpacking warps go on with these
                            if (lane == 0) {
                                const uint2 k = fitting(tile.E - 9, tile.E - 9 - K_WIDE, tile.E + 4),
                                            v = fitting(tile.R - 9, tile.R - 9 - V_WIDE, tile.R + 12);
                                sm_far.fit = make_uint4(k.x, k.y, v.x, v.y);
                                sm_far.E = tile.E;
                                sm_far.R = tile.R;
                            }
                            break;
                        }
                    }
                    marks &= ~(1u << st);
#pragma unroll 1
                    for (int kk = lane; kk < PR_KEYS; kk += 32) {
                        const bool on = sm_far.keys[kk >> 5] >> lane & 1;
                        const uint32_t* src = on ? words(tile0 + kk, 0) : nullptr;
                        uint32_t cw[2] = {0, 0};
#pragma unroll
                        for (int gr = 0; gr < NG; gr++) {
                            const uint32_t kp = on ? sm_far.kp[gr][kk] : 0u;
                            const K4 k(kp, tile.E);
                            cw[gr] = K4::extra(kp, tile.E);
                            const uint32_t dst = base + C::K_OFF + st * C::K + gr * C::ATOM + kk * 128 + ((kk & 7) << 4);
#pragma unroll 1
                            for (int i = 0; i < 8; i++) k.put(dst ^ (i << 4), src ? src[8 * gr + i] : 0u);
                        }
                        put_extra<D>(base, st, kk, cw);
                        // 1 of every row times -infinity
                        sts128(base + C::KX_OFF + st * C::X + kk * 32 + ((1 ^ (kk >> 2 & 1)) << 4), on ? 0u : 0xfc00u, 0, 0, 0);
                        if (__any_sync(0xffffffffu, !on)) marks |= 1u << st;
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane < PR_UNPACK) {
                        mbar_arrive(bar(bars.k_full[st]));
                        mbar_arrive(bar(bars.f_full[t & 3]));
                    }
                    if (t >= 2 && !(ok = warp_all_wait(bar(bars.v_empty[st]), ((t >> 1) - 1) & 1, a.err, 75) && !sm_gave_up)) break;
#pragma unroll 1
                    for (int kk = lane; kk < PR_KEYS; kk += 32) {
                        const bool on = sm_far.keys[kk >> 5] >> lane & 1;
                        const uint32_t* src = on ? words(tile0 + kk, 1) : nullptr;
                        const uint32_t dst = base + C::V_OFF + st * C::V + (kk >> 6) * (D * 128) + (kk & 7) * 2;
#pragma unroll 1
                        for (int gr = 0; gr < NG; gr++) {
                            uint32_t vp = src && (sm_far.values[gr][kk >> 5] >> lane & 1) ? sm_far.vp[gr][kk] : 0u;
                            const unsigned bad = __ballot_sync(0xffffffffu, !finite2(vp));
                            if (!finite2(vp)) vp = 0;
                            const float up = exp2i(24 - tile.R), s = __uint_as_float(vp << 16) * up,
                                        z = __uint_as_float(vp & 0xffff0000u) * up * 0x1p-24f;
                            const uint32_t sl = half2_bits(s, s), ze = half2_bits(z, z);
#pragma unroll 1
                            for (int i = 0; i < 64; i++) {  // (channel by channel, as the unpacking warps' words are)
                                const uint32_t word = src ? src[8 * gr + (i >> 3)] : 0u;
                                const uint32_t y = hfma2(word >> 4 * (i & 7) & 15u, sl, ze);
                                sts16(dst + (64 * gr + i) * 128 + (((kk >> 3 & 7) ^ (i & 7)) << 4), y);
                            }
                            if ((lane & 7) == 0)
                                sm[C::N_OFF + (t & 3) * 32 + gr * 16 + (kk >> 3)] = (uint8_t)(bad >> lane);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane < PR_UNPACK) mbar_arrive(bar(bars.v_full[st]));
                    t++;
                    if (!tile.more) break;
                }
                if (lane == 0) {
                    sm_far.t = t;
                    sm_far.marks = marks;
                    sm_far.done = done;
                    sm_far.ok = ok;
                }
                named_bar(3, PR_UNPACK * 32 + 32);
            }
        }
        if (warp == PR_MMA_WARP) {
            // ======== the tensor core
            const uint32_t lead = elect_one();
            // (a descriptor's address counts 16 bytes: a step of 16 channels is 2, an atom's 64 are ATOM / 16)
            auto qk = [&](int x, uint32_t st) {
                const uint64_t da = smem_desc(base + C::Q_OFF + x * C::Q, 1024, SWZ_128B);
                const uint64_t db = smem_desc(base + C::K_OFF + st * C::K, 1024, SWZ_128B);
                const uint32_t d = tmem + 128 * x;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    const uint32_t off = (i >> 2) * (C::ATOM / 16) + (i & 3) * 2;
                    umma_ss(lead, d, da + off, db + off, IDESC_S, i > 0);
                }
                umma_ss(lead, d, smem_desc(base + C::QX_OFF + x * C::X, 256, SWZ_32B),
                        smem_desc(base + C::KX_OFF + st * C::X, 256, SWZ_32B), IDESC_S, 1);
                commit_if(lead, bar(bars.s_full[x]));
            };
            auto pv = [&](int x, uint32_t st, int h, bool first) {  // 64 keys
                const uint64_t db = smem_desc(base + C::V_OFF + st * C::V, 1024, SWZ_128B);
                const uint32_t d = tmem + 256 + D * x, p = tmem + 128 * x;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    umma_ts(lead, d, p + 32 * h + 8 * i, db + h * (D * 128 / 16) + i * 2, IDESC_O, !(first && i == 0));
            };
            auto wait = [&](uint64_t& b, uint32_t parity, uint32_t site) { return warp_all_wait(bar(b), parity, a.err, site); };
            uint32_t t = 0, tx[2] = {0, 0};
            for (int turn = 0;; turn++) {
                const Piece& p = pieces[turn % RING];
                const int n = p.unit1 - p.unit0;
                const bool two = p.at.tile * PR_ROWS + 128 < p.at.s.qn * a.group;
                ok = wait(bars.q_full, turn & 1, 66) && wait(bars.k_full[t & 1], t >> 1 & 1, 67);
                if (!ok) break;
                tc_fence_after();
                qk(0, t & 1);
                if (two) qk(1, t & 1);
                commit_if(lead, bar(bars.k_empty[t & 1]));
                bool first = true, last = false;
                for (int j = 0; ok && !last; t++) {
                    const uint32_t st = t & 1, nt = t + 1;
                    const bool more = sm_tile[t & 3].more;  // (came with K)
                    last = !more && j + 1 == n;
                    ok = wait(bars.v_full[st], t >> 1 & 1, 68);
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        if (x == 1 && !two) break;
                        ok = ok && wait(bars.p_full[x][0], tx[x] & 1, 69);
                        if (!ok) break;
                        tc_fence_after();
                        pv(x, st, 0, first);
                        commit_if(lead, bar(bars.h_full[x]));
                        ok = wait(bars.p_full[x][1], tx[x] & 1, 73);
                        if (!ok) break;
                        tx[x]++;
                        tc_fence_after();
                        pv(x, st, 1, false);
                        if (x == (two ? 1 : 0)) commit_if(lead, bar(bars.v_empty[st]));
                        if (!last) {
                            if (x == 0) ok = wait(bars.k_full[nt & 1], nt >> 1 & 1, 67);
                            if (!ok) break;
                            tc_fence_after();
                            qk(x, nt & 1);
                        } else
                            commit_if(lead, bar(bars.o_full[x]));
                    }
                    if (ok && !last) commit_if(lead, bar(bars.k_empty[nt & 1]));
                    first = false;
                    if (!more) j++;
                }
                if (!ok || !pieces[(turn + 1) % RING].any) break;
            }
            // Nothing of the tensor core's may be under way when TMEM is
            // freed: after a timeout it is waited for here.
            if (!ok) {
                commit_if(lead, bar(bars.drained));
                mbar_wait(bar(bars.drained), 0, a.err, 71, false);
            }
        }
    }
    __syncthreads();
    if (warp == PR_MMA_WARP) tmem_dealloc(tmem, 512);
}

size_t kv4_prompt_scratch_bytes(int d, int sms) {
    return KV4_COUNTS + (size_t)2 * sms * PR_ROWS * (d + 2) * sizeof(float);
}

template <int D>
static cudaError_t prompt(Kv4Attend a, int sms, cudaStream_t st) {
    using C = PromptCfg<D>;
    if (sms * sizeof(uint32_t) > KV4_COUNTS) return cudaErrorInvalidConfiguration;
    a.done = (uint32_t*)a.scratch;
    a.part_ml = (float2*)((uint8_t*)a.scratch + KV4_COUNTS);
    a.part_o = (float*)(a.part_ml + (size_t)2 * sms * PR_ROWS);
    static std::atomic<uint64_t> ready{0};  // devices whose limit of shared memory is raised, one bit each
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!(ready.load() >> (dev & 63) & 1)) {
        e = cudaFuncSetAttribute(sp_kv4_prompt<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::DYN);
        if (e != cudaSuccess) return e;
        cudaFuncAttributes at;
        if ((e = cudaFuncGetAttributes(&at, sp_kv4_prompt<D>)) != cudaSuccess) return e;
        if (at.numRegs != PR_REGS) return cudaErrorInvalidDeviceFunction;  // the split above counts on it
        ready.fetch_or(1ull << (dev & 63));
    }
    return launch_after_previous(sp_kv4_prompt<D>, dim3(sms), dim3(PR_THREADS), C::DYN, st, a);
}

cudaError_t launch_kv4_prompt(int d, const Kv4Attend& a, int sms, cudaStream_t st) {
    return d == 64 ? prompt<64>(a, sms, st) : prompt<128>(a, sms, st);
}

}  // namespace sp
