// Attention of few query rows over the paged 4-bit KV cache (a decoding
// step): o = softmax(scale q K^T + mask) V, K and V = zero + scale * n per 64
// channels of a token (kv4.h).
//
// Bound by the cache's bytes (144 per token and KV head at D = 128), if
// unpacking keeps up: 8 values arrive with 4 bytes, so the instructions per
// value decide.  Hence:
//   - the products run on mma.sync m16n8k16 with the CACHE as the A operand
//     (16 keys or 16 channels) and the query rows as the 8 columns: S^T = K q^T
//     and O^T = V^T P^T.  A group of up to 8 query heads fills the 8 columns;
//     with the rows as M = 16 half of every product would be padding.  (These
//     shapes are far too small for tcgen05's M = 128.)
//   - K's n enters as the f16 subnormal whose bits are n: (w & 0x000f000f) is
//     the pair (n0, n4) * 2^-24, (w & 0x00f000f0) the pair (n1, n5) * 2^-20:
//     5 instructions for 8 values, no conversion.  q is scaled per row by a
//     power of two into f16's middle (exact: bf16's 8 bits) and once more by
//     2^-4 where the pair carries 2^-20.  The order of the channels within
//     the sum is free, so q's fragments are loaded in the order of the nibbles.
//   - K's scale and zero are per key and group of 64 channels: each group's
//     sum is kept apart and S = s0 a0 + s1 a1 + (z0 Q0 + z1 Q1), Q the row's
//     channel sums.  So S is that of the exact cached values, to f32.
//   - V's n enters the same way.  Its scale goes into the probability, in f16:
//     p * s * 2^(14 - R) is rounded once by 2^-11 of itself (2^-25 * 2^-14 of
//     2^R where it is subnormal).  R follows the magnitudes of the scales that
//     the warp meets, within [2^(R - 12), 2^(R + 1)]; the few keys of a step
//     whose scale lies outside while others' do not are added to the sums in
//     f32, one by one, so that no key takes precision from the rows that do
//     not see it.  sum(p z) is kept in f32.
//   - S^T has a key per row, P^T wants the keys along k: movmatrix transposes
//     the 8x8 blocks in registers.
// Each of the 8 warps streams its own 32-key steps through its own ring in
// shared memory (cp.async, 16 bytes, no barrier but the warp's own) with its
// own running maximum and sums; the warps meet once per tile.  Row maxima are
// looked at by vote and only recomputed when one grows.
//
// Measured, 32 / 8 heads, D = 128: one sequence of 131072 tokens (151 MB) 45 us,
// 64 of up to 8192 (371 MB) 94.5 us; another 151 MB add 29 us (5.2 TB/s, where a
// copy reaches 6.45; the issue slots are 3/4 busy).  The rest is a call's start
// (3 us from the lengths to the first loads), the ends of pieces (about 4 us
// each, beside the SM's other CTA) and the join (4 us).  One sequence of 1000
// tokens 8.9 us, all of it such latencies.
#include <algorithm>
#include <atomic>

#include "kv4_sched.cuh"
#include "sage_kernels.h"

namespace sp {

constexpr int AT_WARPS = 8, AT_STEP = 32, AT_UNIT = 128;
// Units a CTA takes at least: all 8 warps get a step (one sequence of 200 tokens
// 6.2 us, with one unit 8.2, of 1000 8.9 and 8.6, of 3000 9.2 and 10.8).  Where no
// CTA gets more, none gets parts of two tiles (6000 tokens: 11.6 us instead of
// 16.8, 9000: 12.6 and 18.8).
constexpr int AT_LEAST = 2;
// Units that a tile's start and end count for beside its own (two CTAs on an SM
// and one), times before the scales were checked: 64 sequences of up to 8192 tokens, 32 / 8 heads, D = 128, take 93 us
// instead of 102 with none (93.8 with 6, 97.6 with 11), 16 of up to 4096, 16 / 16
// heads, D = 64, 21.8 instead of 28.9; 20 rows in two tiles 40.4 instead of 42
// (41.2 with 4 and 8).
constexpr int AT_BEGIN_1 = 4, AT_BEGIN_2 = 6;

template <int D, int NT>
struct AttnCfg {
    static constexpr int NG = D / KV4_GROUP;
    static constexpr int ROW = D / 2;                      // bytes of a token's values
    static constexpr int VAL = AT_STEP * ROW;              // of a step
    static constexpr int PAR = AT_STEP * NG * 4;
    static constexpr int STAGE = 2 * VAL + 2 * PAR;        // D = 128: 4608, D = 64: 2304
    static constexpr int STAGES = D == 128 ? 3 : 4;
    static constexpr int COLS = 8 * NT;
    // A warp's memory: its ring, and its output at a tile's end.  The output
    // takes the ring's last stage where it fits (the next tile's first steps
    // are loaded into the others meanwhile).
    static constexpr bool OVER = STAGE >= COLS * D * 4;
    static constexpr int OUT = OVER ? STAGE * (STAGES - 1) : STAGE * STAGES;
    static constexpr int WARP = OVER ? STAGE * STAGES : STAGE * STAGES + COLS * D * 4;
    static constexpr int SMEM = AT_WARPS * WARP;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 .. 127
// The same from zero.
__device__ __forceinline__ void mma_f16_0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
    const uint32_t n = real ? 16 : 0;  // 0: zeros are written, src is not read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t lds32(uint32_t p) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(p));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t p) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p));
    return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// Halves of 16 bits: maxima, sums without a carry between them.
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
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Where a token's row and its 16-byte pieces lie in a stage, so that the
// fragments' loads (8 keys in the order 0 4 1 5 2 6 3 7 for K, four keys in a
// row for V) touch every bank once: D = 128 (64-byte rows) swaps the halves
// of some rows, D = 64 (32-byte rows) swaps rows.
template <int D>
__device__ __forceinline__ int stage_at(int key, int byte) {
    if constexpr (D == 128)
        return key * 64 + (byte ^ ((((key >> 1) ^ (key >> 2)) & 1) << 5));
    else
        return (key ^ (((key >> 2) & 1) << 1)) * 32 + byte;
}

// One lane's part of the copy of a 32-key step: `id0`, `id1` the pages of its
// two halves of 16 keys (-1: none, zeros), key0 the step's first key.  Every
// source is a base of the half plus a constant.
template <int D, int NT>
__device__ __forceinline__ void load_step(const Kv4Attend& a, uint32_t stage, const uint8_t* head, int key0, int id0,
                                          int id1) {
    using C = AttnCfg<D, NT>;
    constexpr int PIECES = C::VAL / 16 / 32;  // of K values a lane copies: 4 or 2, half of them in each half
    constexpr int PP = C::PAR / 16;           // parameter pieces of K: 16 or 8
    const int lane = threadIdx.x & 31, P = a.pool.page_tokens;
    const int in0 = key0 & (P - 1), in1 = (key0 + 16) & (P - 1);
    const uint8_t* b0 = head + (uint64_t)(uint32_t)max(id0, 0) * (uint64_t)a.pool.page_stride;
    const uint8_t* b1 = head + (uint64_t)(uint32_t)max(id1, 0) * (uint64_t)a.pool.page_stride;
    const int half = P * C::ROW;
    const uint32_t dst = stage + stage_at<D>(lane / (C::ROW / 16), lane % (C::ROW / 16) * 16);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint8_t* k = (h ? b1 : b0) + (h ? in1 : in0) * C::ROW + lane * 16;
        const uint8_t* v = k + half;
        const bool real = (h ? id1 : id0) >= 0;
#pragma unroll
        for (int r = 0; r < PIECES / 2; r++) {
            cp_async16(dst + h * (C::VAL / 2) + r * 512, k + r * 512, real);
            cp_async16(dst + C::VAL + h * (C::VAL / 2) + r * 512, v + r * 512, real);
        }
    }
    if (lane < 2 * PP) {
        const bool second = (lane % PP) >= PP / 2;
        const uint8_t* src = (second ? b1 : b0) + 2 * half + (lane >= PP ? P * C::NG * 4 : 0) +
                             (second ? in1 : in0) * (C::NG * 4) + lane % (PP / 2) * 16;
        cp_async16(stage + 2 * C::VAL + lane * 16, src, (second ? id1 : id0) >= 0);
    }
}

// V's scales in f16: R with 2^(R - 12) <= |s| < 2^(R + 1) for those that are held (as bf16 bits less `low`, at
// most V_SPAN; bits of another sign or of NaN are not).
constexpr uint32_t V_SPAN = (13u << 7) * 0x10001u, V_UNSET = 0x80008000u;
// |s|, 0 where it is not finite (such a key comes out as NaN in the rows that see it whatever R is).
__device__ __forceinline__ float scale_size(float s) { return fabsf(s) < INFINITY ? fabsf(s) : 0.f; }
__device__ __forceinline__ int scale_R(float top) { return max((int)(__float_as_uint(top) >> 23) - 126, -100); }  // top < 2^R
__device__ __forceinline__ int up_R(float v_up) { return 14 + 127 - (int)(__float_as_uint(v_up) >> 23); }         // 2^(14 - R)
__device__ __forceinline__ bool scale_fits(float size, int R) {
    return size == 0.f || (size >= exp2i(R - 12) && size <= exp2i(min(R + 1, 127)));
}
template <int NG>
__device__ __forceinline__ void set_low(uint32_t& v_low, int gr, int R) {
    const uint32_t low = 0x10000u - (uint32_t)((R - 12 + 127) << 7), in_gr = NG == 1 ? 0xffffffffu : 0xffffu << 16 * gr;
    v_low = (v_low & ~in_gr) | (low * 0x10001u & in_gr);
}

// A step with scales of V that f16 does not hold together with the others: R
// moves where none of the step's fits any more, the sums are scaled to it, and
// the keys that still do not fit are added to the sums one by one in f32 and
// their scales zeroed.  All 32 lanes call it with what they hold of the step;
// a function of its own, since the registers of the kernel's loop are full.
template <int NT, int NG>
struct FarScales {
    float o[NT][NG][4][4], vs[2][2][NG], p[2][2][NT][2], v_up[NG];
    uint32_t v_low;
};
template <int D, int NT>
__device__ __noinline__ void far_scales(FarScales<NT, D / KV4_GROUP>& k, uint32_t v_stage) {
    constexpr int NG = D / KV4_GROUP, MT = 4;
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll 1
    for (int gr = 0; gr < NG; gr++) {
        int R = up_R(k.v_up[gr]);
        float top = 0.f;
        bool any = false;
        for (int hr = 0; hr < 4; hr++) {
            const float y = scale_size(k.vs[hr >> 1][hr & 1][gr]);
            top = fmaxf(top, y);
            any = any || (y > 0.f && scale_fits(y, R));
        }
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
        if (top == 0.f) continue;
        int to = R;
        if (!__any_sync(0xffffffffu, any)) {
            const int Rt = scale_R(top);
            if (Rt > R) {
                if (Rt <= R + 60) to = Rt;  // (more would leave nothing of the sums so far)
            } else {
                // down, as far as the sums so far stay within f32
                float big = 0.f;
                for (int nt = 0; nt < NT; nt++)
                    for (int i = 0; i < 4 * MT; i++) big = fmaxf(big, fabsf(k.o[nt][gr][i / 4][i % 4]));
                big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
                to = max(Rt, R - min(max(120 + 127 - (int)(__float_as_uint(big) >> 23), 0), 120));
            }
        }
        to = max(to, scale_R(top) - 110);  // (the largest scale times 2^(14 - R) stays within f32)
        const float f = exp2i(max(R - to, -126)), up = exp2i(14 - to);
        R = to;
        k.v_up[gr] = up;
        set_low<NG>(k.v_low, gr, R);
        for (int nt = 0; nt < NT; nt++)
            for (int i = 0; i < 4 * MT; i++) k.o[nt][gr][i / 4][i % 4] *= f;
#pragma unroll 1
        for (int hr = 0; hr < 4; hr++) {
            const int h = hr >> 1, r = hr & 1;
            const float scaled = k.vs[h][r][gr] * up * 0x1p-24f;
            const bool out = !scale_fits(scale_size(k.vs[h][r][gr]), R);
            if (out) k.vs[h][r][gr] = 0.f;
            unsigned left = __ballot_sync(0xffffffffu, out && c == 0);
#pragma unroll 1
            while (left) {
                const int src = __ffs(left) - 1, gk = src >> 2;
                left &= left - 1;
                const float sk = __shfl_sync(0xffffffffu, scaled, src);
                const uint32_t w = lds32(v_stage + stage_at<D>(16 * h + 8 * r + (gk >> 1) + 4 * (gk & 1), gr * 32 + g * 4));
                for (int nt = 0; nt < NT; nt++)
                    for (int j = 0; j < 2; j++) {
                        const float p = __shfl_sync(0xffffffffu, k.p[h][r][nt][j], src + c), ps = p == 0.f ? 0.f : p * sk;
                        for (int t = 0; t < MT; t++) {
                            k.o[nt][gr][t][j] = fmaf(ps, (float)(w >> 8 * t & 15), k.o[nt][gr][t][j]);
                            k.o[nt][gr][t][2 + j] = fmaf(ps, (float)(w >> (8 * t + 4) & 15) * 16.f, k.o[nt][gr][t][2 + j]);
                        }
                    }
            }
        }
    }
}

template <int D, int NT>
__global__ void __launch_bounds__(AT_WARPS * 32, NT == 1 ? 2 : 1) sp_kv4_attend(const __grid_constant__ Kv4Attend a) {
    using C = AttnCfg<D, NT>;
    constexpr int NG = C::NG, COLS = C::COLS, MT = 4;  // MT: tiles of 16 channels of a group
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float sm_m[AT_WARPS][COLS], sm_l[AT_WARPS][COLS];
    __shared__ uint16_t sm_q[NT * NG * 4 * 32 * 4];     // q fragments [nt][group][j][lane][4]
    __shared__ float sm_cf[COLS], sm_qs[NG][COLS];
    __shared__ bool sm_last;
    __shared__ float2 sm_join[AT_WARPS * 2];
    __shared__ Shares sh;
    // The piece at work, the next and (a slow warp may still look at it) the
    // last: what changes between them stays out of registers.
    __shared__ Piece pieces[3];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * C::WARP;
    float* const sm_o = (float*)(smem + warp * C::WARP + C::OUT);

    // The lane's places in a stage.  K: key (g >> 1) + 4 (g & 1) (+ 8 and + 16
    // keep the swizzle), group gr; V: key c + 4 i, where an odd i or, at D =
    // 128, the second group is the other half of the row (D = 64: two rows on).
    uint32_t k_off[NG], v_off[2];
#pragma unroll
    for (int gr = 0; gr < NG; gr++) k_off[gr] = stage_at<D>((g >> 1) + 4 * (g & 1), gr * 32 + c * 8);
    v_off[0] = C::VAL + stage_at<D>(c, g * 4);
    v_off[1] = C::VAL + stage_at<D>(c + 4, g * 4) - 4 * C::ROW;
    const uint32_t p_off = 2 * C::VAL + ((g >> 1) + 4 * (g & 1)) * (NG * 4);
    const uint32_t v_own = C::PAR + 8 * c * (NG * 4);  // from there: V's parameters of the one of the lane's four keys that it checks

    griddep_wait();
    griddep_launch_dependents();
    if (blockIdx.x == 0)  // what is out of range is reported once
        for (int b = threadIdx.x; b < a.batch; b += blockDim.x) seq_at<COLS>(a, b, true);
    if (warp == 0) {
        Shares share;
        Piece p;
        p.any = find_share<COLS, AT_UNIT, AT_LEAST, NT == 1 ? AT_BEGIN_1 : AT_BEGIN_2>(a, blockIdx.x, gridDim.x, share,
                                                                                     p.at);
        if (p.any) cut_piece<COLS, AT_UNIT>(a, share, share.first(blockIdx.x), p);
        if (lane == 0) {
            sh = share;
            pieces[0] = p;
        }
    }
    __syncthreads();
    if (!pieces[0].any) return;

    // A piece's keys [k0, k1): the warps take its 32-key steps in turn.
    auto first_key = [&](const Piece& p) { return p.kr.lo + p.unit0 * AT_UNIT; };
    auto end_key = [&](const Piece& p) { return min(p.kr.hi, p.kr.lo + p.unit1 * AT_UNIT); };
    auto steps_of = [&](int k0, int k1) {
        return max(0, (k1 - k0 + AT_STEP - 1) / AT_STEP - warp + AT_WARPS - 1) / AT_WARPS;
    };
    // The page ids of 16 of the warp's steps from step0 on, one lane per 16
    // keys; -1 where no key is wanted.
    auto fetch_ids = [&](const Piece& p, int step0) {
        const int key = first_key(p) + ((step0 + (lane >> 1)) * AT_WARPS + warp) * AT_STEP + 16 * (lane & 1);
        int id = -1;
        if (key < end_key(p) && key + 16 > p.kr.first) {
            id = a.pages[(long long)p.at.b * a.max_pages + (key >> a.pool.page_shift)];
            if (id < 0 || id >= a.pool.pages) {
                atomicOr(a.err + ERR_INDEX_WORD, ERR_INDEX);
                id = -1;
            }
        }
        return id;
    };
    int cur_ids = fetch_ids(pieces[0], 0), next_ids = -1;
    int fill, stage;  // the ring's stage to fill next, and to use next
    auto issue = [&](const Piece& p, int i, int steps) {
        if (i < steps) {
            if (i && (i & 15) == 0) {
                cur_ids = next_ids;
                next_ids = i + 16 < steps ? fetch_ids(p, i + 16) : -1;
            }
            const int id0 = __shfl_sync(0xffffffffu, cur_ids, 2 * (i & 15));
            const int id1 = __shfl_sync(0xffffffffu, cur_ids, 2 * (i & 15) + 1);
            load_step<D, NT>(a, ring + fill * C::STAGE, a.pool.data + (long long)p.at.head * a.pool.block,
                             first_key(p) + (i * AT_WARPS + warp) * AT_STEP, id0, id1);
        }
        fill = fill + 1 == C::STAGES ? 0 : fill + 1;
        cp_commit();
    };
    // The lane's channels of the query rows that the warp prepares.
    uint2 q_raw[NT];
    auto load_q = [&](const Piece& p) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int n = p.at.tile * COLS + 8 * nt + warp;
            q_raw[nt] = make_uint2(0u, 0u);
            if (n < p.at.s.qn * a.group && lane < D / 4) {
                const int tok = by_group(a, n);
                q_raw[nt] = *(const uint2*)((const uint16_t*)a.q.data + (p.at.s.row0 + tok) * a.q.st +
                                            (p.at.head * a.group + n - tok * a.group) * a.q.sh + 4 * lane);
            }
        }
    };
    auto begin = [&](const Piece& p) {
        const int steps = steps_of(first_key(p), end_key(p));
        fill = stage = 0;
        next_ids = steps > 16 ? fetch_ids(p, 16) : -1;
#pragma unroll
        for (int i = 0; i < C::STAGES - 1; i++) issue(p, i, steps);
        load_q(p);
    };
    begin(pieces[0]);

    for (int turn = 0;; turn = turn == 2 ? 0 : turn + 1) {
        const Piece& p = pieces[turn];
        Piece& next = pieces[turn == 2 ? 0 : turn + 1];
        const Seq s = p.at.s;
        const int k0 = first_key(p), k1 = end_key(p), steps = steps_of(k0, k1);
        const int n0 = p.at.tile * COLS, rows = s.qn * a.group;
        if (threadIdx.x == blockDim.x - 1) next_piece<COLS, AT_UNIT>(a, sh, p, next);

        // ---- the query rows as B fragments, column by column: channel 16c +
        // 4i + j of a group is half-word i of lane c's fragment j, the order
        // of K's nibbles.  A warp makes columns `warp` and, with NT = 2, 8 on.
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int col = 8 * nt + warp;
            const uint2 w = q_raw[nt];
            float x[4] = {bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y)};
            const float lane_max = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
            const float amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(lane_max)));
            // 2^k brings the row's largest magnitude to [2^13, 2^14)
            const int e = (int)(__float_as_uint(amax) >> 23) - 127;
            const int k = min(max(13 - e, -100), 100);
            float sum = 0.f;
            if (lane < D / 4) {
                uint16_t* dst = sm_q + (((nt * NG + lane / 16) * 4) * 32 + warp * 4 + lane % 16 / 4) * 4 + lane % 4;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[j] *= exp2i(k);
                    sum += x[j];
                    const __half f = __float2half_rn(x[j] * ((j & 1) ? 0x1p-4f : 1.f));
                    dst[j * 128] = __half_as_ushort(f);
                }
            }
#pragma unroll
            for (int i = 1; i < 16; i <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
            if (lane % 16 == 0 && lane < D / 4) sm_qs[lane / 16][col] = sum * 0x1p-24f;
            if (lane == 0) sm_cf[col] = a.c * exp2i(24 - k);
        }
        __syncthreads();
        const int first_ids = next.any ? fetch_ids(next, 0) : -1;
        uint32_t qf[NT][NG][4][2];
        float cf[NT][2], qs[NT][NG][2];
        int hi[NT][2], lo[NT][2];
        int min_hi = 0x7fffffff, max_lo = 0;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int gr = 0; gr < NG; gr++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint2 w = ((const uint2*)sm_q)[((nt * NG + gr) * 4 + j) * 32 + lane];
                    qf[nt][gr][j][0] = w.x;
                    qf[nt][gr][j][1] = w.y;
                }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int col = 8 * nt + 2 * c + j, tok = by_group(a, min(n0 + col, rows - 1));
                cf[nt][j] = sm_cf[col];
#pragma unroll
                for (int gr = 0; gr < NG; gr++) qs[nt][gr][j] = sm_qs[gr][col];
                hi[nt][j] = key_hi(a, s, tok);
                lo[nt][j] = key_lo(a, s, tok);
                min_hi = min(min_hi, hi[nt][j]);
                max_lo = max(max_lo, lo[nt][j]);
            }
        }
        min_hi = __reduce_min_sync(0xffffffffu, min_hi);
        max_lo = __reduce_max_sync(0xffffffffu, max_lo);
        const int all_hi = min(min_hi, k1);

        float m[NT][2], l[NT][2], zs[NT][NG][2], o[NT][NG][MT][4];
        // Per group: 2^(14 - R), and (group 0 in the low half) less the smallest scale that f16 holds with it, as bf16
        // bits; no scale fits before the first is met.
        float v_up[NG];
        uint32_t v_low = V_UNSET;
#pragma unroll
        for (int gr = 0; gr < NG; gr++) v_up[gr] = 1.f;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                m[nt][j] = -INFINITY;
                l[nt][j] = 0.f;
#pragma unroll
                for (int gr = 0; gr < NG; gr++) zs[nt][gr][j] = 0.f;
            }
#pragma unroll
            for (int gr = 0; gr < NG; gr++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int t = 0; t < MT; t++) o[nt][gr][t][i] = 0.f;
        }

        // ---- the warp's steps
        for (int i = 0; i < steps; i++) {
            cp_wait<C::STAGES - 2>();
            __syncwarp();
            issue(p, i + C::STAGES - 1, steps);
            const uint32_t st = ring + stage * C::STAGE;
            uint32_t k_at[NG], v_at[2];
#pragma unroll
            for (int gr = 0; gr < NG; gr++) k_at[gr] = st + k_off[gr];
            v_at[0] = st + v_off[0];
            v_at[1] = st + v_off[1];
            const uint32_t p_at = st + p_off;
            stage = stage + 1 == C::STAGES ? 0 : stage + 1;
            const int key0 = k0 + (i * AT_WARPS + warp) * AT_STEP;
            const bool edge = key0 + AT_STEP > all_hi || key0 < max_lo;
            // whether a scale of V leaves f16's reach: a lane looks at one key's, all of its groups at once
            uint32_t scales;
            if constexpr (NG == 2) {
                const uint2 t = lds64(p_at + v_own);
                scales = __byte_perm(t.x, t.y, 0x5410);
            } else {
                scales = lds32(p_at + v_own) & 0xffffu;
                scales |= scales << 16;
            }
            const bool far = scales != 0 && umax2(uadd2(scales, v_low), V_SPAN) != V_SPAN;
            float x[2][NT][4];  // [16 keys][columns][C fragment]: S, then P
            float vs[2][2][NG], vz[2][2][NG];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                // S^T rows g and g + 8 of this half: keys kl and kl + 8
                const int kl = 16 * h + (g >> 1) + 4 * (g & 1);
                float acc[NG][NT][4];
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    const uint2 wl = lds64(k_at[gr] + h * (C::VAL / 2));
                    const uint2 wh = lds64(k_at[gr] + h * (C::VAL / 2) + C::VAL / 4);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int sh = j >= 2 ? 8 : 0;
                        const uint32_t mask = (j & 1) ? 0x00f000f0u : 0x000f000fu;
                        const uint32_t f[4] = {(wl.x >> sh) & mask, (wh.x >> sh) & mask, (wl.y >> sh) & mask,
                                               (wh.y >> sh) & mask};
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
                            if (j == 0)
                                mma_f16_0(acc[gr][nt], f, qf[nt][gr][j][0], qf[nt][gr][j][1]);
                            else
                                mma_f16(acc[gr][nt], f, qf[nt][gr][j][0], qf[nt][gr][j][1]);
                    }
                }
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const uint32_t par = p_at + (16 * h + 8 * r) * (NG * 4);
                    uint32_t kp[NG], vp[NG];
                    if constexpr (NG == 2) {
                        const uint2 t = lds64(par), w = lds64(par + C::PAR);
                        kp[0] = t.x; kp[NG - 1] = t.y; vp[0] = w.x; vp[NG - 1] = w.y;
                    } else {
                        kp[0] = lds32(par);
                        vp[0] = lds32(par + C::PAR);
                    }
#pragma unroll
                    for (int gr = 0; gr < NG; gr++) {
                        vs[h][r][gr] = bf_lo(vp[gr]);
                        vz[h][r][gr] = bf_hi(vp[gr]);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            float t = bf_hi(kp[0]) * qs[nt][0][j];
                            t = fmaf(bf_lo(kp[0]), acc[0][nt][2 * r + j], t);
                            if constexpr (NG == 2) {
                                t = fmaf(bf_hi(kp[NG - 1]), qs[nt][NG - 1][j], t);
                                t = fmaf(bf_lo(kp[NG - 1]), acc[NG - 1][nt][2 * r + j], t);
                            }
                            x[h][nt][2 * r + j] = t;
                        }
                }
                if (edge) {
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const int key = key0 + kl + 8 * r;
                        // Parameters that are not finite (a stored NaN; whatever lies behind the last key) reach
                        // the sums of the columns that see the key, and no others.
                        bool bad[NG];
#pragma unroll
                        for (int gr = 0; gr < NG; gr++) {
                            bad[gr] = !(fabsf(vs[h][r][gr]) + fabsf(vz[h][r][gr]) < INFINITY);
                            if (bad[gr] || key >= k1 || key < p.kr.first) vs[h][r][gr] = vz[h][r][gr] = 0.f;
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                const bool see = key < hi[nt][j] && key < k1 && key >= lo[nt][j];
                                if (!see) x[h][nt][2 * r + j] = -INFINITY;
#pragma unroll
                                for (int gr = 0; gr < NG; gr++)
                                    if (see && bad[gr]) zs[nt][gr][j] = NAN;
                            }
                    }
                }
            }

            // ---- a row's maximum grew somewhere in the warp: take the new
            // ones and scale what is summed
            bool grew = false;
            float mx[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    mx[nt][j] = fmaxf(fmaxf(x[0][nt][j], x[0][nt][2 + j]), fmaxf(x[1][nt][j], x[1][nt][2 + j]));
                    grew = grew || mx[nt][j] > m[nt][j];
                }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float v = fmaxf(mx[nt][j], m[nt][j]);
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                        const float f = v == m[nt][j] ? 1.f : ex2((m[nt][j] - v) * cf[nt][j]);
                        m[nt][j] = v;
                        l[nt][j] *= f;
#pragma unroll
                        for (int gr = 0; gr < NG; gr++) {
                            zs[nt][gr][j] *= f;
#pragma unroll
                            for (int t = 0; t < MT; t++) {
                                o[nt][gr][t][j] *= f;
                                o[nt][gr][t][2 + j] *= f;
                            }
                        }
                    }
            }
            // Probabilities are 2^((x - m) cf), the difference first: x cf - (m cf) as one fused step would leave the
            // rounding of m cf in the exponent, which outgrows f32's range where scores pass 2^30.
            uint64_t less[NT], by[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                less[nt] = pk2(m[nt][0] == -INFINITY ? 0.f : -m[nt][0], m[nt][1] == -INFINITY ? 0.f : -m[nt][1]);
                by[nt] = pk2(cf[nt][0], cf[nt][1]);
            }

            // ---- V's scales within f16's reach
            bool cold = false;
            if (__any_sync(0xffffffffu, far)) {
                // The first ones, or a little more than before: R rises.  (Or only a scale of zero or of another sign,
                // or a key that no row sees.)
                const int own = key0 + 8 * c + (g >> 1) + 4 * (g & 1);
                uint32_t mine = own < k1 && own >= p.kr.first ? scales & 0x7fff7fffu : 0u;
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    if ((mine >> 16 * gr & 0xffffu) >= 0x7f80u) mine &= NG == 1 ? 0u : gr ? 0x0000ffffu : 0xffff0000u;  // not finite
                    const int top = __reduce_max_sync(0xffffffffu, mine >> 16 * gr & 0xffffu);
                    const bool unset = (v_low >> 16 * gr & 0xffffu) == (V_UNSET & 0xffffu);
                    const int R = max((top >> 7) - 126, -100), R0 = up_R(v_up[gr]);
                    if (top == 0 || !(unset || (R > R0 + 1 && R <= R0 + 9))) continue;
                    const float f = unset ? 0.f : exp2i(R0 - R);
                    v_up[gr] = exp2i(14 - R);
                    set_low<NG>(v_low, gr, R);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int t = 0; t < MT; t++)
#pragma unroll
                            for (int i4 = 0; i4 < 4; i4++) o[nt][gr][t][i4] *= f;
                }
                const uint32_t off = umax2(uadd2(mine, v_low), V_SPAN) ^ V_SPAN;
                cold = ((mine & 0xffffu) && (off & 0xffffu)) || ((mine >> 16) && (off >> 16));
                cold = __any_sync(0xffffffffu, cold);
            }
            if (cold) {
                FarScales<NT, NG> k;
                k.v_low = v_low;
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    k.v_up[gr] = v_up[gr];
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int r = 0; r < 2; r++) k.vs[h][r][gr] = vs[h][r][gr];
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            float y[2];
                            upk2(mul2(add2(pk2(x[h][nt][2 * r], x[h][nt][2 * r + 1]), less[nt]), by[nt]), y[0], y[1]);
                            k.p[h][r][nt][0] = ex2(y[0]);
                            k.p[h][r][nt][1] = ex2(y[1]);
                        }
#pragma unroll
                    for (int gr = 0; gr < NG; gr++)
#pragma unroll
                        for (int t = 0; t < MT; t++)
#pragma unroll
                            for (int i4 = 0; i4 < 4; i4++) k.o[nt][gr][t][i4] = o[nt][gr][t][i4];
                }
                far_scales<D, NT>(k, st + C::VAL);
                v_low = k.v_low;
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    v_up[gr] = k.v_up[gr];
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int r = 0; r < 2; r++) vs[h][r][gr] = k.vs[h][r][gr];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int t = 0; t < MT; t++)
#pragma unroll
                            for (int i4 = 0; i4 < 4; i4++) o[nt][gr][t][i4] = k.o[nt][gr][t][i4];
                }
            }

#pragma unroll
            for (int h = 0; h < 2; h++) {
                // P^T fragments per group: k index 2c, 2c+1 are rows 2c, 2c+1
                // of S^T, keys c and c + 4 (and 8 more)
                uint32_t pf[NT][NG][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        float y[2];
                        upk2(mul2(add2(pk2(x[h][nt][2 * r], x[h][nt][2 * r + 1]), less[nt]), by[nt]), y[0], y[1]);
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const float p = ex2(y[j]);
                            x[h][nt][2 * r + j] = p;
                            l[nt][j] += p;
#pragma unroll
                            for (int gr = 0; gr < NG; gr++) zs[nt][gr][j] = fmaf(p, vz[h][r][gr], zs[nt][gr][j]);
                        }
                    }
#pragma unroll
                    for (int gr = 0; gr < NG; gr++)
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            const float sc = vs[h][r][gr] * v_up[gr];
                            pf[nt][gr][r] = transpose8(pack_f16x2(x[h][nt][2 * r] * sc, x[h][nt][2 * r + 1] * sc));
                        }
                }
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    uint32_t w[4];  // 8 channels of keys c, c + 4, c + 8, c + 12
#pragma unroll
                    for (int i4 = 0; i4 < 4; i4++)
                        w[i4] = lds32(v_at[D == 128 ? (gr + i4) & 1 : i4 & 1] + h * (C::VAL / 2) + 4 * i4 * C::ROW);
#pragma unroll
                    for (int t = 0; t < MT; t++) {  // channels 8g + 2t (row g, 2^-24) and 8g + 2t + 1 (row g + 8, 2^-20)
                        const uint32_t sel = t | (t << 4) | ((4 + t) << 8) | ((4 + t) << 12);
                        const uint32_t y0 = __byte_perm(w[0], w[1], sel), y1 = __byte_perm(w[2], w[3], sel);
                        const uint32_t f[4] = {y0 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x000f000fu, y1 & 0x00f000f0u};
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) mma_f16(o[nt][gr][t], f, pf[nt][gr][0], pf[nt][gr][1]);
                    }
                }
            }
        }
        cp_wait<0>();
        __syncwarp();
        if (next.any) {
            cur_ids = first_ids;
            begin(next);
        }

        // ---- the warps' outputs meet: acc * 2^24 / 2^(14 - R) + sum(p z),
        // stored [group][channel within 8][g][column], without bank conflicts
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
                float z[2];
                const float back = 1.f / v_up[gr];  // 2^(R - 14), before the rest, so that nothing passes f32 on the way
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    z[j] = zs[nt][gr][j];
#pragma unroll
                    for (int i = 4; i < 32; i <<= 1) z[j] += __shfl_xor_sync(0xffffffffu, z[j], i);
                }
#pragma unroll
                for (int t = 0; t < MT; t++)
#pragma unroll
                    for (int r = 0; r < 2; r++)
                        *(float2*)(sm_o + ((nt * NG + gr) * 64 + (2 * t + r) * 8 + g) * 8 + 2 * c) =
                            make_float2(fmaf(o[nt][gr][t][2 * r] * back, r ? 0x1p20f : 0x1p24f, z[0]),
                                        fmaf(o[nt][gr][t][2 * r + 1] * back, r ? 0x1p20f : 0x1p24f, z[1]));
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float ls = l[nt][j];
#pragma unroll
                for (int i = 4; i < 32; i <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, i);
                if (g == 0) {
                    sm_m[warp][8 * nt + 2 * c + j] = m[nt][j] == -INFINITY ? -INFINITY : m[nt][j] * cf[nt][j];
                    sm_l[warp][8 * nt + 2 * c + j] = ls;
                }
            }
        }
        __syncthreads();
        const bool whole = p.unit0 == 0 && p.unit1 == p.kr.units;
        const int slot = 2 * (int)blockIdx.x + (p.unit0 ? 0 : 1);
        for (int i = threadIdx.x; i < COLS * D / 4; i += blockDim.x) {
            // column, g, half of the 8 channels, group, nt
            const int half = i >> 6 & 1, part = i >> 7, col = 8 * (part / NG) + (i & 7), n = n0 + col;
            const int d4 = part % NG * KV4_GROUP + 8 * (i >> 3 & 7) + 4 * half;
            if (n >= rows) continue;
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < AT_WARPS; w++) mm = fmaxf(mm, sm_m[w][col]);
            const float ref = mm == -INFINITY ? 0.f : mm;
            float sum = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < AT_WARPS; w++) {
                const float f = ex2(sm_m[w][col] - ref);
                const float* y = (const float*)(smem + w * C::WARP + C::OUT) + part * 512 + half * 256 + (i & 63);
                sum = fmaf(f, sm_l[w][col], sum);
                v.x = fmaf(f, y[0], v.x); v.y = fmaf(f, y[64], v.y);
                v.z = fmaf(f, y[128], v.z); v.w = fmaf(f, y[192], v.w);
            }
            if (whole) {
                put_row<D>(a, s, p.at.head, n, d4, v, ref, sum);
            } else {
                *(float4*)(a.part_o + ((long long)slot * COLS + col) * D + d4) = v;
                if (d4 == 0) a.part_ml[slot * COLS + col] = make_float2(mm, sum);
            }
        }
        __syncthreads();
        if (!whole) {
            // ---- a piece of a split tile: the last to finish joins them
            const int c0 = first_holder(sh, p), c1 = last_holder(sh, p);
            if (threadIdx.x == 0) sm_last = last_piece(a, c0, c1);
            __syncthreads();
            if (sm_last)
                join_tile<D, COLS, AT_WARPS * 32, C::WARP>(a, s, p.at.head, n0, min(COLS, rows - n0), c0, c1, smem + C::OUT, sm_join);
        }
        if (!next.any) return;
    }
}

size_t kv4_scratch_bytes(int d, int sms) {
    return std::max(KV4_COUNTS + (size_t)2 * sms * 16 * (d + 2) * sizeof(float), kv4_prompt_scratch_bytes(d, sms));
}

template <int D, int NT>
static cudaError_t attend(Kv4Attend a, int sms, bool alone, cudaStream_t st) {
    using C = AttnCfg<D, NT>;
    constexpr int COLS = C::COLS;
    // No more CTAs than the longest sequences that max_pages admits can give
    // work: those that have some get an SM to themselves then (one sequence of
    // 200, 1000, 3000 tokens: 6.3, 8.9, 9.3 us instead of 7.1, 10.0, 10.4).
    // The shares are the same.
    // With SMs reserved, no more CTAs than there are others, and with so much
    // shared memory each that two cannot share an SM: CTAs are spread over idle
    // SMs first, so that two for each of them would take the reserved ones as well.
    constexpr int ALONE = std::max(C::SMEM, 116 * 1024);
    const int smem = alone ? ALONE : C::SMEM;
    const int full = (NT == 1 && !alone ? 2 : 1) * sms;
    const double tiles = (double)((a.max_q * a.group + COLS - 1) / COLS) * (a.heads / a.group) * a.batch;
    const long long units = (((long long)a.max_pages << a.pool.page_shift) + 31 + AT_UNIT - 1) / AT_UNIT;
    const int G = (int)std::min<double>(full, tiles * ((units + AT_LEAST - 1) / AT_LEAST));
    if (G * sizeof(uint32_t) > KV4_COUNTS) return cudaErrorInvalidConfiguration;
    a.done = (uint32_t*)a.scratch;
    a.part_ml = (float2*)((uint8_t*)a.scratch + KV4_COUNTS);
    a.part_o = (float*)(a.part_ml + (size_t)2 * G * COLS);
    static std::atomic<uint64_t> ready{0};  // devices whose limit of shared memory is raised, one bit each
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!(ready.load() >> (dev & 63) & 1)) {
        e = cudaFuncSetAttribute(sp_kv4_attend<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, ALONE);
        if (e != cudaSuccess) return e;
        ready.fetch_or(1ull << (dev & 63));
    }
    return launch_after_previous(sp_kv4_attend<D, NT>, dim3(G), dim3(AT_WARPS * 32), smem, st, a);
}

cudaError_t launch_kv4_attend(int d, const Kv4Attend& a, int sms, bool alone, cudaStream_t st) {
    const int rows = a.max_q * a.group;
    // Above 128 rows the tensor-core kernel with a tile of up to 256 rows, up
    // to there this one's tiles of 16 (which read the cache again from the L2).
    // 32 / 8 heads, D = 128, us here and there: 8 sequences, window 8192: 20
    // rows 41 and 110, 64 rows 65 and 114, 128 rows 110 and 119, 160 rows 121
    // and 127, 200 rows 185 and 133, 256 rows 200 and 137; one sequence of 32000
    // tokens: 128 rows 97 and 88.  With little work the border lies higher (one
    // sequence of 2000 tokens: 256 rows 26 and 45, 1024 rows 71 and 50): lengths
    // are not known here, and the rule does not guess them.
    if (rows > 128) return launch_kv4_prompt(d, a, sms, st);
    if (d == 64) return rows <= 8 ? attend<64, 1>(a, sms, alone, st) : attend<64, 2>(a, sms, alone, st);
    return rows <= 8 ? attend<128, 1>(a, sms, alone, st) : attend<128, 2>(a, sms, alone, st);
}

}  // namespace sp
