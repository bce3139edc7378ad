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
//   - V's n sits at mantissa bits 3-6 of a bf16 with exponent 2^4: 16 + n.  V's
//     scale goes into the probability (one bf16 rounding of p * s, 2^-9
//     relative; bf16 has the range of any scale), and o = sum(p s (n - 8)) +
//     sum(p (z + 8 s)): 24 * sum(p s) is taken out of the first sum through
//     one more product with ones (of the same rounded p s), the second is kept
//     in f32.  About n's middle the rounding weighs |n - 8| instead of n: the
//     output's error against 64 bits fell from 0.0038 to 0.0020 (0.0017 is
//     the rounding of the output itself).
//   - S^T has a key per row, P^T wants the keys along k: movmatrix transposes
//     the 8x8 blocks in registers.
// Each of the 8 warps streams its own 32-key steps through its own ring in
// shared memory (cp.async, 16 bytes, no barrier but the warp's own) with its
// own running maximum and sums; the warps meet once per tile.  Row maxima are
// looked at by vote and only recomputed when one grows.
#include "kv4_sched.cuh"
#include "sage_kernels.h"

namespace sp {

constexpr int AT_WARPS = 8, AT_STEP = 32, AT_UNIT = 128;

template <int D, int NT>
struct AttnCfg {
    static constexpr int NG = D / KV4_GROUP;
    static constexpr int ROW = D / 2;                      // bytes of a token's values
    static constexpr int VAL = AT_STEP * ROW;              // of a step
    static constexpr int PAR = AT_STEP * NG * 4;
    static constexpr int STAGE = 2 * VAL + 2 * PAR;        // D = 128: 4608, D = 64: 2304
    static constexpr int STAGES = D == 128 ? 3 : 4;
    static constexpr int COLS = 8 * NT;
    static constexpr int WARP = STAGE * STAGES;            // ring of a warp, and its output at a tile's end
    static_assert(WARP >= COLS * D * 4, "the ring holds a warp's output");
    static constexpr int SMEM = AT_WARPS * WARP;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// two halves of 16 keys (-1: none, zeros), key0 the step's first key.
template <int D, int NT>
__device__ __forceinline__ void load_step(const Kv4Attend& a, uint32_t stage, long long head_off, int key0, int id0,
                                          int id1) {
    using C = AttnCfg<D, NT>;
    const int lane = threadIdx.x & 31, P = a.pool.page_tokens, mask = P - 1;
    const uint8_t* b0 = a.pool.data + (long long)max(id0, 0) * a.pool.page_stride + head_off;
    const uint8_t* b1 = a.pool.data + (long long)max(id1, 0) * a.pool.page_stride + head_off;
    const int half = P * C::ROW;
    constexpr int PIECES = C::VAL / 16 / 32;  // of K values a lane copies: 4 or 2
#pragma unroll
    for (int r = 0; r < PIECES; r++) {
        const int p = lane + 32 * r, key = p / (C::ROW / 16), byte = p % (C::ROW / 16) * 16;
        const bool first = r < PIECES / 2;
        const uint8_t* src = (first ? b0 : b1) + ((key0 + key) & mask) * C::ROW + byte;
        const bool real = (first ? id0 : id1) >= 0;
        const uint32_t dst = stage + stage_at<D>(key, byte);
        cp_async16(dst, src, real);
        cp_async16(dst + C::VAL, src + half, real);
    }
    constexpr int PP = C::PAR / 16;  // parameter pieces of K: 16 or 8
    if (lane < 2 * PP) {
        const int p = lane % PP, key = p * (16 / (C::NG * 4));
        const bool first = p < PP / 2;
        const uint8_t* src = (first ? b0 : b1) + 2 * half + (lane >= PP ? P * C::NG * 4 : 0) +
                             ((key0 + key) & mask) * (C::NG * 4);
        cp_async16(stage + 2 * C::VAL + lane * 16, src, (first ? id0 : id1) >= 0);
    }
}

// Four channels of row n of the sequence, from sums relative to 2^ref.  A row
// that saw no key (sum 0) is written as zeros, its lse as -infinity.
template <int D>
__device__ __forceinline__ void put_row(const Kv4Attend& a, const Seq& s, int kv_head, int n, int d, float4 v, float ref,
                                        float sum) {
    const int tok = n / a.group, head = kv_head * a.group + n - tok * a.group;
    const float inv = 1.f / sum;
    uint2 r = make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
    if (sum == 0.f) r = make_uint2(0u, 0u);
    *(uint2*)((uint16_t*)a.out.data + (s.row0 + tok) * a.out.st + head * a.out.sh + d) = r;
    if (a.lse && d == 0)
        a.lse[(long long)(s.row0 + tok) * a.heads + head] = (ref + log2f(sum)) * 0.6931471805599453f;
}

template <int D, int NT>
__global__ void __launch_bounds__(AT_WARPS * 32, NT == 1 ? 2 : 1) sp_kv4_attend(const __grid_constant__ Kv4Attend a) {
    using C = AttnCfg<D, NT>;
    constexpr int NG = C::NG, COLS = C::COLS, MT = 4;  // MT: tiles of 16 channels of a group
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float sm_m[AT_WARPS][COLS], sm_l[AT_WARPS][COLS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * C::WARP;
    float* const sm_o = (float*)(smem + warp * C::WARP);  // [COLS][D] at a tile's end

    griddep_launch_dependents();
    if (blockIdx.x == 0)  // what is out of range is reported once
        for (int b = threadIdx.x; b < a.batch; b += blockDim.x) seq_at<COLS>(a, b, true);
    long long total, none;
    count_units<COLS, AT_UNIT>(a, 0, total, none);
    total *= a.pool.kv_heads;
    const int G = shares(total, gridDim.x);
    if ((int)blockIdx.x >= G) return;
    long long u = first_unit(blockIdx.x, total, G);
    const long long u_end = first_unit(blockIdx.x + 1, total, G);
    const long long u_begin = u;
    Place at = find_unit<COLS, AT_UNIT>(a, u);

    while (u < u_end) {
        const Seq s = seq_at<COLS>(a, at.b);
        const KeyRange kr = keys_of<COLS, AT_UNIT>(a, s, at.tile);
        const long long tile_end = at.start + kr.units, piece_end = min(tile_end, u_end);
        const int k0 = kr.lo + (int)(u - at.start) * AT_UNIT;
        const int k1 = min(kr.hi, kr.lo + (int)(piece_end - at.start) * AT_UNIT);
        const int n0 = at.tile * COLS, rows = s.qn * a.group;
        const long long head_off = (long long)at.head * a.pool.block;
        const int* ids = a.pages + (long long)at.b * a.max_pages;

        // ---- page ids of the warp's next 16 steps, one lane per 16 keys
        const int steps = max(0, (k1 - k0 + AT_STEP - 1) / AT_STEP - warp + AT_WARPS - 1) / AT_WARPS;
        auto fetch_ids = [&](int step0) {
            const int key = k0 + ((step0 + (lane >> 1)) * AT_WARPS + warp) * AT_STEP + 16 * (lane & 1);
            int id = -1;
            if (key < k1 && key + 16 > kr.first) {
                id = ids[key >> a.pool.page_shift];
                if (id < 0 || id >= a.pool.pages) {
                    atomicOr(a.err, ERR_INDEX);
                    id = -1;
                }
            }
            return id;
        };
        int cur_ids = fetch_ids(0), next_ids = steps > 16 ? fetch_ids(16) : -1;
        auto issue = [&](int i) {
            if (i < steps) {
                if (i && (i & 15) == 0) {
                    cur_ids = next_ids;
                    next_ids = i + 16 < steps ? fetch_ids(i + 16) : -1;
                }
                const int id0 = __shfl_sync(0xffffffffu, cur_ids, 2 * (i & 15));
                const int id1 = __shfl_sync(0xffffffffu, cur_ids, 2 * (i & 15) + 1);
                load_step<D, NT>(a, ring + (i % C::STAGES) * C::STAGE, head_off,
                                 k0 + (i * AT_WARPS + warp) * AT_STEP, id0, id1);
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < C::STAGES - 1; i++) issue(i);

        // ---- the query rows as B fragments: column g, channels in the order
        // of K's nibbles; and per column pair the lane's constants
        uint32_t qf[NT][NG][4][2];
        float cf[NT][2], qs[NT][NG][2];
        int hi[NT][2], lo[NT][2];
        int min_hi = 0x7fffffff, max_lo = 0;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int n = n0 + 8 * nt + g;
            float x[NG][16];
            float amax = 0.f;
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
                uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
                if (n < rows) {
                    const int tok = n / a.group;
                    const uint16_t* p = (const uint16_t*)a.q.data + (s.row0 + tok) * a.q.st +
                                        (at.head * a.group + n - tok * a.group) * a.q.sh + gr * KV4_GROUP + 16 * c;
                    w0 = ((const uint4*)p)[0];
                    w1 = ((const uint4*)p)[1];
                }
                unpack_bf16x8(w0, x[gr]);
                unpack_bf16x8(w1, x[gr] + 8);
#pragma unroll
                for (int i = 0; i < 16; i++) amax = fmaxf(amax, fabsf(x[gr][i]));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // 2^k brings the row's largest magnitude to [2^13, 2^14)
            const int e = (int)(__float_as_uint(amax) >> 23) - 127;
            const int k = min(max(13 - e, -100), 100);
            const float up = __uint_as_float((uint32_t)(k + 127) << 23);
            float sum[NG];
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
                sum[gr] = 0.f;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    x[gr][i] *= up;
                    sum[gr] += x[gr][i];
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float f = (j & 1) ? 0x1p-4f : 1.f;
                    const __half2 h0 = __floats2half2_rn(x[gr][j] * f, x[gr][4 + j] * f);
                    const __half2 h1 = __floats2half2_rn(x[gr][8 + j] * f, x[gr][12 + j] * f);
                    qf[nt][gr][j][0] = *(const uint32_t*)&h0;
                    qf[nt][gr][j][1] = *(const uint32_t*)&h1;
                }
                sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 1);
                sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 2);
            }
            const float down = a.c * __uint_as_float((uint32_t)(24 - k + 127) << 23);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                cf[nt][j] = __shfl_sync(0xffffffffu, down, 4 * (2 * c + j));
#pragma unroll
                for (int gr = 0; gr < NG; gr++)
                    qs[nt][gr][j] = __shfl_sync(0xffffffffu, sum[gr], 4 * (2 * c + j)) * 0x1p-24f;
                const int m = n0 + 8 * nt + 2 * c + j, tok = min(m, rows - 1) / a.group;
                hi[nt][j] = key_hi(a, s, tok);
                lo[nt][j] = key_lo(a, s, tok);
                min_hi = min(min_hi, hi[nt][j]);
                max_lo = max(max_lo, lo[nt][j]);
            }
        }
        min_hi = __reduce_min_sync(0xffffffffu, min_hi);
        max_lo = __reduce_max_sync(0xffffffffu, max_lo);

        float m[NT][2], l[NT][2], zs[NT][NG][2], o[NT][NG][MT][4], ones[NT][NG][4];
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
                for (int i = 0; i < 4; i++) {
                    ones[nt][gr][i] = 0.f;
#pragma unroll
                    for (int t = 0; t < MT; t++) o[nt][gr][t][i] = 0.f;
                }
        }

        // ---- the warp's steps
        for (int i = 0; i < steps; i++) {
            cp_wait<C::STAGES - 2>();
            __syncwarp();
            issue(i + C::STAGES - 1);
            const uint32_t st = ring + (i % C::STAGES) * C::STAGE;
            const int key0 = k0 + (i * AT_WARPS + warp) * AT_STEP;
            const bool edge = key0 + AT_STEP > min(min_hi, k1) || key0 < max_lo;
            float x[2][NT][4];  // [16 keys][columns][C fragment]: S, then P
            float vs[2][2][NG], vz[2][2][NG];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                // S^T rows g and g + 8 of this half: keys kl and kl + 8
                const int kl = 16 * h + (g >> 1) + 4 * (g & 1);
                float acc[NG][NT][4];
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    const uint2 wl = lds64(st + stage_at<D>(kl, gr * 32 + c * 8));
                    const uint2 wh = lds64(st + stage_at<D>(kl + 8, gr * 32 + c * 8));
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int q = 0; q < 4; q++) acc[gr][nt][q] = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int sh = j >= 2 ? 8 : 0;
                        const uint32_t mask = (j & 1) ? 0x00f000f0u : 0x000f000fu;
                        const uint32_t f[4] = {(wl.x >> sh) & mask, (wh.x >> sh) & mask, (wl.y >> sh) & mask,
                                               (wh.y >> sh) & mask};
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) mma_f16(acc[gr][nt], f, qf[nt][gr][j][0], qf[nt][gr][j][1]);
                    }
                }
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const uint32_t par = st + 2 * C::VAL + (kl + 8 * r) * (NG * 4);
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
                        vz[h][r][gr] = fmaf(8.f, vs[h][r][gr], bf_hi(vp[gr]));
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
                            if (bad[gr]) vs[h][r][gr] = vz[h][r][gr] = 0.f;
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
                            ones[nt][gr][j] *= f;
#pragma unroll
                            for (int t = 0; t < MT; t++) {
                                o[nt][gr][t][j] *= f;
                                o[nt][gr][t][2 + j] *= f;
                            }
                        }
                    }
            }
            float mc[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) mc[nt][j] = m[nt][j] == -INFINITY ? 0.f : m[nt][j] * cf[nt][j];

#pragma unroll
            for (int h = 0; h < 2; h++) {
                // P^T fragments per group: k index 2c, 2c+1 are rows 2c, 2c+1
                // of S^T, keys c and c + 4 (and 8 more)
                uint32_t pf[NT][NG][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int i4 = 0; i4 < 4; i4++) {
                        const int r = i4 >> 1, j = i4 & 1;
                        const float p = ex2(fmaf(x[h][nt][i4], cf[nt][j], -mc[nt][j]));
                        x[h][nt][i4] = p;
                        l[nt][j] += p;
#pragma unroll
                        for (int gr = 0; gr < NG; gr++) zs[nt][gr][j] = fmaf(p, vz[h][r][gr], zs[nt][gr][j]);
                    }
#pragma unroll
                    for (int gr = 0; gr < NG; gr++)
#pragma unroll
                        for (int r = 0; r < 2; r++)
                            pf[nt][gr][r] = transpose8(pack_bf16x2(x[h][nt][2 * r] * vs[h][r][gr],
                                                                   x[h][nt][2 * r + 1] * vs[h][r][gr]));
                }
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    uint32_t w[4];  // 8 channels of keys c, c + 4, c + 8, c + 12
#pragma unroll
                    for (int i4 = 0; i4 < 4; i4++)
                        w[i4] = lds32(st + C::VAL + stage_at<D>(16 * h + c + 4 * i4, gr * 32 + g * 4));
                    uint32_t up[4], dn[4];
#pragma unroll
                    for (int i4 = 0; i4 < 4; i4++) {
                        up[i4] = w[i4] << 3;
                        dn[i4] = w[i4] >> 1;
                    }
#pragma unroll
                    for (int t = 0; t < MT; t++) {  // channels 8g + 2t (row g) and 8g + 2t + 1 (row g + 8)
                        const uint32_t sel = t | (t << 4) | ((4 + t) << 8) | ((4 + t) << 12);
                        const uint32_t f[4] = {(__byte_perm(up[0], up[1], sel) & 0x00780078u) | 0x41804180u,
                                               (__byte_perm(dn[0], dn[1], sel) & 0x00780078u) | 0x41804180u,
                                               (__byte_perm(up[2], up[3], sel) & 0x00780078u) | 0x41804180u,
                                               (__byte_perm(dn[2], dn[3], sel) & 0x00780078u) | 0x41804180u};
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) mma_bf16(o[nt][gr][t], f, pf[nt][gr][0], pf[nt][gr][1]);
                    }
                    const uint32_t one[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) mma_bf16(ones[nt][gr], one, pf[nt][gr][0], pf[nt][gr][1]);
                }
            }
        }
        cp_wait<0>();
        __syncwarp();

        // ---- the warps' outputs meet: own = acc - 24 sum(p s) + sum(p (z + 8 s))
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int col = 8 * nt + 2 * c + j;
                float z[NG], ls = l[nt][j];
#pragma unroll
                for (int i = 4; i < 32; i <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, i);
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    z[gr] = zs[nt][gr][j];
#pragma unroll
                    for (int i = 4; i < 32; i <<= 1) z[gr] += __shfl_xor_sync(0xffffffffu, z[gr], i);
                    z[gr] -= 24.f * ones[nt][gr][j];
#pragma unroll
                    for (int t = 0; t < MT; t++) {
                        float2 v = make_float2(o[nt][gr][t][j] + z[gr], o[nt][gr][t][2 + j] + z[gr]);
                        *(float2*)(sm_o + col * D + gr * KV4_GROUP + 8 * g + 2 * t) = v;
                    }
                }
                if (g == 0) {
                    sm_m[warp][col] = m[nt][j] == -INFINITY ? -INFINITY : m[nt][j] * cf[nt][j];
                    sm_l[warp][col] = ls;
                }
            }
        __syncthreads();
        const bool whole = u == at.start && piece_end == tile_end;
        const int slot = 2 * (int)blockIdx.x + (at.start < u_begin ? 0 : 1);
        for (int i = threadIdx.x; i < COLS * D / 4; i += blockDim.x) {
            const int col = i / (D / 4), d4 = i % (D / 4) * 4, n = n0 + col;
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
                const float4 y = *(const float4*)((const float*)(smem + w * C::WARP) + col * D + d4);
                sum = fmaf(f, sm_l[w][col], sum);
                v.x = fmaf(f, y.x, v.x); v.y = fmaf(f, y.y, v.y);
                v.z = fmaf(f, y.z, v.z); v.w = fmaf(f, y.w, v.w);
            }
            if (whole) {
                put_row<D>(a, s, at.head, n, d4, v, ref, sum);
            } else {
                *(float4*)(a.part_o + ((long long)slot * COLS + col) * D + d4) = v;
                if (d4 == 0) a.part_ml[slot * COLS + col] = make_float2(mm, sum);
            }
        }
        __syncthreads();

        // ---- the next tile
        u = piece_end;
        if (u < u_end) {
            at.start = tile_end;
            if (++at.tile >= s.tiles) {
                at.tile = 0;
                if (++at.head >= a.pool.kv_heads) {
                    at.head = 0;
                    do at.b++;
                    while (at.b < a.batch && seq_at<COLS>(a, at.b).tiles == 0);
                }
            }
        }
    }
}

// Joins the pieces of split tiles: block (c, column) joins that column of the
// tile that begins in CTA c and ends in a later one.  A thread holds 4
// channels of every (128 / (D/4))-th piece.
template <int D, int COLS, int UNIT>
__global__ void __launch_bounds__(128) sp_kv4_join(const __grid_constant__ Kv4Attend a) {
    constexpr int LANES = D / 4, SLICES = 128 / LANES;
    __shared__ float4 sm_v[SLICES][LANES];
    __shared__ float2 sm_ml[SLICES];
    const int col = blockIdx.y, lane = threadIdx.x % LANES, slice = threadIdx.x / LANES;
    long long total, none;
    count_units<COLS, UNIT>(a, 0, total, none);
    total *= a.pool.kv_heads;
    const int G = shares(total, gridDim.x);
    if ((int)blockIdx.x >= G) return;
    const long long u0 = first_unit(blockIdx.x, total, G), u1 = first_unit(blockIdx.x + 1, total, G);
    const Place at = find_unit<COLS, UNIT>(a, u1 - 1);
    const Seq s = seq_at<COLS>(a, at.b);
    const long long end = at.start + keys_of<COLS, UNIT>(a, s, at.tile).units;
    const int n = at.tile * COLS + col;
    if (at.start < u0 || end <= u1 || n >= s.qn * a.group) return;
    const int c0 = blockIdx.x, c1 = cta_of(end - 1, total, G);
    griddep_wait();
    float m = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0 + slice; c <= c1; c += SLICES) m = fmaxf(m, a.part_ml[(2 * c + (c == c0)) * COLS + col].x);
    const float own_ref = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int c = c0 + slice; c <= c1; c += SLICES) {
        const long long slot = (long long)(2 * c + (c == c0)) * COLS + col;
        const float2 ml = a.part_ml[slot];
        const float4 y = *(const float4*)(a.part_o + slot * D + 4 * lane);
        const float f = ex2(ml.x - own_ref);
        sum = fmaf(f, ml.y, sum);
        v.x = fmaf(f, y.x, v.x); v.y = fmaf(f, y.y, v.y);
        v.z = fmaf(f, y.z, v.z); v.w = fmaf(f, y.w, v.w);
    }
    sm_v[slice][lane] = v;
    if (lane == 0) sm_ml[slice] = make_float2(m, sum);
    __syncthreads();
    if (slice) return;
    float mm = -INFINITY;
#pragma unroll
    for (int i = 0; i < SLICES; i++) mm = fmaxf(mm, sm_ml[i].x);
    const float ref = mm == -INFINITY ? 0.f : mm;
    sum = 0.f;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < SLICES; i++) {
        const float f = ex2(sm_ml[i].x - ref);
        const float4 y = sm_v[i][lane];
        sum = fmaf(f, sm_ml[i].y, sum);
        v.x = fmaf(f, y.x, v.x); v.y = fmaf(f, y.y, v.y);
        v.z = fmaf(f, y.z, v.z); v.w = fmaf(f, y.w, v.w);
    }
    put_row<D>(a, s, at.head, n, 4 * lane, v, ref, sum);
}

size_t kv4_scratch_bytes(int d, int sms) { return (size_t)2 * 2 * sms * 16 * (d + 2) * sizeof(float); }

template <int D, int NT>
static cudaError_t attend(Kv4Attend a, int sms, cudaStream_t st) {
    using C = AttnCfg<D, NT>;
    constexpr int COLS = C::COLS;
    const int G = (NT == 1 ? 2 : 1) * sms;
    a.part_ml = (float2*)a.scratch;
    a.part_o = (float*)(a.part_ml + (size_t)2 * G * COLS);
    cudaError_t e = cudaFuncSetAttribute(sp_kv4_attend<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    sp_kv4_attend<D, NT><<<G, AT_WARPS * 32, C::SMEM, st>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    return launch_after_previous(sp_kv4_join<D, COLS, AT_UNIT>, dim3(G, COLS), dim3(128), 0, st, a);
}

cudaError_t launch_kv4_attend(int d, const Kv4Attend& a, int sms, cudaStream_t st) {
    const int rows = a.max_q * a.group;
    if (d == 64) return rows <= 8 ? attend<64, 1>(a, sms, st) : attend<64, 2>(a, sms, st);
    return rows <= 8 ? attend<128, 1>(a, sms, st) : attend<128, 2>(a, sms, st);
}

}  // namespace sp
