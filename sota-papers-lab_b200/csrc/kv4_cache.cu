// Tokens into and out of the paged 4-bit KV cache (kv4.h has its layout).
//
// Append, per token: K rotated by its position, then K and V quantised with
// one scale and zero per 64 channels:
//   zero = bf16(min), scale = bf16((max - min) * (1/15)),
//   n = clamp(rint((x - zero) / scale), 0, 15)
// from the rotated channels in f32 (they are not rounded to bf16 in between).
// All steps are single IEEE operations, so the stored bytes are defined to
// the bit.  A group with a NaN or an infinity, or whose range does not fit
// bf16, is stored as scale = zero = NaN, n = 0; one whose scale is below
// 2^-100 (a constant group) as scale = 0, n = 0.  Q, where given, is rotated
// on the way (one launch a layer instead of three).
//
// Bound by latency for a few tokens (64 tokens of 32 / 8 heads: 4.3 us with the
// read back), by memory and the ALUs together for many (8192 tokens of 32 / 8
// heads, D = 128, 181 MB: 38 us, 4.8 TB/s, the hottest pipe 55% busy).  A thread
// holds one unit (16 channels, rotary.cuh) of HPT heads, so that one read of
// its angles serves them all; the minimum and maximum of a group come from
// shuffles among the D/16 lanes of a row.
#include "rotary.cuh"
#include "sage_kernels.h"

namespace sp {

constexpr float FINITE_MAX = 3.402823466e38f;

// Minimum and maximum that a NaN gets through.
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

__device__ __forceinline__ float min_nan(float a, float b, float c) {
    float d;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// One 8-channel chunk's minimum and maximum.
__device__ __forceinline__ void chunk_range(const float (&x)[8], float& mn, float& mx) {
    mn = min_nan(x[0], x[1], x[2]);
    mx = max_nan(x[0], x[1], x[2]);
#pragma unroll
    for (int i = 3; i < 7; i += 2) {
        mn = min_nan(mn, x[i], x[i + 1]);
        mx = max_nan(mx, x[i], x[i + 1]);
    }
    mn = min_nan(mn, x[7]);
    mx = max_nan(mx, x[7]);
}

// Scale and zero of a group (bf16 bits, scale in the low half) and what the
// division by the scale needs.
struct GroupScale {
    float inv;  // 0: every n is 0
    uint32_t bits;
};

__device__ __forceinline__ GroupScale group_scale(float mn, float mx) {
    GroupScale g;
    const float range = __fsub_rn(mx, mn);
    g.bits = pack_bf16x2(__fmul_rn(range, 1.0f / 15.0f), mn);
    const float scale = __uint_as_float(g.bits << 16), zero = __uint_as_float(g.bits & 0xffff0000u);
    const bool fine = range <= FINITE_MAX && fabsf(scale) <= FINITE_MAX && fabsf(zero) <= FINITE_MAX;
    g.inv = 0.f;
    if (!fine) {
        g.bits = 0x7fc07fc0u;
    } else if (scale < 0x1p-100f) {
        g.bits &= 0xffff0000u;
    } else {
        g.inv = __frcp_rn(scale);
    }
    return g;
}

// n of 8 channels, channel i at bits 4i.  (x - zero) / scale is the product
// with the reciprocal corrected once by its exact remainder (Markstein: the
// quotient rounded to nearest, given a correctly rounded reciprocal); ties of
// the quotient, common for bf16 inputs, come out as ties.  It is below 2^20 in
// size: zero is off by 2^-9 of the minimum at most, and the range is a 2^-24th
// of it or nothing.  So adding 1.5 * 2^23 rounds it to the nearest even integer
// and leaves that in the low bits, from where pairs are packed with saturation.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], const GroupScale& g) {
    constexpr int BITS = 0x4b400000;  // of 1.5 * 2^23
    auto mul2 = [](uint64_t a, uint64_t b) {  // (its result is only ever multiplied or added to: nothing to fuse it with)
        uint64_t d;
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
        return d;
    };
    const float z = __uint_as_float(g.bits & 0xffff0000u), s = __uint_as_float(g.bits << 16);
    const uint64_t zero = pk2(z, z), less = pk2(-s, -s), inv = pk2(g.inv, g.inv);
    uint32_t w = 0;
#pragma unroll
    for (int i = 6; i >= 0; i -= 2) {
        const uint64_t y = sub2(pk2(x[i], x[i + 1]), zero);
        uint64_t q = mul2(y, inv);
        q = fma2(fma2(q, less, y), inv, q);
        float q0, q1;
        upk2(add2(q, pk2(12582912.f, 12582912.f)), q0, q1);
        asm("cvt.pack.sat.u4.s32.b32 %0, %1, %2, %0;"
            : "+r"(w)
            : "r"(__float_as_int(q1) - BITS), "r"(__float_as_int(q0) - BITS));
    }
    return g.inv == 0.f ? 0u : w;
}

// Small blocks, because warps of Q are done long before those of K and V.
constexpr int APPEND_THREADS = 64;

// A warp takes 32 / (D/16) * HPT heads of one token, all of Q, of K or of V
// (row_blocks warps a token; q_blocks of them Q's, half of the rest K's).
template <int D, int HPT>
__global__ void __launch_bounds__(APPEND_THREADS, 16) sp_kv4_append(const Kv4Pool pool, const Rows q, const Rows q_out,
                                                                const Rows k, const Rows v, const RotaryArgs r,
                                                                const int* __restrict__ slots, int tokens, int q_heads,
                                                                int q_blocks, int row_blocks,
                                                                uint32_t* __restrict__ err) {
    constexpr int UNITS = D / 16, HL = 32 / UNITS, NG = D / KV4_GROUP;
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t w = blockIdx.x * (APPEND_THREADS / 32) + threadIdx.x / 32;
    const int t = (int)(w / (uint32_t)row_blocks);
    if (t >= tokens) return;
    int rb = (int)(w - (uint32_t)t * (uint32_t)row_blocks);
    const int lane = threadIdx.x & 31, u = lane % UNITS;
    const int slot = slots[t], page = slot >> pool.page_shift;
    const bool turned = r.table != nullptr;
    const int pos = turned ? r.positions[t] : 0;
    const int kv_blocks = (row_blocks - q_blocks) / 2;
    const bool is_q = rb < q_blocks, is_v = rb >= q_blocks + kv_blocks;
    if (!is_q) rb -= is_v ? q_blocks + kv_blocks : q_blocks;
    const Rows src = is_q ? q : is_v ? v : k;
    const int heads = is_q ? q_heads : pool.kv_heads, first = rb * HL * HPT, h0 = first + lane / UNITS;
    Unit x = unit_at(u, r);
    if (is_v) x = {16 * u, 16 * u + 8, false};
    // the rows are on their way before the slot and the position are looked at
    const uint16_t* from = (const uint16_t*)src.data + t * src.st;
    Chunk<0> lo[HPT], hi[HPT];
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        if (first + i * HL >= heads) break;
        const uint16_t* row = from + min(h0 + i * HL, heads - 1) * src.sh;  // (lanes without a row take the last)
        lo[i].load(row, x.c0);
        hi[i].load(row, x.c1);
    }
    if ((turned && (pos < 0 || pos >= r.limit)) || page >= pool.pages) {  // the token is left out
        if (lane == 0) atomicOr(err + ERR_INDEX_WORD, ERR_INDEX);
        return;
    }
    if (!is_q && slot < 0) return;  // not cached
    float cs[16];
    if (x.turns) load_angles(r, pos, u, cs);
    if (is_q) {
        uint16_t* to = (uint16_t*)q_out.data + t * q_out.st;
#pragma unroll
        for (int i = 0; i < HPT; i++) {
            if (h0 + i * HL >= heads) break;
            if (x.turns) {
                float a[8], b[8];
                lo[i].to(a);
                hi[i].to(b);
                turn(a, b, cs, r.interleaved, false);
                lo[i].from(a);
                hi[i].from(b);
            }
            uint16_t* row = to + (h0 + i * HL) * q_out.sh;
            lo[i].store(row, x.c0);
            hi[i].store(row, x.c1);
        }
        return;
    }
    const int in_page = slot & (pool.page_tokens - 1);
    const int half = pool.page_tokens * (D / 2), par = pool.page_tokens * NG * 4;
    uint8_t* blk = pool.data + page * pool.page_stride + (long long)h0 * pool.block;
    uint8_t* val = blk + (is_v ? half : 0) + in_page * (D / 2);
    uint8_t* params = blk + 2 * half + (is_v ? par : 0) + (in_page * NG + u) * 4;
    // D = 128: an even lane gathers its row's group 0, an odd one group 1
    const int mine = NG == 2 ? u & 1 : 0;
    const bool ma = x.c0 / KV4_GROUP == mine, mb = x.c1 / KV4_GROUP == mine;
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        if (first + i * HL >= heads) break;
        float a[8], b[8];
        lo[i].to(a);
        hi[i].to(b);
        if (x.turns) turn(a, b, cs, r.interleaved, false);
        // all lanes of the warp meet in the shuffles
        float amn, amx, bmn, bmx;
        chunk_range(a, amn, amx);
        chunk_range(b, bmn, bmx);
        float mn = min_nan(ma ? amn : INFINITY, mb ? bmn : INFINITY);
        float mx = max_nan(ma ? amx : -INFINITY, mb ? bmx : -INFINITY);
        if constexpr (NG == 2) {
            const float omn = min_nan(ma ? INFINITY : amn, mb ? INFINITY : bmn);
            const float omx = max_nan(ma ? -INFINITY : amx, mb ? -INFINITY : bmx);
            mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, omn, 1));
            mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, omx, 1));
        }
#pragma unroll
        for (int m = NG; m < UNITS; m *= 2) {
            mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, m));
            mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, m));
        }
        const GroupScale g = group_scale(mn, mx);
        GroupScale o = g;
        if constexpr (NG == 2) {
            o.bits = __shfl_xor_sync(0xffffffffu, g.bits, 1);
            o.inv = __shfl_xor_sync(0xffffffffu, g.inv, 1);
        }
        if (h0 + i * HL >= heads) break;  // (of the last i only)
        *(uint32_t*)(val + x.c0 / 2) = quantise8(a, ma ? g : o);
        *(uint32_t*)(val + x.c1 / 2) = quantise8(b, mb ? g : o);
        if (u < NG) *(uint32_t*)params = g.bits;
        val += HL * pool.block;
        params += HL * pool.block;
    }
}

template <int D>
static cudaError_t append(const Kv4Pool& pool, const Rows& q, const Rows& q_out, const Rows& k, const Rows& v,
                          const RotaryArgs& r, const int* slots, int tokens, int q_heads, int sms,
                          uint32_t* err, cudaStream_t st) {
    constexpr int HL = 512 / D;
    // Two heads a thread, which share the angles, once that makes two rounds of
    // warps (append and read back, two heads against one: 8192 tokens of 32 / 8
    // heads, D = 128, 45 us and 60, 1024 tokens 9.8 and 9.4; 1370 tokens of 16
    // heads, D = 64, 9.2 and 7.9, 4096 tokens 16.5 and 18.7; four: 52 and 8.4).
    constexpr int MANY = 2;
    auto blocks = [](int heads, int per) { return (heads + per - 1) / per; };
    const bool many =
        (long long)tokens * (blocks(q_heads, MANY * HL) + 2 * blocks(pool.kv_heads, MANY * HL)) >= sms * 64;
    const int per = many ? MANY * HL : HL, qb = blocks(q_heads, per), rb = qb + 2 * blocks(pool.kv_heads, per);
    const unsigned grid = (unsigned)(((long long)tokens * rb + APPEND_THREADS / 32 - 1) / (APPEND_THREADS / 32));
    return launch_after_previous(many ? sp_kv4_append<D, MANY> : sp_kv4_append<D, 1>, dim3(grid), dim3(APPEND_THREADS), 0,
                                 st, pool, q, q_out, k, v, r, slots, tokens, q_heads, qb, rb, err);
}

cudaError_t launch_kv4_append(int d, const Kv4Pool& pool, const Rows& q, const Rows& q_out, const Rows& k,
                              const Rows& v, const RotaryArgs& r, const int* slots, int tokens, int q_heads, int sms,
                              uint32_t* err, cudaStream_t st) {
    return d == 64 ? append<64>(pool, q, q_out, k, v, r, slots, tokens, q_heads, sms, err, st)
                   : append<128>(pool, q, q_out, k, v, r, slots, tokens, q_heads, sms, err, st);
}

// The values at given slots, zero + scale * n rounded once to bf16.  A thread
// reads one word (8 channels) of READ_TOKENS tokens and writes 16 bytes of
// each; bound by the bf16 rows it writes.
constexpr int READ_TOKENS = 4;

template <int D>
__global__ void __launch_bounds__(256) sp_kv4_read(const Kv4Pool pool, const int* __restrict__ slots, const Rows k,
                                                   const Rows v, int tokens, uint32_t* __restrict__ err) {
    constexpr int CH = D / 8, NG = D / KV4_GROUP;
    griddep_wait();
    griddep_launch_dependents();
    const int c = threadIdx.x % CH, row = blockIdx.y * (256 / CH) + threadIdx.x / CH;
    if (row >= 2 * pool.kv_heads) return;
    const bool is_v = row >= pool.kv_heads;
    const int h = is_v ? row - pool.kv_heads : row, t0 = blockIdx.x * READ_TOKENS;
    const int half = pool.page_tokens * (D / 2), par = pool.page_tokens * NG * 4;
    const uint8_t* head = pool.data + (long long)h * pool.block;
    uint32_t w[READ_TOKENS], p[READ_TOKENS];
    bool put[READ_TOKENS];
#pragma unroll
    for (int i = 0; i < READ_TOKENS; i++) {
        w[i] = p[i] = 0;
        put[i] = t0 + i < tokens;
        if (!put[i]) continue;
        const int slot = slots[t0 + i], page = slot >> pool.page_shift;
        if (page >= pool.pages) {
            if (c == 0 && row == 0) atomicOr(err + ERR_INDEX_WORD, ERR_INDEX);
            put[i] = false;
        } else if (slot >= 0) {
            const int in_page = slot & (pool.page_tokens - 1);
            const uint8_t* blk = head + page * pool.page_stride;
            w[i] = *(const uint32_t*)(blk + (is_v ? half : 0) + in_page * (D / 2) + c * 4);
            p[i] = ((const uint32_t*)(blk + 2 * half + (is_v ? par : 0)))[in_page * NG + c * 8 / KV4_GROUP];
        }
    }
    const Rows& dst = is_v ? v : k;
#pragma unroll
    for (int i = 0; i < READ_TOKENS; i++) {
        if (!put[i]) continue;
        // nibble j of a half word under 2^23's exponent: 2^23 + 16^j n, hence 16^j n,
        // which meets scale / 16^j (exact: a scale is at least 2^-100 or none)
        const float s = __uint_as_float(p[i] << 16), z = __uint_as_float(p[i] & 0xffff0000u);
        const uint64_t zero = pk2(z, z), s01 = pk2(s, s * 0x1p-4f), s23 = pk2(s * 0x1p-8f, s * 0x1p-12f);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint32_t h = j < 4 ? w[i] : w[i] >> 16, m = 15u << (4 * (j & 3));
            const uint64_t n = add2(pk2(__uint_as_float((h & m) | 0x4b000000u), __uint_as_float((h & m << 4) | 0x4b000000u)),
                                    pk2(-8388608.f, -8388608.f));
            upk2(fma2(n, (j & 2) ? s23 : s01, zero), f[j], f[j + 1]);
        }
        Chunk<0> o;
        o.from(f);
        o.store((void*)dst.data, (t0 + i) * dst.st + h * dst.sh + 8 * c);
    }
}

cudaError_t launch_kv4_read(int d, const Kv4Pool& pool, const int* slots, const Rows& k, const Rows& v, int tokens,
                            uint32_t* err, cudaStream_t st) {
    const int rows_a_block = 256 / (d / 8);
    const dim3 grid((tokens + READ_TOKENS - 1) / READ_TOKENS, (2 * pool.kv_heads + rows_a_block - 1) / rows_a_block);
    return launch_after_previous(d == 64 ? sp_kv4_read<64> : sp_kv4_read<128>, grid, dim3(256), 0, st, pool, slots, k, v,
                                 tokens, err);
}

}  // namespace sp
