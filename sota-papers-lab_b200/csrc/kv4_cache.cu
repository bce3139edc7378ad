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
// Bound by memory (and by latency for a few tokens): a thread holds one unit
// (16 channels, rotary.cuh) of HPT rows, so that one read of its angles
// serves them all; the minimum and maximum of a group come from shuffles
// among the D/16 lanes of a row.
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

// One 8-channel chunk's minimum and maximum.
__device__ __forceinline__ void chunk_range(const float (&x)[8], float& mn, float& mx) {
    mn = mx = x[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        mn = min_nan(mn, x[i]);
        mx = max_nan(mx, x[i]);
    }
}

// Scale and zero of a group (bf16 bits, scale in the low half) and what the
// division by the scale needs.
struct GroupScale {
    float zero, scale, inv;  // inv = 0: every n is 0
    uint32_t bits;
};

__device__ __forceinline__ GroupScale group_scale(float mn, float mx) {
    GroupScale g;
    const float range = __fsub_rn(mx, mn);
    g.bits = pack_bf16x2(__fmul_rn(range, 1.0f / 15.0f), mn);
    g.scale = __uint_as_float(g.bits << 16);
    g.zero = __uint_as_float(g.bits & 0xffff0000u);
    const bool fine = range <= FINITE_MAX && fabsf(g.scale) <= FINITE_MAX && fabsf(g.zero) <= FINITE_MAX;
    g.inv = 0.f;
    if (!fine) {
        g.bits = 0x7fc07fc0u;
        g.zero = g.scale = 0.f;
    } else if (g.scale < 0x1p-100f) {
        g.bits &= 0xffff0000u;
        g.scale = 0.f;
    } else {
        g.inv = __frcp_rn(g.scale);
    }
    return g;
}

// n of 8 channels, channel i at bits 4i.  (x - zero) / scale is the product
// with the reciprocal corrected once by its exact remainder (Markstein: the
// quotient rounded to nearest, given a correctly rounded reciprocal); ties of
// the quotient, common for bf16 inputs, come out as ties.  Adding 1.5 * 2^23
// rounds to the nearest even integer and leaves it in the low bits; the eight
// are put together by Horner's rule in 32-bit arithmetic, in which the
// constant's bits add up to another constant.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], const GroupScale& g) {
    constexpr uint32_t BITS = 0x4b400000u;  // of 1.5 * 2^23
    auto mul2 = [](uint64_t a, uint64_t b) {  // (its result is only ever multiplied or added to: nothing to fuse it with)
        uint64_t d;
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
        return d;
    };
    const uint64_t zero = pk2(g.zero, g.zero), less = pk2(-g.scale, -g.scale), inv = pk2(g.inv, g.inv);
    uint32_t w = 0;
#pragma unroll
    for (int i = 6; i >= 0; i -= 2) {
        const uint64_t y = sub2(pk2(x[i], x[i + 1]), zero);
        uint64_t q = mul2(y, inv);
        q = fma2(fma2(q, less, y), inv, q);
        float q0, q1;
        upk2(q, q0, q1);
        q0 = fminf(fmaxf(q0, 0.f), 15.f);  // (a NaN: 0)
        q1 = fminf(fmaxf(q1, 0.f), 15.f);
        upk2(add2(pk2(q0, q1), pk2(12582912.f, 12582912.f)), q0, q1);
        w = w * 16u + __float_as_uint(q1);
        w = w * 16u + __float_as_uint(q0);
    }
    return w - BITS * 0x11111111u;
}

template <int D, int HPT>
__global__ void __launch_bounds__(256) sp_kv4_append(const Kv4Pool pool, const Rows q, const Rows q_out, const Rows k,
                                                     const Rows v, const RotaryArgs r, const int* __restrict__ slots,
                                                     int tokens, int q_heads, int row_blocks,
                                                     uint32_t* __restrict__ err) {
    constexpr int UNITS = D / 16, HL = 32 / UNITS, NG = D / KV4_GROUP;
    griddep_wait();
    griddep_launch_dependents();
    const long long w = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int t = (int)(w / row_blocks), rb = (int)(w % row_blocks);
    if (t >= tokens) return;
    const int lane = threadIdx.x & 31, u = lane % UNITS;
    const int row0 = rb * HL * HPT + lane / UNITS;  // rows: Q heads, K heads, V heads
    const int hkv = pool.kv_heads, rows = q_heads + 2 * hkv;
    const Unit un = unit_at(u, r);
    const RotaryArgs still = {nullptr, nullptr, 0, 0, 0};
    const Unit vn = unit_at(u, still);
    int pos = 0;
    bool ok = true;
    if (r.table) {
        pos = r.positions[t];
        ok = pos >= 0 && pos < r.limit;
    }
    const int slot = slots[t];
    const int page = slot >> pool.page_shift;
    if (!ok || page >= pool.pages) {  // the token is left out
        if (lane == 0) atomicOr(err + ERR_INDEX_WORD, ERR_INDEX);
        return;
    }
    Chunk<0> lo[HPT], hi[HPT];
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        const int row = row0 + i * HL;
        if (row < rows) {
            const bool is_v = row >= q_heads + hkv;
            const Rows& src = row < q_heads ? q : is_v ? v : k;
            const int h = row < q_heads ? row : is_v ? row - q_heads - hkv : row - q_heads;
            const long long at = t * src.st + h * src.sh;
            lo[i].load(src.data, at + (is_v ? vn.c0 : un.c0));
            hi[i].load(src.data, at + (is_v ? vn.c1 : un.c1));
        }
    }
    float cs[16];
    if (un.turns) load_angles(r, pos, u, cs);
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        const int row = row0 + i * HL;
        const bool is_q = row < q_heads, is_v = row >= q_heads + hkv;
        float a[8] = {}, b[8] = {};
        if (row < rows) {
            lo[i].to(a);
            hi[i].to(b);
            if (!is_v && un.turns) turn(a, b, cs, r.interleaved, false);
            if (is_q) {
                const long long at = t * q_out.st + row * q_out.sh;
                lo[i].from(a);
                hi[i].from(b);
                lo[i].store((void*)q_out.data, at + un.c0);
                hi[i].store((void*)q_out.data, at + un.c1);
            }
        }
        // all lanes of the warp meet in the shuffles below
        if (slot < 0 || !__any_sync(0xffffffffu, !is_q && row < rows)) continue;
        const Unit x = is_v ? vn : un;
        float amn, amx, bmn, bmx;
        chunk_range(a, amn, amx);
        chunk_range(b, bmn, bmx);
        GroupScale g[NG];
#pragma unroll
        for (int j = 0; j < NG; j++) {
            const bool ia = x.c0 / KV4_GROUP == j, ib = x.c1 / KV4_GROUP == j;
            float mn = min_nan(ia ? amn : INFINITY, ib ? bmn : INFINITY);
            float mx = max_nan(ia ? amx : -INFINITY, ib ? bmx : -INFINITY);
#pragma unroll
            for (int m = 1; m < UNITS; m *= 2) {
                mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, m));
                mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, m));
            }
            g[j] = group_scale(mn, mx);
        }
        if (is_q || row >= rows) continue;
        const int in_page = slot & (pool.page_tokens - 1);
        uint8_t* blk = pool.data + page * pool.page_stride +
                       (long long)(is_v ? row - q_heads - hkv : row - q_heads) * pool.block;
        const int half = pool.page_tokens * (D / 2), par = pool.page_tokens * NG * 4;
        uint8_t* val = blk + (is_v ? half : 0) + in_page * (D / 2);
        *(uint32_t*)(val + x.c0 / 2) = quantise8(a, x.c0 < KV4_GROUP ? g[0] : g[NG - 1]);
        *(uint32_t*)(val + x.c1 / 2) = quantise8(b, x.c1 < KV4_GROUP ? g[0] : g[NG - 1]);
        if (u < NG)
            ((uint32_t*)(blk + 2 * half + (is_v ? par : 0)))[in_page * NG + u] = u == 0 ? g[0].bits : g[NG - 1].bits;
    }
}

template <int D>
static cudaError_t append(const Kv4Pool& pool, const Rows& q, const Rows& q_out, const Rows& k, const Rows& v,
                          const RotaryArgs& r, const int* slots, int tokens, int q_heads, uint32_t* err,
                          cudaStream_t st) {
    constexpr int HL = 512 / D;
    const int rows = q_heads + 2 * pool.kv_heads;
    // Two rows a thread once that still leaves every SM a few warps (append and
    // read back of 8192 tokens, 32 / 8 heads, D = 128: 62 us, with 1 66, with 4
    // 70, whose registers leave two blocks on an SM; 1370 tokens of 16 heads, D
    // = 64: 9.1, 8.9, 10.7).
    constexpr int MANY = 2;
    const bool many = (long long)tokens * ((rows + MANY * HL - 1) / (MANY * HL)) >= 148 * 16;
    const int per = many ? MANY : 1, rb = (rows + per * HL - 1) / (per * HL);
    const unsigned grid = (unsigned)(((long long)tokens * rb + 7) / 8);
    return launch_after_previous(many ? sp_kv4_append<D, MANY> : sp_kv4_append<D, 1>, dim3(grid), dim3(256), 0, st, pool, q,
                                 q_out, k, v, r, slots, tokens, q_heads, rb, err);
}

cudaError_t launch_kv4_append(int d, const Kv4Pool& pool, const Rows& q, const Rows& q_out, const Rows& k,
                              const Rows& v, const RotaryArgs& r, const int* slots, int tokens, int q_heads,
                              uint32_t* err, cudaStream_t st) {
    return d == 64 ? append<64>(pool, q, q_out, k, v, r, slots, tokens, q_heads, err, st)
                   : append<128>(pool, q, q_out, k, v, r, slots, tokens, q_heads, err, st);
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
        const float scale = __uint_as_float(p[i] << 16), zero = __uint_as_float(p[i] & 0xffff0000u);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float n = __uint_as_float(((w[i] >> (4 * j)) & 15u) | 0x4b000000u) - 8388608.f;  // 2^23 + n, n
            f[j] = __fmaf_rn(scale, n, zero);
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
