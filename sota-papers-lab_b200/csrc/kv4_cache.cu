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

// One 8-channel chunk's minimum and maximum; a NaN or an infinity makes the
// range infinite, which marks the group.
__device__ __forceinline__ void chunk_range(const float (&x)[8], float& mn, float& mx) {
    mn = mx = x[0];
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        mn = fminf(mn, x[i]);
        mx = fmaxf(mx, x[i]);
        fine = fine && fabsf(x[i]) <= FINITE_MAX;
    }
    if (!fine) mn = -INFINITY;
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
// the quotient, common for bf16 inputs, come out as ties.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], const GroupScale& g) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float y = __fsub_rn(x[i], g.zero);
        float q = __fmul_rn(y, g.inv);
        q = __fmaf_rn(__fmaf_rn(-q, g.scale, y), g.inv, q);
        const int n = __float2int_rn(fminf(fmaxf(q, 0.f), 15.f));
        w |= (uint32_t)n << (4 * i);
    }
    return w;
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
            float mn = fminf(ia ? amn : INFINITY, ib ? bmn : INFINITY);
            float mx = fmaxf(ia ? amx : -INFINITY, ib ? bmx : -INFINITY);
#pragma unroll
            for (int m = 1; m < UNITS; m *= 2) {
                mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, m));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, m));
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
    // Four rows a thread once that still leaves every SM a few warps.
    const bool many = (long long)tokens * ((rows + 4 * HL - 1) / (4 * HL)) >= 148 * 16;
    const int per = many ? 4 : 1, rb = (rows + per * HL - 1) / (per * HL);
    const unsigned grid = (unsigned)(((long long)tokens * rb + 7) / 8);
    return launch_after_previous(many ? sp_kv4_append<D, 4> : sp_kv4_append<D, 1>, dim3(grid), dim3(256), 0, st, pool, q,
                                 q_out, k, v, r, slots, tokens, q_heads, rb, err);
}

cudaError_t launch_kv4_append(int d, const Kv4Pool& pool, const Rows& q, const Rows& q_out, const Rows& k,
                              const Rows& v, const RotaryArgs& r, const int* slots, int tokens, int q_heads,
                              uint32_t* err, cudaStream_t st) {
    return d == 64 ? append<64>(pool, q, q_out, k, v, r, slots, tokens, q_heads, err, st)
                   : append<128>(pool, q, q_out, k, v, r, slots, tokens, q_heads, err, st);
}

// The values at given slots, zero + scale * n rounded once to bf16.  A thread
// reads one word (8 channels) and writes 16 bytes; bound by the bf16 rows it
// writes.
template <int D>
__global__ void __launch_bounds__(256) sp_kv4_read(const Kv4Pool pool, const int* __restrict__ slots, const Rows k,
                                                   const Rows v, int tokens, uint32_t* __restrict__ err) {
    constexpr int CH = D / 8, NG = D / KV4_GROUP;
    griddep_wait();
    griddep_launch_dependents();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int c = (int)(i % CH);
    const long long rowi = i / CH;
    const int rows = 2 * pool.kv_heads;
    const int row = (int)(rowi % rows);
    const long long t = rowi / rows;
    if (t >= tokens) return;
    const int slot = slots[t];
    const int page = slot >> pool.page_shift;
    if (page >= pool.pages) {
        if (c == 0 && row == 0) atomicOr(err + ERR_INDEX_WORD, ERR_INDEX);
        return;
    }
    const bool is_v = row >= pool.kv_heads;
    const int h = is_v ? row - pool.kv_heads : row;
    const Rows& dst = is_v ? v : k;
    float f[8] = {};
    if (slot >= 0) {
        const int in_page = slot & (pool.page_tokens - 1);
        const uint8_t* blk = pool.data + page * pool.page_stride + (long long)h * pool.block;
        const int half = pool.page_tokens * (D / 2), par = pool.page_tokens * NG * 4;
        const uint32_t w = *(const uint32_t*)(blk + (is_v ? half : 0) + in_page * (D / 2) + c * 4);
        const uint32_t p = ((const uint32_t*)(blk + 2 * half + (is_v ? par : 0)))[in_page * NG + c * 8 / KV4_GROUP];
        const float scale = __uint_as_float(p << 16), zero = __uint_as_float(p & 0xffff0000u);
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = __fmaf_rn(scale, (float)((w >> (4 * j)) & 15u), zero);
    }
    Chunk<0> o;
    o.from(f);
    o.store((void*)dst.data, t * dst.st + h * dst.sh + 8 * c);
}

cudaError_t launch_kv4_read(int d, const Kv4Pool& pool, const int* slots, const Rows& k, const Rows& v, int tokens,
                            uint32_t* err, cudaStream_t st) {
    const long long n = (long long)tokens * 2 * pool.kv_heads * (d / 8);
    const unsigned grid = (unsigned)((n + 255) / 256);
    return launch_after_previous(d == 64 ? sp_kv4_read<64> : sp_kv4_read<128>, dim3(grid), dim3(256), 0, st, pool, slots,
                                 k, v, tokens, err);
}

}  // namespace sp
