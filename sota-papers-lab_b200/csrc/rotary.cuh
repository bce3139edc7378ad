// Rotary positions on 16 channels at a time, shared by the rope and the
// cache append kernels.
//
// One unit is 16 channels: 8 pairs (a, b) that rotate by 8 consecutive
// angles, or 16 channels that pass unrotated.  With R rotated channels of D
// (both multiples of 16), units 0 .. R/16 - 1 rotate pairs 8u .. 8u + 7:
// half layout: channels 8u + i with R/2 + 8u + i; interleaved: 16u + 2i with
// 16u + 2i + 1.  Units from R/16 on hold channels 16u .. 16u + 15.  Either
// way a unit is two 8-channel chunks, each 16 bytes of a 16-bit type.
#pragma once

#include <cuda_fp16.h>

#include "kv4.h"
#include "sage_dev.cuh"

namespace sp {

// Bit of the device error word: an index read from device memory (a
// position, slot, page or length) was out of range (SPL_SAGE_DEVERR_INDEX).
// In the word beside the one that the kernels' waits look at: a wait gives up
// when another kernel's wait has, but not because of an index.
constexpr uint32_t ERR_INDEX = 1u << 2;
constexpr int ERR_INDEX_WORD = 1;

struct Unit {
    int c0, c1;  // first channel of each chunk
    bool turns;  // rotated
};

__device__ __forceinline__ Unit unit_at(int u, const RotaryArgs& r) {
    Unit x;
    x.turns = r.table != nullptr && 16 * u < r.rot;
    const bool halves = x.turns && !r.interleaved;
    x.c0 = halves ? 8 * u : 16 * u;
    x.c1 = halves ? r.rot / 2 + 8 * u : 16 * u + 8;
    return x;
}

// cos and sin of the unit's 8 pairs at one position.
__device__ __forceinline__ void load_angles(const RotaryArgs& r, int position, int u, float (&cs)[16]) {
    const float4* t = (const float4*)(r.table + (long long)position * r.rot + 16 * u);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float4 v = __ldg(t + i);
        cs[4 * i] = v.x; cs[4 * i + 1] = v.y; cs[4 * i + 2] = v.z; cs[4 * i + 3] = v.w;
    }
}

// y = (a c - b s, b c + a s) on the unit's 16 channels (lo, hi: its chunks).
// Every product and sum is rounded on its own: no fused multiply-add, so that
// the same formula written with separate operations gives the same bits (the
// 4-bit values that follow depend on them).  (Not as packed f32x2 products and
// sums, which are fused all the same.)  `back`: the transposed rotation (the
// gradient), s with the other sign.
__device__ __forceinline__ void turn(float (&lo)[8], float (&hi)[8], const float (&cs)[16], bool interleaved,
                                     bool back) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float c = cs[2 * i], s = back ? -cs[2 * i + 1] : cs[2 * i + 1];
        if (interleaved) {
            float* x = i < 4 ? lo : hi;
            const int j = 2 * (i & 3);
            const float a = x[j], b = x[j + 1];
            x[j] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
            x[j + 1] = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
        } else {
            const float a = lo[i], b = hi[i];
            lo[i] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
            hi[i] = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
        }
    }
}

// 8 channels of a type, as they lie in memory.
template <int DT>
struct Chunk {
    uint4 w;
    __device__ __forceinline__ void load(const void* p, long long at) { w = *((const uint4*)((const uint16_t*)p + at)); }
    __device__ __forceinline__ void store(void* p, long long at) const { *((uint4*)((uint16_t*)p + at)) = w; }
    __device__ __forceinline__ void to(float (&f)[8]) const {
        if constexpr (DT == 0) {
            unpack_bf16x8(w, f);
        } else {
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 t = __half22float2(*(const __half2*)&v[i]);
                f[2 * i] = t.x; f[2 * i + 1] = t.y;
            }
        }
    }
    __device__ __forceinline__ void from(const float (&f)[8]) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == 0) {
                v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
            } else {
                const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                v[i] = *(const uint32_t*)&h;
            }
        }
        w = make_uint4(v[0], v[1], v[2], v[3]);
    }
};

template <>
struct Chunk<2> {
    float4 a, b;
    __device__ __forceinline__ void load(const void* p, long long at) {
        a = ((const float4*)((const float*)p + at))[0];
        b = ((const float4*)((const float*)p + at))[1];
    }
    __device__ __forceinline__ void store(void* p, long long at) const {
        ((float4*)((float*)p + at))[0] = a;
        ((float4*)((float*)p + at))[1] = b;
    }
    __device__ __forceinline__ void to(float (&f)[8]) const {
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
    __device__ __forceinline__ void from(const float (&f)[8]) {
        a = make_float4(f[0], f[1], f[2], f[3]);
        b = make_float4(f[4], f[5], f[6], f[7]);
    }
};

}  // namespace sp
