// Rotary positions on [token][head][D] rows: y = R(position) x on the first
// `rot` channels of each head, the rest copied (rotary.cuh has the layout of
// the pairs); backward: y = R(position)^T x.
//
// Bound by memory: every element is read and written once; the 8192-token bf16
// case runs at 0.91 of the measured copy rate.  A thread keeps
// the cosines and sines of its 8 pairs in registers and applies them to HPT
// heads of its token, whose loads are all issued before the first is used:
// with one head a thread the table (64 bytes for 32 bytes of bf16 channels)
// would pass the L1 twice as often as the data.
#include "rotary.cuh"
#include "sage_kernels.h"

namespace sp {

// A warp's lanes are D/16 units times 512/D heads, so that a warp's access is
// 512/D whole rows.  blockIdx.x * blockDim.y + threadIdx.y counts (token,
// head block).
template <int D, int DT, int HPT>
__global__ void __launch_bounds__(256) sp_rope(const Rows x, const Rows out, const RotaryArgs r, int tokens, int heads,
                                               int head_blocks, int backward, uint32_t* __restrict__ err) {
    constexpr int UNITS = D / 16, HL = 32 / UNITS;
    griddep_wait();
    griddep_launch_dependents();
    const long long w = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int t = (int)(w / head_blocks), hb = (int)(w % head_blocks);
    if (t >= tokens) return;
    const int lane = threadIdx.x & 31, u = lane % UNITS;
    const int h0 = hb * HL * HPT + lane / UNITS;
    const Unit un = unit_at(u, r);
    const int pos = r.positions[t];
    if (pos < 0 || pos >= r.limit) {  // the row is left as it was
        if (lane == 0) atomicOr(err + ERR_INDEX_WORD, ERR_INDEX);
        return;
    }
    Chunk<DT> lo[HPT], hi[HPT];
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        const int h = h0 + i * HL;
        if (h < heads) {
            const long long at = t * x.st + h * x.sh;
            lo[i].load(x.data, at + un.c0);
            hi[i].load(x.data, at + un.c1);
        }
    }
    float cs[16];
    if (un.turns) load_angles(r, pos, u, cs);
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        const int h = h0 + i * HL;
        if (h >= heads) continue;
        if (un.turns) {
            float a[8], b[8];
            lo[i].to(a);
            hi[i].to(b);
            turn(a, b, cs, r.interleaved, backward);
            lo[i].from(a);
            hi[i].from(b);
        }
        const long long at = t * out.st + h * out.sh;
        lo[i].store((void*)out.data, at + un.c0);
        hi[i].store((void*)out.data, at + un.c1);
    }
}

template <int D, int DT>
static cudaError_t rope(const Rows& x, const Rows& out, const RotaryArgs& r, int tokens, int heads, bool backward,
                        int sms, uint32_t* err, cudaStream_t st) {
    constexpr int HL = 512 / D;  // heads a warp covers at once
    // Several heads a thread once that still leaves every SM a few warps: 4 of
    // a 16-bit type (8192 x 40 x 128 bf16: 29.2 us, 5.89 TB/s, with 1 41.6), 2
    // in f32, whose loads are twice as many (4099 x 32 x 64: 14.5 us, with 4 16.3).
    constexpr int MANY = DT == 2 ? 2 : 4;
    const bool many = (long long)tokens * ((heads + MANY * HL - 1) / (MANY * HL)) >= sms * 16;
    const int per = many ? MANY : 1, hb = (heads + per * HL - 1) / (per * HL);
    const long long warps = (long long)tokens * hb;
    const unsigned grid = (unsigned)((warps + 7) / 8);
    return launch_after_previous(many ? sp_rope<D, DT, MANY> : sp_rope<D, DT, 1>, dim3(grid), dim3(256), 0, st, x, out, r,
                                 tokens, heads, hb, backward, err);
}

cudaError_t launch_rope(int d, int dtype, const Rows& x, const Rows& out, const RotaryArgs& r, int tokens, int heads,
                        bool backward, int sms, uint32_t* err, cudaStream_t st) {
    if (d == 64)
        return dtype == 0   ? rope<64, 0>(x, out, r, tokens, heads, backward, sms, err, st)
               : dtype == 1 ? rope<64, 1>(x, out, r, tokens, heads, backward, sms, err, st)
                            : rope<64, 2>(x, out, r, tokens, heads, backward, sms, err, st);
    return dtype == 0   ? rope<128, 0>(x, out, r, tokens, heads, backward, sms, err, st)
           : dtype == 1 ? rope<128, 1>(x, out, r, tokens, heads, backward, sms, err, st)
                        : rope<128, 2>(x, out, r, tokens, heads, backward, sms, err, st);
}

}  // namespace sp
