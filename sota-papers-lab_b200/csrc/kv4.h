// The serving operators (rotary positions, the paged 4-bit KV cache and
// attention over it): what their kernels and their host code share.
//
// The cache is a pool of pages, each holding `page_tokens` (P) consecutive
// tokens of one sequence.  One page of one KV head is a block of P * (D + D/8)
// bytes:
//   K values  [P][D/2]      two channels a byte, channel 2j in its low half
//   V values  [P][D/2]
//   K params  [P][D/64][2]  bf16 (scale, zero) per 64 channels of a token
//   V params  [P][D/64][2]
// and stands for zero + scale * n, n = 0..15.  Scale and zero per token (not
// per channel over tokens), so that a token is appended without touching any
// other; bf16, whose range is that of the tensors (no overflow), and n is
// chosen after both are rounded, so that their rounding costs only a little
// of the range's ends.  The block is contiguous: attention reads a page of a
// head as one run of memory.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace sp {

constexpr int KV4_GROUP = 64;  // channels per scale

struct Kv4Pool {
    uint8_t* data;
    long long page_stride;  // bytes from page to page
    int pages;
    int page_tokens, page_shift;  // P = 1 << page_shift
    int kv_heads;
    int block;  // bytes of one page of one head
};

// Rows of a [token][head][D] tensor, strides in elements.
struct Rows {
    const void* data;
    long long st, sh;
};

struct RotaryArgs {
    const float* table;  // [positions][rot/2][2]; nullptr: no rotation
    const int* positions;
    int limit;  // positions in the table
    int rot, interleaved;
};

// dtype: 0 bf16, 1 f16, 2 f32
cudaError_t launch_rope(int d, int dtype, const Rows& x, const Rows& out, const RotaryArgs& r, int tokens, int heads,
                        bool backward, int sms, uint32_t* err, cudaStream_t st);
cudaError_t launch_kv4_append(int d, const Kv4Pool& pool, const Rows& q, const Rows& q_out, const Rows& k,
                              const Rows& v, const RotaryArgs& r, const int* slots, int tokens, int q_heads, int sms,
                              uint32_t* err, cudaStream_t st);
cudaError_t launch_kv4_read(int d, const Kv4Pool& pool, const int* slots, const Rows& k, const Rows& v, int tokens,
                            uint32_t* err, cudaStream_t st);

struct Kv4Attend {
    Kv4Pool pool;
    Rows q, out;
    float* lse;          // [tokens][heads] natural log, or nullptr
    const int* q_start;  // [batch + 1], or nullptr: sequence b's one query is row b
    const int* kv_len;   // [batch]
    const int* pages;    // [batch][max_pages]
    int max_pages;
    int batch, heads, group, tokens, max_q;  // group = heads / kv_heads
    uint32_t group_mul;   // n / group = (n * group_mul) >> (32 + group_shift) for n < 2^31; 0: group is 1
    int group_shift;
    int causal, window;
    float c;  // softmax scale * log2(e)
    void* scratch;        // kv4_scratch_bytes
    uint32_t* done;       // (set by the launch) [CTAs] pieces of a split tile that are finished, zero between calls
    float2* part_ml;      // (set by the launch) [2 * CTAs][cols] running maximum (log2) and sum of split tiles
    float* part_o;        // (set by the launch) [2 * CTAs][cols][D] their outputs
    uint32_t* err;
};

// Scratch of one attend call: partial outputs of at most two pieces per CTA,
// behind counts that must be zero before the first call.
constexpr size_t KV4_COUNTS = 8192;  // bytes
size_t kv4_scratch_bytes(int d, int sms);
// On `sms` SMs; `alone`: the others stay free (no CTA shares an SM with another).
cudaError_t launch_kv4_attend(int d, const Kv4Attend& a, int sms, bool alone, cudaStream_t st);
// The same for many query rows (kv4_prompt.cu).
size_t kv4_prompt_scratch_bytes(int d, int sms);
cudaError_t launch_kv4_prompt(int d, const Kv4Attend& a, int sms, cudaStream_t st);

}  // namespace sp
