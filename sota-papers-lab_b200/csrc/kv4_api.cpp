// C ABI of the serving operators (include/splsage.h): rotary positions, the
// paged 4-bit KV cache and attention over it.  Arguments are checked before
// any launch; what only the device knows (positions, slots, lengths, page
// ids) is checked by the kernels and reported through the engine's error word.
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>
#include <new>

#include "kv4.h"
#include "sage_host.h"

using sp::cuda_fail;
using sp::fail;

struct spl_sage_kv4_ws {
    int device, head_dim;
    void* mem;
    size_t bytes;
};

namespace {

constexpr int64_t MOST = 1 << 30;  // tokens, keys and rows that 32-bit indices hold with room to add

int null_engine(const char* call) { return fail(SPL_SAGE_ERR_INVALID, "%s: NULL engine", call); }

// The last check before a launch: the engine's stream belongs to its device.
int check_device(const char* call, const spl_sage* s) {
    int dev = -1;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    if (dev != s->device)
        return fail(SPL_SAGE_ERR_INVALID, "%s: the current device is %d, the engine is on device %d", call, dev,
                    s->device);
    return SPL_SAGE_OK;
}

// A [token][head][D] tensor: its rows lie inside `len` elements, start on 16
// bytes and, for an output, do not overlap one another.
int check_rows(const char* what, const void* data, int64_t len, int64_t st, int64_t sh, int64_t tokens, int64_t heads,
               int64_t d, bool out) {
    if (st < 0 || sh < 0 || st % 8 || sh % 8)
        return fail(SPL_SAGE_ERR_INVALID,
                    "%s strides must be multiples of 8 elements: Strides { token: %lld, head: %lld }", what,
                    (long long)st, (long long)sh);
    if (!data) return fail(SPL_SAGE_ERR_INVALID, "%s is NULL", what);
    if ((uintptr_t)data % 16)
        return fail(SPL_SAGE_ERR_INVALID, "%s must start on a multiple of 8 elements (16 bytes)", what);
    if (st > INT64_MAX / MOST / 4 || sh > INT64_MAX / MOST / 4)
        return fail(SPL_SAGE_ERR_INVALID, "%s strides are too large", what);
    const int64_t need = (tokens - 1) * st + (heads - 1) * sh + d;
    if (len < need)
        return fail(SPL_SAGE_ERR_INVALID, "%s holds %lld elements, its shape and strides need %lld", what,
                    (long long)len, (long long)need);
    if (out && tokens > 1 && heads > 1 && st < (heads - 1) * sh + d && sh < (tokens - 1) * st + d)
        return fail(SPL_SAGE_ERR_INVALID, "%s: its rows overlap one another", what);
    if (out && ((tokens > 1 && st < d) || (heads > 1 && sh < d)))
        return fail(SPL_SAGE_ERR_INVALID, "%s: its rows overlap one another", what);
    return SPL_SAGE_OK;
}

bool ranges_meet(const void* a, int64_t an, const void* b, int64_t bn) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + (uintptr_t)bn && y < x + (uintptr_t)an;
}

int64_t extent(int64_t st, int64_t sh, int64_t tokens, int64_t heads, int64_t d) {
    return (tokens - 1) * st + (heads - 1) * sh + d;
}

// Whether a row of one [token][head][D] tensor overlaps a row of another (their
// rows may lie between one another's: heads of one packed projection).  Element
// sizes are the same.  Exact where the token strides are equal or one of them
// is never used; otherwise by the range that each tensor spans.
bool rows_meet(const void* a, int64_t ast, int64_t ash, int64_t ah, const void* b, int64_t bst, int64_t bsh, int64_t bh,
               int64_t tokens, int64_t d, int64_t size) {
    if (!ranges_meet(a, extent(ast, ash, tokens, ah, d) * size, b, extent(bst, bsh, tokens, bh, d) * size)) return false;
    if (tokens > 1 && ast != bst) return true;
    const int64_t off = (int64_t)((uintptr_t)b - (uintptr_t)a);  // in bytes
    // rows i, j of a and k, l of b are off + (k - i) * st + l * bsh - j * ash apart
    auto token_meets = [&](int64_t apart) {
        if (tokens == 1 || ast == 0) return apart > -d * size && apart < d * size;
        const int64_t st = ast * size, n = -(apart / st);  // the nearest token distances: n and one to either side
        for (int64_t k = n - 1; k <= n + 1; k++)
            if (k > -tokens && k < tokens && apart + k * st > -d * size && apart + k * st < d * size) return true;
        return false;
    };
    if (ash == bsh || ah == 1 || bh == 1) {
        const int64_t sh = (ah == 1 ? bsh : ash) * size;
        for (int64_t m = 1 - ah; m < bh; m++)
            if (token_meets(off + m * sh)) return true;
        return false;
    }
    if (ah * bh > 1 << 16) return true;
    for (int64_t j = 0; j < ah; j++)
        for (int64_t l = 0; l < bh; l++)
            if (token_meets(off + (l * bsh - j * ash) * size)) return true;
    return false;
}

int check_rotary(const char* call, const spl_sage_rotary* r, const int32_t* positions, int head_dim,
                 sp::RotaryArgs* out) {
    *out = sp::RotaryArgs{};
    if (!r) {
        if (positions) return fail(SPL_SAGE_ERR_INVALID, "%s: positions without a rotary table", call);
        return SPL_SAGE_OK;
    }
    if (!r->table || !positions) return fail(SPL_SAGE_ERR_INVALID, "%s: NULL rotary table or positions", call);
    if (r->rot_dim <= 0 || r->rot_dim > head_dim || r->rot_dim % 16)
        return fail(SPL_SAGE_ERR_INVALID,
                    "%s: %d rotated channels: a multiple of 16 up to the head dim (%d) is needed", call, r->rot_dim,
                    head_dim);
    if (r->positions <= 0 || r->positions > MOST)
        return fail(SPL_SAGE_ERR_INVALID, "%s: a table of %lld positions", call, (long long)r->positions);
    if ((uintptr_t)r->table % 16) return fail(SPL_SAGE_ERR_INVALID, "%s: the rotary table must start on 16 bytes", call);
    if ((uintptr_t)positions % 4) return fail(SPL_SAGE_ERR_INVALID, "%s: positions must start on 4 bytes", call);
    out->table = r->table;
    out->positions = positions;
    out->limit = (int)r->positions;
    out->rot = r->rot_dim;
    out->interleaved = r->interleaved ? 1 : 0;
    return SPL_SAGE_OK;
}

int64_t block_bytes(int head_dim, int page_tokens) {
    return (int64_t)page_tokens * (head_dim + head_dim / sp::KV4_GROUP * 8);
}

int check_cache(const char* call, const spl_sage_kv4* c, int head_dim, sp::Kv4Pool* out) {
    if (!c) return fail(SPL_SAGE_ERR_INVALID, "%s: NULL cache", call);
    const int64_t block = spl_sage_kv4_block_bytes(head_dim, c->page_tokens);
    if (!block)
        return fail(SPL_SAGE_ERR_INVALID, "%s: pages of %d tokens: 16, 32, 64 or 128 are supported", call,
                    c->page_tokens);
    if (!c->data) return fail(SPL_SAGE_ERR_INVALID, "%s: the cache is NULL", call);
    if ((uintptr_t)c->data % 16) return fail(SPL_SAGE_ERR_INVALID, "%s: the cache must start on 16 bytes", call);
    if (c->kv_heads <= 0 || c->kv_heads > 65535)
        return fail(SPL_SAGE_ERR_INVALID, "%s: %d KV heads", call, c->kv_heads);
    if (c->pages <= 0 || c->pages > 0x7fffffffLL || c->pages * c->page_tokens > 0x7fffffffLL)
        return fail(SPL_SAGE_ERR_INVALID, "%s: %lld pages of %d tokens: slots must fit 31 bits", call,
                    (long long)c->pages, c->page_tokens);
    if (c->page_stride % 16 || c->page_stride < block * c->kv_heads)
        return fail(SPL_SAGE_ERR_INVALID,
                    "%s: a page stride of %lld bytes: a multiple of 16, at least %lld (%d heads of %lld), is needed",
                    call, (long long)c->page_stride, (long long)(block * c->kv_heads), c->kv_heads, (long long)block);
    out->data = (uint8_t*)c->data;
    out->page_stride = c->page_stride;
    out->pages = (int)c->pages;
    out->page_tokens = c->page_tokens;
    out->page_shift = c->page_tokens == 16 ? 4 : c->page_tokens == 32 ? 5 : c->page_tokens == 64 ? 6 : 7;
    out->kv_heads = c->kv_heads;
    out->block = (int)block;
    return SPL_SAGE_OK;
}

int check_count(const char* call, const char* what, int64_t n, int64_t per) {
    if (n < 0 || per < 0 || n > MOST || per > 65535 || n * per > MOST)
        return fail(SPL_SAGE_ERR_INVALID, "%s: %lld %s of %lld heads", call, (long long)n, what, (long long)per);
    return SPL_SAGE_OK;
}

}  // namespace

extern "C" {

int spl_sage_device(const spl_sage* s) { return s ? s->device : -1; }

int spl_sage_rope_table(double base, int rot_dim, int64_t positions, const spl_sage_rope_scaling* scaling,
                        float* out) {
    const char* call = "spl_sage_rope_table";
    if (!out || positions <= 0 || rot_dim <= 0 || rot_dim > 128 || rot_dim % 16 || !(base > 1.0) || std::isinf(base))
        return fail(SPL_SAGE_ERR_INVALID, "%s: bad arguments", call);
    spl_sage_rope_scaling sc;
    memset(&sc, 0, sizeof sc);
    if (scaling) sc = *scaling;
    const int pairs = rot_dim / 2;
    const double pi2 = 6.283185307179586476925;
    if (sc.kind < SPL_SAGE_ROPE_PLAIN || sc.kind > SPL_SAGE_ROPE_BANDS)
        return fail(SPL_SAGE_ERR_INVALID, "%s: unknown scaling %d", call, sc.kind);
    if (sc.kind != SPL_SAGE_ROPE_PLAIN && !(sc.factor >= 1.0 && sc.factor <= 1e6))
        return fail(SPL_SAGE_ERR_INVALID, "%s: a scaling factor of %g: 1 to 1e6 is needed", call, sc.factor);
    if (sc.kind == SPL_SAGE_ROPE_YARN || sc.kind == SPL_SAGE_ROPE_BANDS) {
        if (sc.original <= 0) return fail(SPL_SAGE_ERR_INVALID, "%s: the original context must be given", call);
        if (!(sc.low > 0.0 && sc.high > sc.low && sc.high < 1e9))
            return fail(SPL_SAGE_ERR_INVALID, "%s: the bands need 0 < low < high, got %g and %g", call, sc.low,
                        sc.high);
        if (sc.kind == SPL_SAGE_ROPE_YARN && !(sc.attention >= 0.0 && sc.attention < 1e6))
            return fail(SPL_SAGE_ERR_INVALID, "%s: an attention factor of %g", call, sc.attention);
    }
    double freq[64], m = 1.0;
    double b = base;
    if (sc.kind == SPL_SAGE_ROPE_NTK) b = base * pow(sc.factor, (double)rot_dim / (rot_dim - 2));
    double lo = 0, hi = 0;
    if (sc.kind == SPL_SAGE_ROPE_YARN) {
        // the pair whose angle makes `high` (`low`) turns over the original context
        lo = fmax(floor(pairs * log(sc.original / (sc.high * pi2)) / log(base)), 0.0);
        hi = fmin(ceil(pairs * log(sc.original / (sc.low * pi2)) / log(base)), rot_dim - 1.0);
        m = sc.attention > 0.0 ? sc.attention : 0.1 * log(sc.factor) + 1.0;
    }
    for (int p = 0; p < pairs; p++) {
        const double f = pow(b, -(double)p / (double)pairs);
        freq[p] = f;
        double stretch = 0.0;  // the share of the pair's frequency that is divided by the factor
        if (sc.kind == SPL_SAGE_ROPE_LINEAR) stretch = 1.0;
        if (sc.kind == SPL_SAGE_ROPE_YARN) stretch = fmin(fmax((p - lo) / fmax(hi - lo, 1e-3), 0.0), 1.0);
        if (sc.kind == SPL_SAGE_ROPE_BANDS)
            stretch = 1.0 - fmin(fmax((sc.original * f / pi2 - sc.low) / (sc.high - sc.low), 0.0), 1.0);
        if (stretch > 0.0) freq[p] = f * (1.0 - stretch) + f / sc.factor * stretch;
    }
    for (int64_t t = 0; t < positions; t++)
        for (int p = 0; p < pairs; p++) {
            const double a = (double)t * freq[p];
            out[(t * pairs + p) * 2] = (float)(cos(a) * m);
            out[(t * pairs + p) * 2 + 1] = (float)(sin(a) * m);
        }
    return SPL_SAGE_OK;
}

int spl_sage_rope(spl_sage* s, int dtype, int64_t tokens, int64_t heads, spl_sage_tensor x, spl_sage_tensor_mut out,
                  const spl_sage_rotary* rotary, const int32_t* positions, int backward) {
    const char* call = "spl_sage_rope";
    if (!s) return null_engine(call);
    int rc;
    if (dtype != SPL_SAGE_BF16 && dtype != SPL_SAGE_F16 && dtype != SPL_SAGE_F32)
        return fail(SPL_SAGE_ERR_INVALID, "%s: unknown type %d", call, dtype);
    if ((rc = check_count(call, "tokens", tokens, heads))) return rc;
    if (!rotary) return fail(SPL_SAGE_ERR_INVALID, "%s: NULL rotary table", call);
    if (tokens == 0 || heads == 0) return SPL_SAGE_OK;
    sp::RotaryArgs r;
    if ((rc = check_rotary(call, rotary, positions, s->head_dim, &r))) return rc;
    const int64_t d = s->head_dim, size = dtype == SPL_SAGE_F32 ? 4 : 2;
    if ((rc = check_rows("x", x.data, x.len, x.token, x.head, tokens, heads, d, false))) return rc;
    if ((rc = check_rows("output", out.data, out.len, out.token, out.head, tokens, heads, d, true))) return rc;
    const bool in_place = x.data == out.data && x.token == out.token && x.head == out.head;
    if (!in_place && rows_meet(x.data, x.token, x.head, heads, out.data, out.token, out.head, heads, tokens, d, size))
        return fail(SPL_SAGE_ERR_INVALID, "%s: the output overlaps x without being x", call);
    if ((rc = check_device(call, s))) return rc;
    const cudaError_t e = sp::launch_rope(s->head_dim, dtype, {x.data, x.token, x.head}, {out.data, out.token, out.head},
                                          r, (int)tokens, (int)heads, backward != 0, s->sm_count, s->err,
                                          s->stream);
    if (e != cudaSuccess) return cuda_fail(e, "launch rope");
    return SPL_SAGE_OK;
}

int64_t spl_sage_kv4_block_bytes(int head_dim, int page_tokens) {
    if (head_dim != 64 && head_dim != 128) return 0;
    if (page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128) return 0;
    return block_bytes(head_dim, page_tokens);
}

int spl_sage_kv4_append(spl_sage* s, const spl_sage_kv4* cache, int64_t tokens, spl_sage_tensor k, spl_sage_tensor v,
                        const int32_t* slots, const spl_sage_rotary* rotary, const int32_t* positions,
                        int64_t q_heads, spl_sage_tensor q, spl_sage_tensor_mut q_out) {
    const char* call = "spl_sage_kv4_append";
    if (!s) return null_engine(call);
    int rc;
    sp::Kv4Pool pool;
    if ((rc = check_cache(call, cache, s->head_dim, &pool))) return rc;
    if ((rc = check_count(call, "tokens", tokens, q_heads < 0 ? -1 : q_heads + 2 * (int64_t)pool.kv_heads))) return rc;
    if (tokens == 0) return SPL_SAGE_OK;
    sp::RotaryArgs r;
    if ((rc = check_rotary(call, rotary, positions, s->head_dim, &r))) return rc;
    if (!slots || (uintptr_t)slots % 4) return fail(SPL_SAGE_ERR_INVALID, "%s: slots must be given, on 4 bytes", call);
    const int64_t d = s->head_dim, hk = pool.kv_heads;
    if ((rc = check_rows("K", k.data, k.len, k.token, k.head, tokens, hk, d, false))) return rc;
    if ((rc = check_rows("V", v.data, v.len, v.token, v.head, tokens, hk, d, false))) return rc;
    if (q_heads) {
        if (!rotary) return fail(SPL_SAGE_ERR_INVALID, "%s: Q is taken to be rotated, but there is no rotary table", call);
        if ((rc = check_rows("Q", q.data, q.len, q.token, q.head, tokens, q_heads, d, false))) return rc;
        if ((rc = check_rows("Q output", q_out.data, q_out.len, q_out.token, q_out.head, tokens, q_heads, d, true)))
            return rc;
        const bool in_place = q.data == q_out.data && q.token == q_out.token && q.head == q_out.head;
        auto meets = [&](const spl_sage_tensor& x, int64_t heads) {
            return rows_meet(q_out.data, q_out.token, q_out.head, q_heads, x.data, x.token, x.head, heads, tokens, d, 2);
        };
        if ((!in_place && meets(q, q_heads)) || meets(k, hk) || meets(v, hk))
            return fail(SPL_SAGE_ERR_INVALID, "%s: the Q output overlaps an input without being Q", call);
    }
    if ((rc = check_device(call, s))) return rc;
    const cudaError_t e = sp::launch_kv4_append(
        s->head_dim, pool, {q.data, q.token, q.head}, {q_out.data, q_out.token, q_out.head}, {k.data, k.token, k.head},
        {v.data, v.token, v.head}, r, slots, (int)tokens, (int)q_heads, s->sm_count, s->err,
        s->stream);
    if (e != cudaSuccess) return cuda_fail(e, "launch the cache append");
    return SPL_SAGE_OK;
}

int spl_sage_kv4_read(spl_sage* s, const spl_sage_kv4* cache, int64_t tokens, const int32_t* slots,
                      spl_sage_tensor_mut k, spl_sage_tensor_mut v) {
    const char* call = "spl_sage_kv4_read";
    if (!s) return null_engine(call);
    int rc;
    sp::Kv4Pool pool;
    if ((rc = check_cache(call, cache, s->head_dim, &pool))) return rc;
    if ((rc = check_count(call, "tokens", tokens, 2 * (int64_t)pool.kv_heads))) return rc;
    if (tokens == 0) return SPL_SAGE_OK;
    if (!slots || (uintptr_t)slots % 4) return fail(SPL_SAGE_ERR_INVALID, "%s: slots must be given, on 4 bytes", call);
    const int64_t d = s->head_dim, hk = pool.kv_heads;
    if ((rc = check_rows("K", k.data, k.len, k.token, k.head, tokens, hk, d, true))) return rc;
    if ((rc = check_rows("V", v.data, v.len, v.token, v.head, tokens, hk, d, true))) return rc;
    if (rows_meet(k.data, k.token, k.head, hk, v.data, v.token, v.head, hk, tokens, d, 2))
        return fail(SPL_SAGE_ERR_INVALID, "%s: K and V overlap", call);
    const int64_t pool_bytes = (pool.pages - 1) * pool.page_stride + (int64_t)pool.kv_heads * pool.block;
    if (ranges_meet(k.data, extent(k.token, k.head, tokens, hk, d) * 2, pool.data, pool_bytes) ||
        ranges_meet(v.data, extent(v.token, v.head, tokens, hk, d) * 2, pool.data, pool_bytes))
        return fail(SPL_SAGE_ERR_INVALID, "%s: an output overlaps the cache", call);
    if ((rc = check_device(call, s))) return rc;
    const cudaError_t e = sp::launch_kv4_read(s->head_dim, pool, slots, {k.data, k.token, k.head},
                                              {v.data, v.token, v.head}, (int)tokens, s->err, s->stream);
    if (e != cudaSuccess) return cuda_fail(e, "launch the cache read");
    return SPL_SAGE_OK;
}

int spl_sage_kv4_ws_create(spl_sage* s, spl_sage_kv4_ws** out) {
    const char* call = "spl_sage_kv4_ws_create";
    if (!out) return fail(SPL_SAGE_ERR_INVALID, "%s: out is NULL", call);
    *out = nullptr;
    if (!s) return null_engine(call);
    const int rc = check_device(call, s);
    if (rc) return rc;
    spl_sage_kv4_ws* ws = new (std::nothrow) spl_sage_kv4_ws;
    if (!ws) return fail(SPL_SAGE_ERR_CUDA, "%s: out of host memory", call);
    ws->device = s->device;
    ws->head_dim = s->head_dim;
    ws->bytes = sp::kv4_scratch_bytes(s->head_dim, s->sm_count);
    cudaError_t e = cudaMalloc(&ws->mem, ws->bytes);
    if (e == cudaSuccess) {
        e = cudaMemsetAsync(ws->mem, 0, sp::KV4_COUNTS, s->stream);
        if (e == cudaSuccess) e = cudaStreamSynchronize(s->stream);  // another engine's stream may use it first
        if (e != cudaSuccess) cudaFree(ws->mem);
    }
    if (e != cudaSuccess) {
        delete ws;
        return cuda_fail(e, "allocate the cache attention's workspace");
    }
    *out = ws;
    return SPL_SAGE_OK;
}

void spl_sage_kv4_ws_destroy(spl_sage_kv4_ws* ws) {
    if (!ws) return;
    cudaFree(ws->mem);
    delete ws;
}

int64_t spl_sage_kv4_ws_bytes(const spl_sage_kv4_ws* ws) { return ws ? (int64_t)ws->bytes : 0; }

int spl_sage_kv4_attend(spl_sage* s, spl_sage_kv4_ws* ws, const spl_sage_kv4* cache, const spl_sage_kv4_shape* shape,
                        spl_sage_tensor q, const int32_t* q_start, const int32_t* kv_len, const int32_t* pages,
                        const spl_sage_options* opts, spl_sage_tensor_mut out, float* lse) {
    const char* call = "spl_sage_kv4_attend";
    if (!s) return null_engine(call);
    int rc;
    if (!ws || !shape) return fail(SPL_SAGE_ERR_INVALID, "%s: NULL workspace or shape", call);
    if (ws->head_dim != s->head_dim || ws->device != s->device)
        return fail(SPL_SAGE_ERR_INVALID, "%s: the workspace was made for head dim %d on device %d, the engine is %d on %d",
                    call, ws->head_dim, ws->device, s->head_dim, s->device);
    sp::Kv4Attend a{};
    if ((rc = check_cache(call, cache, s->head_dim, &a.pool))) return rc;
    const spl_sage_kv4_shape& sh = *shape;
    const int64_t hk = a.pool.kv_heads, d = s->head_dim;
    if ((rc = check_count(call, "query tokens", sh.tokens, sh.heads))) return rc;
    if (sh.heads <= 0 || sh.heads % hk != 0)
        return fail(SPL_SAGE_ERR_INVALID, "heads (%lld) must be a multiple of kv_heads (%lld)", (long long)sh.heads,
                    (long long)hk);
    if (sh.batch < 0 || sh.batch > MOST) return fail(SPL_SAGE_ERR_INVALID, "%s: %lld sequences", call, (long long)sh.batch);
    if (sh.batch == 0 || sh.tokens == 0) return SPL_SAGE_OK;
    if (sh.max_q <= 0 || sh.max_q > MOST || sh.max_q * sh.heads > MOST)
        return fail(SPL_SAGE_ERR_INVALID, "%s: at most %lld queries a sequence", call, (long long)sh.max_q);
    if (sh.max_pages <= 0 || sh.max_pages > MOST || sh.max_pages * a.pool.page_tokens > MOST)
        return fail(SPL_SAGE_ERR_INVALID, "%s: %lld pages a sequence", call, (long long)sh.max_pages);
    if (sh.window < 0 || sh.window > MOST)
        return fail(SPL_SAGE_ERR_INVALID, "%s: a window of %d keys", call, sh.window);
    if (!kv_len || !pages || (uintptr_t)kv_len % 4 || (uintptr_t)pages % 4 || (uintptr_t)q_start % 4)
        return fail(SPL_SAGE_ERR_INVALID, "%s: lengths and pages must be given, on 4 bytes", call);
    if (!q_start && (sh.max_q != 1 || sh.tokens < sh.batch))
        return fail(SPL_SAGE_ERR_INVALID,
                    "%s: without q_start every sequence has one query: %lld query tokens for %lld sequences, max_q %lld",
                    call, (long long)sh.tokens, (long long)sh.batch, (long long)sh.max_q);
    if ((uintptr_t)lse % 4) return fail(SPL_SAGE_ERR_INVALID, "%s: lse must start on 4 bytes", call);
    if ((rc = check_rows("Q", q.data, q.len, q.token, q.head, sh.tokens, sh.heads, d, false))) return rc;
    if ((rc = check_rows("output", out.data, out.len, out.token, out.head, sh.tokens, sh.heads, d, true))) return rc;
    if (rows_meet(q.data, q.token, q.head, sh.heads, out.data, out.token, out.head, sh.heads, sh.tokens, d, 2))
        return fail(SPL_SAGE_ERR_INVALID, "%s: the output overlaps Q", call);
    float scale = 1.0f / sqrtf((float)d);
    if (opts) {
        if (opts->qk_norm_params) return fail(SPL_SAGE_ERR_INVALID, "%s: the QK LayerNorm is not part of it", call);
        if (opts->has_softmax_scale) scale = opts->softmax_scale;
    }
    if (!(scale >= 1e-10f && scale <= 1e10f))
        return fail(SPL_SAGE_ERR_INVALID, "%s: a softmax scale of %g: 1e-10 to 1e10 is needed", call, scale);
    a.q = {q.data, q.token, q.head};
    a.out = {out.data, out.token, out.head};
    a.lse = lse;
    a.q_start = q_start;
    a.kv_len = kv_len;
    a.pages = pages;
    a.max_pages = (int)sh.max_pages;
    a.batch = (int)sh.batch;
    a.heads = (int)sh.heads;
    a.group = (int)(sh.heads / hk);
    if (a.group > 1) {
        while ((2 << a.group_shift) < a.group) a.group_shift++;
        a.group_mul = (uint32_t)(((uint64_t)1 << (32 + a.group_shift)) / a.group + 1);
    }
    a.tokens = (int)sh.tokens;
    a.max_q = (int)sh.max_q;
    a.causal = sh.causal ? 1 : 0;
    a.window = sh.window;
    a.c = scale * 1.44269504088896340736f;
    a.scratch = ws->mem;
    a.err = s->err;
    if ((rc = check_device(call, s))) return rc;
    const cudaError_t e = sp::launch_kv4_attend(s->head_dim, a, s->sm_count - s->reserved_sms,
                                                s->reserved_sms > 0, s->stream);
    if (e != cudaSuccess) return cuda_fail(e, "launch the cache attention");
    return SPL_SAGE_OK;
}

}  // extern "C"
