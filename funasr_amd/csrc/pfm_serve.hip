// C entry points of token-by-token decoding over a paged key / value cache (include/pfm.h): argument checks and
// launches. The kernels are in k_paged.hip and k_sample.hip.
#include <math.h>

#include <algorithm>
#include <initializer_list>
#include <string>
#include <utility>

#include "../../include/pfm.h"
#include "pfm_serve.h"

int pfm_fail(int code, const char* msg);                                        // pfm_api.hip
int pfm_check_dev_ops(const char* fn, const PfmDevOp* ops, int n);

namespace {

int fail(const char* fn, int code, const char* what) { return pfm_fail(code, (std::string(fn) + ": " + what).c_str()); }

// No C++ exception leaves a C entry point.
template <typename F> int guarded(const char* fn, F f) noexcept {
    try {
        return f();
    } catch (...) {
        try {
            return fail(fn, PFM_E_NOMEM, "host memory");
        } catch (...) {
            return PFM_E_NOMEM;
        }
    }
}

int elem_bytes(int dtype) { return dtype == PFM_F32 ? 4 : 2; }
bool is_dtype(int dtype) { return dtype == PFM_F32 || dtype == PFM_BF16 || dtype == PFM_F16; }

// pointers and strides that let a row be read 16 bytes at a time
bool wide(const void* p, int dtype, const int64_t* st, int n) {
    const int per = 16 / elem_bytes(dtype);
    if ((uintptr_t)p & 15) return false;
    for (int i = 0; i < n; ++i)
        if (st[i] % per || st[i] < 0) return false;
    return true;
}

int check_cache(const char* fn, const pfm_paged_kv* c, PagedKv& o) {
    if (!c) return fail(fn, PFM_E_ARG, "no cache given");
    if (!is_dtype(c->dtype)) return fail(fn, PFM_E_ARG, "dtype must be PFM_F32, PFM_BF16 or PFM_F16");
    if (c->batch < 0 || c->tokens < 0 || c->pages < 0 || c->table_width < 0)
        return fail(fn, PFM_E_ARG, "negative size");
    if (c->batch > 1 << 24 || c->tokens > 1 << 24) return fail(fn, PFM_E_ARG, "batch and tokens must not pass 2^24");
    if (c->page_size < 1 || c->heads < 1 || c->heads > 65535) return fail(fn, PFM_E_ARG, "page_size and heads must be at least 1, heads at most 65535");
    if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8)
        return fail(fn, PFM_E_ARG, "head_dim must be a multiple of 8 up to 256");
    // (a position is at least -tokens; less a window it stays in 32 bits)
    if ((long long)c->table_width * c->page_size > (1ll << 31) - (1 << 25))
        return fail(fn, PFM_E_ARG, "table_width * page_size must not pass 2^31 - 2^25");
    if (!c->cu_q && c->tokens != c->batch)
        return fail(fn, PFM_E_ARG, "without cu_q every sequence has one new token: tokens must equal batch");
    if (c->batch > 0 && c->tokens > 0) {
        if ((c->pages && (!c->k || !c->v)) || (c->table_width && !c->block_table) || !c->kv_len)
            return fail(fn, PFM_E_ARG, "null operand");
        if (c->table_stride < c->table_width) return fail(fn, PFM_E_ARG, "table_stride is smaller than table_width");
        if (!wide(c->k, c->dtype, c->k_stride, 3) || !wide(c->v, c->dtype, c->v_stride, 3))
            return fail(fn, PFM_E_ARG, "k and v pages must be aligned to 16 bytes, their strides multiples of 16 bytes");
    }
    o.k = (char*)c->k;
    o.v = (char*)c->v;
    const int per = 16 / elem_bytes(c->dtype);
    for (int i = 0; i < 3; ++i) {
        if (c->k_stride[i] / per > 0xffffffffll || c->v_stride[i] / per > 0xffffffffll)
            return fail(fn, PFM_E_ARG, "strides of the pages must stay under 64 GiB");
        o.ks[i] = (uint32_t)(c->k_stride[i] / per);
        o.vs[i] = (uint32_t)(c->v_stride[i] / per);
    }
    if (c->pages > 0x7fffffffll) return fail(fn, PFM_E_ARG, "at most 2^31 - 1 pages");
    o.pages = c->pages;
    o.table = c->block_table;
    o.table_stride = c->table_stride;
    o.width = c->table_width;
    o.page = c->page_size;
    o.heads = c->heads;
    o.dim = c->head_dim;
    o.batch = c->batch;
    o.tokens = c->tokens;
    o.by_page = fast_div((uint32_t)c->page_size);
    o.kv_len = c->kv_len;
    o.cu_q = c->cu_q;
    return PFM_OK;
}

int check_rows(const char* fn, const char* name, const pfm_rows* r, int dtype, Rows& o) {
    if (!r || !r->p) return fail(fn, PFM_E_ARG, (std::string("null operand '") + name + "'").c_str());
    const int64_t st[2] = {r->token_stride, r->head_stride};
    if (!wide(r->p, dtype, st, 2))
        return fail(fn, PFM_E_ARG, (std::string("'") + name + "' must be aligned to 16 bytes, its strides multiples of 16 bytes").c_str());
    o = Rows{(char*)r->p, r->token_stride, r->head_stride};
    return PFM_OK;
}

// Places that are written must not lie on each other: in the order of their strides, each dimension longer than one
// steps over all that the ones before it reach.
bool apart(std::initializer_list<std::pair<int64_t, int64_t>> extent_stride, int dim) {
    std::pair<int64_t, int64_t> d[3];      // (stride, extent)
    int n = 0;
    for (const auto& e : extent_stride)
        if (e.first > 1) d[n++] = {e.second, e.first};
    std::sort(d, d + n);
    __int128 reach = dim;
    for (int i = 0; i < n; ++i) {
        if (d[i].first < reach) return false;
        reach += (__int128)d[i].first * (d[i].second - 1);
    }
    return true;
}

int hip(const char* fn, hipError_t e) { return e == hipSuccess ? PFM_OK : fail(fn, PFM_E_HIP, hipGetErrorString(e)); }

#define TRY(x)                    \
    do {                          \
        const int _rc = (x);      \
        if (_rc) return _rc;      \
    } while (0)

long long attention_ws(const PagedAttnArgs& a) {
    const long long rows = std::max(a.splits > 1 ? a.splits * a.rows_part.rows : 0, a.tile_splits > 1 ? a.tile_splits * a.tile_part.rows : 0);
    return rows * (a.c.dim + 2) * 4;
}

}  // namespace

extern "C" {

int pfm_op_kv_append(void* stream, const pfm_paged_kv* cache, const pfm_rows* k, const pfm_rows* v, const pfm_rows* q,
                     const pfm_rows* q_out, int q_heads, const float* inv_freq, int rot_dim, int interleaved,
                     const int32_t* pos) {
    static const char fn[] = "pfm_op_kv_append";
    return guarded(fn, [&]() -> int {
        AppendArgs a{};
        TRY(check_cache(fn, cache, a.c));
        if (q_heads < 0 || q_heads > 65535) return fail(fn, PFM_E_ARG, "q_heads out of range");
        if (inv_freq && (rot_dim < 16 || rot_dim % 16 || rot_dim > cache->head_dim))
            return fail(fn, PFM_E_ARG, "rot_dim must be a multiple of 16 up to head_dim");
        if (cache->batch == 0 || cache->tokens == 0) return PFM_OK;
        TRY(check_rows(fn, "k", k, cache->dtype, a.k));
        TRY(check_rows(fn, "v", v, cache->dtype, a.v));
        if (q_heads) {
            TRY(check_rows(fn, "q", q, cache->dtype, a.q));
            TRY(check_rows(fn, "q_out", q_out, cache->dtype, a.qo));
            if (!apart({{cache->tokens, a.qo.ts}, {q_heads, a.qo.hs}}, a.c.dim))
                return fail(fn, PFM_E_ARG, "q_out overlaps itself");
        }
        for (const int64_t* st : {cache->k_stride, cache->v_stride})
            if (!apart({{a.c.pages, st[0]}, {a.c.page, st[1]}, {a.c.heads, st[2]}}, a.c.dim))
                return fail(fn, PFM_E_ARG, "the pages overlap themselves");
        a.q_heads = q_heads;
        a.inv_freq = inv_freq;
        a.rot = inv_freq ? rot_dim : 0;
        a.interleaved = interleaved ? 1 : 0;
        a.pos = pos;
        const PfmDevOp ops[] = {{"k", a.k.p}, {"v", a.v.p}, {"q", a.q.p}, {"q_out", a.qo.p}, {"k_pages", a.c.k},
                                {"v_pages", a.c.v}, {"block_table", a.c.table}, {"kv_len", a.c.kv_len},
                                {"cu_q", a.c.cu_q}, {"inv_freq", inv_freq}, {"pos", pos}};
        TRY(pfm_check_dev_ops(fn, ops, (int)(sizeof(ops) / sizeof(ops[0]))));
        return hip(fn, pfm_kv_append(cache->dtype, a, (hipStream_t)stream));
    });
}

int64_t pfm_paged_attention_ws_bytes(const pfm_paged_kv* cache, int q_heads) {
    if (!cache || cache->heads < 1 || q_heads < cache->heads || cache->batch < 1 || cache->tokens < 1) return 0;
    PagedAttnArgs a{};
    a.c.batch = cache->batch;
    a.c.tokens = cache->tokens;
    a.c.heads = cache->heads;
    a.c.dim = cache->head_dim;
    a.c.width = cache->table_width;
    a.c.page = cache->page_size;
    a.c.cu_q = cache->cu_q;
    a.q_heads = q_heads;
    a.group = q_heads / cache->heads;
    pfm_paged_attention_plan(cache->dtype, a);
    return attention_ws(a);
}

int pfm_op_paged_attention(void* stream, const pfm_paged_kv* cache, const pfm_rows* q, const pfm_rows* out, int q_heads,
                           float scale, int causal, int window, void* ws, int64_t ws_bytes) {
    static const char fn[] = "pfm_op_paged_attention";
    return guarded(fn, [&]() -> int {
        PagedAttnArgs a{};
        TRY(check_cache(fn, cache, a.c));
        if (q_heads < 1 || q_heads % cache->heads) return fail(fn, PFM_E_ARG, "q_heads must be a multiple of the cache's heads");
        if (window < 0) return fail(fn, PFM_E_ARG, "window must not be negative (0: no window)");
        if (!(fabsf(scale) < INFINITY)) return fail(fn, PFM_E_ARG, "scale must be finite");
        if ((long long)cache->tokens * (q_heads / cache->heads) > 0x7fffff00ll)
            return fail(fn, PFM_E_ARG, "tokens * q_heads / heads must stay under 2^31");
        if (cache->batch == 0 || cache->tokens == 0) return PFM_OK;
        TRY(check_rows(fn, "q", q, cache->dtype, a.q));
        TRY(check_rows(fn, "out", out, cache->dtype, a.o));
        if (!apart({{cache->tokens, a.o.ts}, {q_heads, a.o.hs}}, a.c.dim))
            return fail(fn, PFM_E_ARG, "out overlaps itself");
        a.q_heads = q_heads;
        a.group = q_heads / cache->heads;
        a.by_group = fast_div((uint32_t)a.group);
        a.scale_log2 = scale == 0.f ? 1.f : fabsf(scale) * 1.44269504088896340736f;
        a.q_sign = (scale > 0.f) - (scale < 0.f);
        a.causal = causal ? 1 : 0;
        a.window = window < (long long)a.c.width * a.c.page + a.c.tokens ? window : 0;     // reaches over all there is
        pfm_paged_attention_plan(cache->dtype, a);
        // a launch has under 2^32 threads
        if ((a.rows_tiles + 2 * a.tiles) * cache->heads >= 1ll << 24)
            return fail(fn, PFM_E_ARG, "too many sequences, tokens and heads for one call");
        const long long need = attention_ws(a);
        if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
            return fail(fn, PFM_E_ARG, "workspace missing, not aligned to 16 bytes or under pfm_paged_attention_ws_bytes");
        if (need) a.ws = (float*)ws;
        const PfmDevOp ops[] = {{"q", a.q.p}, {"out", a.o.p}, {"k_pages", a.c.k}, {"v_pages", a.c.v},
                                {"block_table", a.c.table}, {"kv_len", a.c.kv_len}, {"cu_q", a.c.cu_q},
                                {"ws", a.ws}};
        TRY(pfm_check_dev_ops(fn, ops, (int)(sizeof(ops) / sizeof(ops[0]))));
        return hip(fn, pfm_paged_attention(cache->dtype, a, (hipStream_t)stream));
    });
}

int64_t pfm_sample_ws_size(int B, int V) { return B < 1 || V < 1 ? 0 : pfm_sample_ws_bytes(B, V); }

int pfm_op_sample(void* stream, int dtype, const void* logits, int64_t ld, int B, int V, const float* u,
                  const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                  int32_t* token, float* prob, void* ws, int64_t ws_bytes) {
    static const char fn[] = "pfm_op_sample";
    return guarded(fn, [&]() -> int {
        if (!is_dtype(dtype)) return fail(fn, PFM_E_ARG, "dtype must be PFM_F32, PFM_BF16 or PFM_F16");
        if (B < 0 || B > (1 << 20) || V < 1 || V > (1 << 20))
            return fail(fn, PFM_E_ARG, "need 0 <= B <= 2^20 and 1 <= V <= 2^20");
        if (ld < V) return fail(fn, PFM_E_ARG, "ld is smaller than V");
        if (B == 0) return PFM_OK;
        if (!logits || !u || !token) return fail(fn, PFM_E_ARG, "null operand");
        if ((uintptr_t)logits % elem_bytes(dtype)) return fail(fn, PFM_E_ARG, "logits must be aligned to their type");
        const long long need = pfm_sample_ws_bytes(B, V);
        if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
            return fail(fn, PFM_E_ARG, "workspace missing, not aligned to 16 bytes or under pfm_sample_ws_size");
        const PfmDevOp ops[] = {{"logits", logits}, {"u", u}, {"temperature", temperature}, {"top_k", top_k},
                                {"top_p", top_p}, {"min_p", min_p}, {"token", token}, {"prob", prob},
                                {"ws", need ? ws : nullptr}};
        TRY(pfm_check_dev_ops(fn, ops, (int)(sizeof(ops) / sizeof(ops[0]))));
        const SampleArgs a{logits, ld, B, V, u, temperature, top_p, min_p, top_k, token, prob, ws};
        return hip(fn, pfm_sample(dtype, a, (hipStream_t)stream));
    });
}

}  // extern "C"
