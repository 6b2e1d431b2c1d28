// Token-by-token decoding over a paged key / value cache: argument blocks shared by the kernels (k_paged.hip,
// k_sample.hip) and their C entry points (pfm_serve.hip).
#pragma once
#include <atomic>

#include "pfm_common.h"

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <> __device__ __forceinline__ float to_f<f16>(f16 x) { return (float)x; }
template <> __device__ __forceinline__ f16 from_f<f16>(float x) { return (f16)x; }

// dtype code of the serving entry points beside DT_F32 / DT_BF16 (include/pfm.h PFM_F16; 2 is DT_X3 inside)
enum { DT_F16 = 3 };

// An operand of a C entry point, for the check that it is device memory (pfm_api.hip).
struct PfmDevOp { const char* name; const void* p; };

// x / d for 0 <= x < 2^31 by one multiply: m = ceil(2^(32 + s) / d) with s = ceil(log2 d) gives the exact quotient
// (m < 2^33; the part above 2^32 is added back as x itself, which cannot overflow 64 bits; d = 1 gives x).
struct FastDiv {
    uint32_t mul, shift, d;
    __device__ __forceinline__ int div(int x) const {
        return (int)(((unsigned long long)__umulhi((uint32_t)x, mul) + (uint32_t)x) >> shift);
    }
};
static inline FastDiv fast_div(uint32_t d) {
    FastDiv f{0, 0, d};
    while (f.shift < 31 && (1u << f.shift) < d) ++f.shift;
    f.mul = (uint32_t)((((1ull << f.shift) - d) << 32) / d + 1);
    return f;
}

// More LDS than 64 KiB is asked for once per kernel and device.
template <auto KERNEL> hipError_t pfm_allow_lds(int bytes) {
    static std::atomic<unsigned long long> done{0};
    if (bytes <= 64 * 1024) return hipSuccess;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load() & bit)) return hipSuccess;
    e = hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) done.fetch_or(bit);
    return e;
}
// A batch of sequences whose keys and values lie in pages. Strides count 16-byte pieces (so that an offset takes one
// 32 x 32 -> 64 bit multiply-add per stride); the head dimension is contiguous.
struct PagedKv {
    char *k, *v;                        // pages
    uint32_t ks[3], vs[3];              // strides of page, slot in the page, head
    long long pages;
    const int* table;                   // [batch][table_stride]: page of key positions P i .. P i + P - 1
    long long table_stride;
    int width;                          // entries of a table row that may be read
    int page, heads, dim, batch, tokens;
    FastDiv by_page;
    const int* kv_len;                  // [batch]: keys of the sequence, this call's new tokens included
    const int* cu_q;                    // [batch + 1]: first row of each sequence's new tokens, or null: one token each

    // Byte offsets of head 0 of a slot.
    __device__ __forceinline__ unsigned long long k_at(int pg, int slot) const {
        return ((unsigned long long)(uint32_t)pg * ks[0] + (unsigned long long)(uint32_t)slot * ks[1]) * 16;
    }
    __device__ __forceinline__ unsigned long long v_at(int pg, int slot) const {
        return ((unsigned long long)(uint32_t)pg * vs[0] + (unsigned long long)(uint32_t)slot * vs[1]) * 16;
    }
    __device__ __forceinline__ char* k_head(int h) const { return k + (unsigned long long)(uint32_t)h * ks[2] * 16; }
    __device__ __forceinline__ char* v_head(int h) const { return v + (unsigned long long)(uint32_t)h * vs[2] * 16; }

    // The sequence's keys: never more than its table row can name.
    __device__ __forceinline__ int len(int b) const {
        const long long cap = (long long)width * page;
        const int n = kv_len[b];
        return n < 0 ? 0 : n > cap ? (int)cap : n;
    }
    // New rows [first, end) of sequence b, kept inside [0, tokens); none if they descend.
    __device__ __forceinline__ void rows(int b, int& first, int& end) const {
        if (!cu_q) { first = b; end = b + 1; return; }
        first = max(cu_q[b], 0);
        end = max(min(cu_q[b + 1], tokens), 0);       // end - first stays in 32 bits
    }
};
struct Rows {                           // [tokens][heads][dim] with any token / head stride
    char* p;
    long long ts, hs;
};

struct AppendArgs {
    PagedKv c;
    Rows q, k, v, qo;
    int q_heads;                        // 0: no queries to rotate
    const float* inv_freq;              // [rot / 2] or null: nothing is rotated
    int rot, interleaved;
    const int* pos;                     // [tokens] rotation positions, or null: the cache positions
    int row0;                           // the launch's first row
};
hipError_t pfm_kv_append(int dtype, const AppendArgs& a, hipStream_t st);

// Where a kernel whose row tiles are split leaves its parts in the workspace: [splits][rows] sums of dim floats, then
// as many pairs of maximum and sum. A query row's place is token * q_heads + head, or that of its row tile (by_tile).
struct PagedParts {
    long long rows;
    bool by_tile;
};

struct PagedAttnArgs {
    PagedKv c;
    Rows q, o;
    int q_heads, group;                 // group = q_heads / c.heads
    FastDiv by_group;
    float scale_log2;                   // |scale| * log2(e), or 1 for a scale of 0
    int q_sign;                         // the scale's sign, -1, 0 or 1
    int causal, window;
    // the launch (pfm_paged_attention_plan)
    int rows_upto;                      // sequences of at most so many query rows go to the rows kernel
    long long rows_tiles, tiles;        // row tiles of the rows and of the tile kernel at most
    int splits, tile_splits;            // workgroups that share one row tile's keys, at most
    int fill;                           // of `splits`, as many as fill the chip
    PagedParts rows_part, tile_part;
    float* ws;                          // the parts of one kernel after the other's
};
void pfm_paged_attention_plan(int dtype, PagedAttnArgs& a);   // of a.c, a.q_heads, a.group and a.window
hipError_t pfm_paged_attention(int dtype, const PagedAttnArgs& a, hipStream_t st);

struct SampleArgs {
    const void* x;                      // logits [batch][ld]
    long long ld;
    int batch, vocab;
    const float *u, *temperature, *top_p, *min_p;   // [batch]; null: off
    const int* top_k;
    int* token;
    float* prob;
    void* ws;
};
long long pfm_sample_ws_bytes(int batch, int vocab);
hipError_t pfm_sample(int dtype, const SampleArgs& a, hipStream_t st);
