// Paged key / value cache: appending new tokens' keys and values with their rotation, and attention of new tokens
// over the cache.
//
// Row n of the new tokens belongs to sequence b with cu_q[b] <= n < cu_q[b + 1] and stands at cache position
// kv_len[b] - (cu_q[b + 1] - cu_q[b]) + (n - cu_q[b]); position t lies in slot t % P of page block_table[b][t / P].
// A page id outside [0, pages) names no page: nothing is written there and its keys are not seen, so no table
// content can reach memory outside the pages.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "pfm_serve.h"

namespace {

// Sequence of row n: how many sequences end at or before it, 64 at a time. All lanes of the wave take part and n is the
// same in each of them. c.batch for rows behind the last sequence.
__device__ __forceinline__ int seq_of_row(const PagedKv& c, int n, int lane) {
    if (!c.cu_q) return n;
    int b = 0;
    for (int i0 = 0; i0 < c.batch; i0 += 64) {
        const int i = i0 + lane;
        const int ended = __popcll(__ballot(i < c.batch && c.cu_q[i + 1] <= n));
        b += ended;
        if (ended < 64) break;
    }
    return b;
}

__device__ __forceinline__ int page_of(const PagedKv& c, int b, int t) {   // t inside the table's reach
    const int pg = c.table[b * c.table_stride + t];
    return pg >= 0 && pg < c.pages ? pg : -1;
}

template <typename T> struct Vec8 { T x[8]; };
template <typename T> struct Pack16 { T x[16 / sizeof(T)]; };
template <typename T> __device__ __forceinline__ Vec8<T> load8(const char* p) {
    Vec8<T> v;
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i) ((float4*)&v)[i] = ((const float4*)p)[i];
    return v;
}
template <typename T> __device__ __forceinline__ void store8(char* p, const Vec8<T>& v) {
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i) ((float4*)p)[i] = ((const float4*)&v)[i];
}

// ---- append -------------------------------------------------------------------------------------------------------
// (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin) by the angle pos * inv_freq, then one rounding to the type. It is a copy
// that memory bounds: one workgroup per token (four tokens each: 95 us where this takes 88, 16384 tokens of 32 query and 8
// kv heads of 128 dims in 16 bits). The angles are reduced to a turn in 64 bits (a far position's angle has lost its
// fraction in 32), the sine and cosine are taken once per pair and shared by all heads through LDS; a thread moves 16 or
// 32 bytes of a head at a time. One token of 64 sequences takes 4 us: three reads that wait for each other, and a launch.
constexpr int AP_T = 256;

template <typename T>
__global__ __launch_bounds__(AP_T) void kv_append_kernel(AppendArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, n = a.row0 + blockIdx.x;
    const int half = a.inv_freq ? a.rot / 2 : 0;
    float2* cs = (float2*)smem;             // [half] (cos, sin)
    const PagedKv& c = a.c;

    const int b = seq_of_row(c, n, lane);   // every wave for itself
    if (b >= c.batch) return;
    int first, end;
    c.rows(b, first, end);
    if (n < first) return;
    const int len = c.len(b), at = len - (end - first) + (n - first);
    int page = -1, slot = 0;                // no page: rotated, but no place to write
    if (at >= 0 && at < len) {
        const int pi = c.by_page.div(at);
        page = page_of(c, b, pi);
        slot = at - pi * c.page;
    }
    const int pos = a.pos ? a.pos[n] : at;
    for (int f = tid; f < half; f += AP_T) {
        double r = (double)pos * (double)a.inv_freq[f] * 0.15915494309189533577;   // turns
        r -= rint(r);
        float s, co;
        sincospif((float)(2.0 * r), &s, &co);
        cs[f] = make_float2(co, s);
    }
    __syncthreads();

    // work items of a token: rotated pairs of 8-wide pieces, the unrotated rest of q and k, the pieces of v
    const int D8 = c.dim / 8, h8 = half / 8, rest8 = D8 - 2 * h8;
    const int turned = (a.q_heads + c.heads) * h8, kept = (a.q_heads + c.heads) * rest8, vals = c.heads * D8;
    const int per = turned + kept + vals;
    constexpr int E = sizeof(T);
    for (int i = tid; i < per; i += AP_T) {
        int w = i;
        if (w < turned + kept) {
            const bool turn = w < turned;
            if (!turn) w -= turned;
            const int per_h = turn ? h8 : rest8;
            int h = w / per_h;
            const int j = w - h * per_h;
            const bool isq = h < a.q_heads;
            const char* src;
            char* dst;
            if (isq) {
                src = a.q.p + ((long long)n * a.q.ts + (long long)h * a.q.hs) * E;
                dst = a.qo.p + ((long long)n * a.qo.ts + (long long)h * a.qo.hs) * E;
            } else {
                h -= a.q_heads;
                if (page < 0) continue;
                src = a.k.p + ((long long)n * a.k.ts + (long long)h * a.k.hs) * E;
                dst = c.k_head(h) + c.k_at(page, slot);
            }
            if (!turn) {
                const int o = (2 * h8 + j) * 8 * E;
                store8<T>(dst + o, load8<T>(src + o));
                continue;
            }
            // the two pieces of a pair group: (x1 | x2) half a rotated width apart, or 16 neighbours
            const int o1 = a.interleaved ? j * 16 * E : j * 8 * E, o2 = a.interleaved ? o1 + 8 * E : o1 + half * E;
            Vec8<T> p = load8<T>(src + o1), q = load8<T>(src + o2), p2, q2;
            const float2* m = cs + j * 8;
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = m[e], g = m[e + 4];
                    const float x = to_f(p.x[2 * e]), y = to_f(p.x[2 * e + 1]), z = to_f(q.x[2 * e]), u = to_f(q.x[2 * e + 1]);
                    p2.x[2 * e] = from_f<T>(x * f.x - y * f.y);
                    p2.x[2 * e + 1] = from_f<T>(y * f.x + x * f.y);
                    q2.x[2 * e] = from_f<T>(z * g.x - u * g.y);
                    q2.x[2 * e + 1] = from_f<T>(u * g.x + z * g.y);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 f = m[e];
                    const float x = to_f(p.x[e]), y = to_f(q.x[e]);
                    p2.x[e] = from_f<T>(x * f.x - y * f.y);
                    q2.x[e] = from_f<T>(y * f.x + x * f.y);
                }
            }
            store8<T>(dst + o1, p2);
            store8<T>(dst + o2, q2);
        } else {
            w -= turned + kept;
            if (page < 0) continue;
            const int h = w / D8, o = (w - h * D8) * 8 * E;
            store8<T>(c.v_head(h) + c.v_at(page, slot) + o,
                      load8<T>(a.v.p + ((long long)n * a.v.ts + (long long)h * a.v.hs) * E + o));
        }
    }
}

// ---- attention ----------------------------------------------------------------------------------------------------
// o_i = sum_j p_ij v_j / sum_j p_ij with p_ij = exp(scale q_i . k_j - m_i), in one pass over the keys: m is the running
// maximum, and o and the sum are scaled down when it grows. The exponent's base is 2 (log2 e goes into the scale). All
// of it is held in 32 bits; p is rounded to the cache's 16-bit type for the second product, since the matrix instruction
// takes its operands so: relative to itself by half a step, as the values are. f16's step stops shrinking at 2^-14, which a
// long tail behind one dominant key lies under, so there m is less than the maximum by LOWER and p reaches 2^15: half
// a step is relative down to 2^-29 of the largest p, and absolute 2^-40 under it (2^-32 in the tile kernel). (Each p as the
// sum of two 16-bit numbers: 0.6 .. 1.7 % more time for single tokens, half as many products again for prompts; the
// result's own rounding is as large as what it would save.) Two kernels: rows (16 query rows, memory bounds it: the single tokens) and tile (256 query
// rows that share their keys, the matrix products bound it: the chunks of prompts), and a join where keys are split.
//
// Operand traits. The products run swapped, S^T = K Q^T and O^T = V^T P^T: in both accumulators the query row is the
// lane (lane & 15), so a row's maximum, sum and rescale are per lane, and the probabilities of two 16-key tiles are, as
// they stand in S^T's registers, the second product's operand: its contraction index 8 g + j is key 4 g + j of the
// first tile (j < 4) or key 4 g + j - 4 of the second, for the lane group g = lane >> 4.
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef short v8i16 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

template <typename T> struct Mma;
template <> struct Mma<bf16> {
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x4 mul(frag a, frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct Mma<f16> {
    typedef f16x8 frag;
    static __device__ __forceinline__ f32x4 mul(frag a, frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

// the maximum's distance above m; the tile kernel lets a score pass its m by LATE more before it rescales
constexpr float LATE = 8.f;
template <typename T, bool TILE> constexpr float LOWER = std::is_same<T, f16>::value ? (TILE ? 15.f - LATE : 15.f) : 0.f;
// From FAR on a score's own step is 1/8 and more, and grows to where it alone would carry p out of its type's range:
// differences are taken between scores that are rounded alike, and m is one of them.
constexpr float FAR = 1048576.f;
template <typename T, bool TILE> __device__ __forceinline__ float lowered(float mt) {
    return LOWER<T, TILE> == 0.f || fabsf(mt) >= FAR ? mt : mt - LOWER<T, TILE>;
}

__device__ __forceinline__ float group_max(float x) {   // over the four lanes of a query row
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float group_sum(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

// A scale's sign goes to the queries, and a scale of 0 as well (the scores' scale is 1 then): what is hidden stays at -inf.
template <typename T> __device__ __forceinline__ T times(T x, int sign) { return from_f<T>(to_f(x) * (float)sign); }

// a 32-bit word of values with zeros for those that are not finite; bad: there were such
template <typename T> __device__ __forceinline__ float finite_word(float x, bool& bad) {
    constexpr uint32_t M = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, f16>::value ? 0x7c00u : 0x7f80u;   // exponent
    const uint32_t w = __float_as_uint(x);
    uint32_t clear = (w & M) == M ? (sizeof(T) == 4 ? ~0u : 0xffffu) : 0u;
    if (sizeof(T) == 2) clear |= ((w >> 16) & M) == M ? 0xffff0000u : 0u;
    bad = bad || clear;
    return __uint_as_float(w & ~clear);
}

// o[i ..] += the values that are not finite among the four dims dd .. of a value row
template <typename T, typename V>
__device__ __forceinline__ void add_odd(const T* row, int dd, int dim, V& o, int i) {
    if (dd >= dim) return;
    struct alignas(4 * sizeof(T)) Four { T x[4]; };
    const Four v = *(const Four*)(row + dd);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float x = to_f(v.x[k]);
        if (!(fabsf(x) < INFINITY)) o[i + k] += x;
    }
}

// a value that is the same in all lanes, as a scalar
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

constexpr int DEC_W = 4;      // waves of a workgroup; each runs over key blocks of its own
template <typename T, int DP, int NTILES> struct DecGeom {
    static constexpr int PITCH = DP * sizeof(T) + (sizeof(T) == 2 ? 32 : 16);   // rows of V: no bank met twice
    static constexpr int NT = NTILES;                                          // 16-key tiles of a block
    static constexpr int KB = 16 * NT;
    static constexpr int WAVE = KB * PITCH;
    static constexpr int MERGE = DEC_W * 16 * (DP + 4) * 4;                     // overlays the V blocks at the end
    static constexpr int LDS = DEC_W * WAVE > MERGE ? DEC_W * WAVE : MERGE;
};

// Row tile x, `rows` query rows (token, head of the group) each, of the sequences that have more than `over` and at most
// `upto` rows: its sequence and place there. Every lane of every wave comes to the same answer.
__device__ __forceinline__ bool find_tile(const PagedKv& c, int group, int rows, int over, int upto, int x, int lane,
                                          int& b, int& tile) {
    if (!c.cu_q) {
        const int per = (group + rows - 1) / rows;
        b = x / per;
        tile = x - b * per;
        return b < c.batch;
    }
    for (int i0 = 0; i0 < c.batch; i0 += 64) {
        const int i = i0 + lane;
        int tiles = 0;
        if (i < c.batch) {
            int first, end;
            c.rows(i, first, end);
            const int n = max(end - first, 0) * group;
            tiles = n > over && n <= upto ? (n + rows - 1) / rows : 0;
        }
        int sum = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int s = __shfl_up(sum, o, 64);
            if (lane >= o) sum += s;
        }
        const unsigned long long past = __ballot(sum > x);
        if (past) {
            const int l = __ffsll((long long)past) - 1;
            b = i0 + l;
            tile = x - __builtin_amdgcn_readlane(sum - tiles, l);
            return true;
        }
        x -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// The same with the sequences of most keys first (among 64 neighbours in the batch), and of each the tiles that see most:
// a tile runs as long as its keys are many, and long ones that start last leave most of the chip idle at the end. 8
// sequences of 136 .. 700 new tokens over 1218 .. 6418 keys: 331 us in the batch's order, 279 in this one.
__device__ __forceinline__ bool find_longest(const PagedKv& c, int group, int rows, int over, int x, int lane, int& b,
                                             int& tile) {
    for (int i0 = 0; i0 < c.batch; i0 += 64) {
        const int i = i0 + lane;
        int tiles = 0, len = -1;
        if (i < c.batch) {
            int first, end;
            c.rows(i, first, end);
            const int n = max(end - first, 0) * group;
            tiles = n > over ? (n + rows - 1) / rows : 0;
            len = c.len(i);
        }
        int all = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) all += __shfl_xor(all, o, 64);
        all = __builtin_amdgcn_readfirstlane(all);
        if (x < all) {
            int start = 0;                       // tiles of the sequences before the lane's
            for (int k = 0; k < min(64, c.batch - i0); ++k) {
                const int n = __builtin_amdgcn_readlane(tiles, k), l = __builtin_amdgcn_readlane(len, k);
                start += l > len || (l == len && k < lane) ? n : 0;
            }
            const int l = __ffsll((long long)__ballot(start <= x && x < start + tiles)) - 1;
            b = i0 + l;
            tile = __builtin_amdgcn_readlane(start + tiles, l) - 1 - x;
            return true;
        }
        x -= all;
    }
    return false;
}

// The keys that the query rows row0 .. row1 of a sequence see, [lo, hi) of all, and their blocks of kb keys.
struct Span { int pmin, pmax, lo, hi, blk0, nblk; };
__device__ __forceinline__ Span span_of(const PagedAttnArgs& a, int nq, int len, int row0, int row1, int kb) {
    Span s;
    s.pmin = len - nq + a.by_group.div(row0);
    s.pmax = len - nq + a.by_group.div(row1);
    s.hi = a.causal ? min(len, s.pmax + 1) : len;
    s.lo = a.window ? max(0, s.pmin - a.window + 1) : 0;
    s.blk0 = s.lo / kb;
    s.nblk = s.hi > s.lo ? (s.hi + kb - 1) / kb - s.blk0 : 0;
    return s;
}
// Parts that a row tile of the rows kernel is split into: enough to fill the chip with parts of at least PART_MIN keys, and
// none longer than PART_MAX where the launch has that many. 255 caches of 1024 keys and one of 65536, 32 heads on 8: 1758
// us whole, 493 with the long one in 8 parts; 300 caches of 8192: 1709 us whole, 1742 in halves.
constexpr int PART_MIN = 256, PART_MAX = 8192;
__device__ __forceinline__ int parts_of(const PagedAttnArgs& a, int nblk, int kb) {
    const int keys = nblk * kb, n = max((keys + PART_MAX - 1) / PART_MAX, min(a.fill, (keys + PART_MIN - 1) / PART_MIN));
    return max(1, min(n, a.splits));
}

// One workgroup = 16 query rows of one sequence and kv head; its waves take key blocks in turn, each with its own V
// block in LDS and no barrier until the waves' results are joined. The matrix instruction has 16 rows whether the group of
// query heads fills them or not: its time is hidden. K goes from memory to registers as the product's operand, V over
// LDS, which transposes it; both of the next block are under way while this one is worked on (387 us without, 265 with).
// 64 caches of 1000 .. 9216 keys, 32 heads on 8 of 128 dims in 16 bits: 1.20 GB in 254 .. 271 us, 4.4 .. 4.7 TB/s, where a
// copy of 4 GiB makes 4.75. One cache of 201 keys takes 10 us, of which most is waiting: length, page id, keys, values.
template <typename T, int DP, int NTILES>
__global__ __launch_bounds__(DEC_W * 64) void paged_rows_kernel(PagedAttnArgs a) {
    using G = DecGeom<T, DP, NTILES>;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int ND = DP / 16;
    constexpr int E = sizeof(T), NT = G::NT, KB = G::KB;
    constexpr unsigned ALL = NT == 2 ? ~0u : 0xffffu;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ float ml[DEC_W][16][2];
    const PagedKv& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wid = uniform(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int hk = blockIdx.x % c.heads;
    int b, tile;
    if (!find_tile(c, a.group, 16, 0, a.rows_upto, blockIdx.x / c.heads, lane, b, tile)) return;
    b = uniform(b);
    tile = uniform(tile);
    int first, end;
    c.rows(b, first, end);
    first = uniform(first);
    const int nq = uniform(end) - first, len = uniform(c.len(b));
    const int rows = min(16, nq * a.group - tile * 16);            // of this tile
    const int row = min(tile * 16 + r, nq * a.group - 1);
    const int place = a.by_group.div(row);
    const int head = hk * a.group + row - place * a.group;
    const int pos = len - nq + place;
    const Span span = span_of(a, nq, len, tile * 16, tile * 16 + rows - 1, KB);
    const int pmin = span.pmin, pmax = span.pmax, lo = span.lo, hi = span.hi, blk0 = span.blk0, nblk = span.nblk;
    const int split = blockIdx.y, parts = uniform(parts_of(a, nblk, KB));
    if (split >= parts) return;
    const int s0 = (int)((long long)nblk * split / parts), s1 = (int)((long long)nblk * (split + 1) / parts);

    unsigned char* Vs = smem + wid * G::WAVE;

    // Q in the operand layout: 16-bit: dims 32 c + 8 g ..; 32-bit: dims 16 c + 4 g .. (the same order as K below)
    Vec8<T> qf[DP / 32];
    {
        const char* qp = a.q.p + ((long long)(first + place) * a.q.ts + (long long)head * a.q.hs) * E;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k) {
            const int d0 = F32 ? 32 * k + 4 * g : 32 * k + 8 * g;
            qf[k] = Vec8<T>{};
            if constexpr (F32) {
                if (d0 < c.dim) ((float4*)&qf[k])[0] = *(const float4*)(qp + d0 * E);
                if (d0 + 16 < c.dim) ((float4*)&qf[k])[1] = *(const float4*)(qp + (d0 + 16) * E);
            } else if (d0 < c.dim) {
                qf[k] = load8<T>(qp + d0 * E);
            }
        }
        if (a.q_sign != 1) {
#pragma unroll
            for (int k = 0; k < DP / 32; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) qf[k].x[e] = times(qf[k].x[e], a.q_sign);
        }
    }
    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    // The lane's key rows of a block are j0 + r and j0 + 16 + r, of K (operand layout as it is) and of V alike. A block is
    // loaded while the one before it is worked on: its K goes into the registers that the products have just read, its
    // V into those that LDS has just taken, and the page ids of the block after it are on their way.
    constexpr int NL = DP * E / 64;              // 16-byte pieces of a row that a lane holds: at 64 k + 16 g
    float4 kf[NT][NL], vf[NT][NL];
    int page[NT];                                // of the block to be loaded next; -1: no such key
    long long ko[NT], vo[NT];
    unsigned here = 0;                           // keys of the loaded block that exist
    auto pages = [&](int blk) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int j = (blk0 + blk) * KB + 16 * t + r;
            page[t] = -1;
            if (blk < s1 && j >= lo && j < hi) page[t] = c.table[b * c.table_stride + c.by_page.div(j)];
            if ((unsigned long long)(long long)page[t] >= (unsigned long long)c.pages) page[t] = -1;
        }
    };
    auto address = [&](int blk) {
        here = (unsigned)(__ballot(page[0] >= 0) & 0xffff);
        if constexpr (NT == 2) here |= (unsigned)(__ballot(page[NT - 1] >= 0) & 0xffff) << 16;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int j = (blk0 + blk) * KB + 16 * t + r, slot = j - c.by_page.div(j) * c.page;
            ko[t] = (long long)c.k_at(page[t], slot);
            vo[t] = (long long)c.v_at(page[t], slot);
        }
        if (here != ALL && here) {               // rows that are not there read one that is
            const int f = __ffs((int)here) - 1;
            const long long k1 = __shfl(f < 16 ? ko[0] : ko[NT - 1], f & 15, 64);
            const long long v1 = __shfl(f < 16 ? vo[0] : vo[NT - 1], f & 15, 64);
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if (page[t] < 0) { ko[t] = k1; vo[t] = v1; }
        }
    };
    // pieces behind the head's dims read its last ones: their K is cleared, their V is not used
    auto load = [&](const char* base, const long long (&off)[NT], float4 (&x)[NT][NL]) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < NL; ++k)
                x[t][k] = *(const float4*)(base + off[t] + min(64 * k, c.dim * E - 16 - 16 * g));
    };
    const char *k0 = c.k_head(hk) + 16 * g, *v0 = c.v_head(hk) + 16 * g;
    int blk = s0 + wid;
    pages(blk);
    address(blk);
    if (here) { load(k0, ko, kf); load(v0, vo, vf); }
    pages(blk + DEC_W);

    for (; blk < s1; blk += DEC_W) {
        const int j0 = (blk0 + blk) * KB;
        const unsigned there = here;
        // keys this lane's scores belong to (rows 4 g + i of each tile) that exist
        const unsigned exist = ((there >> (4 * g)) & 15) | ((there >> (16 + 4 * g)) & 15) << 4;
        // S^T = K Q^T
        f32x4 s[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NL; ++k) {
                float4 x = kf[t][k];
                if (DP * E > c.dim * E && 64 * k + 16 * g >= c.dim * E) x = make_float4(0.f, 0.f, 0.f, 0.f);
                if constexpr (F32) {
                    const float4 q4 = ((const float4*)qf)[k];
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, q4.x, s[t], 0, 0, 0);
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, q4.y, s[t], 0, 0, 0);
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, q4.z, s[t], 0, 0, 0);
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, q4.w, s[t], 0, 0, 0);
                } else {
                    s[t] = Mma<T>::mul(*(typename Mma<T>::frag*)&x, *(typename Mma<T>::frag*)&qf[k], s[t]);
                }
            }
        }
        address(blk + DEC_W);
        if (here) load(k0, ko, kf);
        // V rows into LDS, absent ones as zeros
        // (rows at one position see the same keys, and the others are not there)
        const bool part = pmin < pmax && ((a.causal && j0 + KB - 1 > pmin) || (a.window && j0 <= pmax - a.window));
        bool odd = false;     // a value that is not finite, in a block that the rows do not all see whole
        if (there != ALL) {
            asm volatile("" ::: "memory");       // branches of their own: not folded into every block
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < NL; ++k)
                    if (!((there >> (16 * t + r)) & 1)) vf[t][k] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (part) {
            asm volatile("" ::: "memory");
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < NL; ++k) {
                    const float4 x = vf[t][k];
                    vf[t][k] = make_float4(finite_word<T>(x.x, odd), finite_word<T>(x.y, odd), finite_word<T>(x.z, odd),
                                           finite_word<T>(x.w, odd));
                }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < NL; ++k) *(float4*)(Vs + (16 * t + r) * G::PITCH + 64 * k + 16 * g) = vf[t][k];
        if (here) load(v0, vo, vf);
        pages(blk + 2 * DEC_W);
        // scores in base-2 exponents; a key that the row does not see is replaced, whatever its score is
        unsigned seen = exist;
        if (part) {
#pragma unroll
            for (int e = 0; e < 4 * NT; ++e) {
                const int j = j0 + 16 * (e >> 2) + 4 * g + (e & 3);
                if ((a.causal && j > pos) || (a.window && j <= pos - a.window)) seen &= ~(1u << e);
            }
        }
        float mt = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4 * NT; ++e) {
            float x = s[e >> 2][e & 3] * a.scale_log2;
            x = (seen >> e) & 1 ? x : -INFINITY;
            s[e >> 2][e & 3] = x;
            mt = fmaxf(mt, x);      // passes a NaN over: its own probability carries it on
        }
        mt = group_max(mt);
        const float mn = fmaxf(m, lowered<T, false>(mt)), mu = mn == -INFINITY ? 0.f : mn;
        const float corr = __builtin_amdgcn_exp2f(m - mu);
        m = mn;
        float p[4 * NT], ls = 0.f;
#pragma unroll
        for (int e = 0; e < 4 * NT; ++e) {
            p[e] = __builtin_amdgcn_exp2f(s[e >> 2][e & 3] - mu);
            ls += p[e];
        }
        l = l * corr + ls;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= corr;
        // O^T += V^T P^T (the wave reads what it wrote itself: a wait, no barrier)
        __builtin_amdgcn_wave_barrier();
        if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4 * NT; ++e) {
                const float* vr = (const float*)(Vs + (16 * (e >> 2) + 4 * g + (e & 3)) * G::PITCH) + r;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[16 * d], p[e], o[d], 0, 0, 0);
            }
        } else {
            Vec8<T> pb;      // probabilities rounded to the type: relative to each its half step, as the values are
#pragma unroll
            for (int e = 0; e < 8; ++e) pb.x[e] = from_f<T>(p[e]);
            // transposing read: of 4 rows x 16 dims, lane r of the group gets dim r of the 4 rows
            const unsigned char* vp = Vs + (4 * g + (r >> 2)) * G::PITCH + (r & 3) * 8;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const v4i16 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vp + 32 * d));
                const v4i16 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vp + 16 * G::PITCH + 32 * d));
                const v8i16 va = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                o[d] = Mma<T>::mul(*(const typename Mma<T>::frag*)&va, *(typename Mma<T>::frag*)&pb, o[d]);
            }
        }
        // values that are not finite belong to the rows that see them only (whatever their weight): 0 x inf in the product
        // would reach the rest
        if (part && __any(odd)) {
            for (int kr = 0; kr < KB; ++kr) {
                const int j = j0 + kr;
                if (!((there >> kr) & 1) || (a.causal && j > pos) || (a.window && j <= pos - a.window)) continue;
                const int pi = c.by_page.div(j);
                const T* vr = (const T*)(c.v_head(hk) + c.v_at(page_of(c, b, pi), j - pi * c.page));
                int d0 = 4 * g;
                asm volatile("" : "+v"(d0));       // nothing of this is kept ready for every block
#pragma unroll
                for (int d = 0; d < ND; ++d) add_odd<T>(vr, d0 + 16 * d, c.dim, o[d], 0);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }

    // join the waves: their maxima, then their sums scaled to the common one
    l = group_sum(l);
    if (g == 0) { ml[wid][r][0] = m; ml[wid][r][1] = l; }
    __syncthreads();
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < DEC_W; ++w) mm = fmaxf(mm, ml[w][r][0]);
    const float sc = __builtin_amdgcn_exp2f(m - (mm == -INFINITY ? 0.f : mm));
    float* os = (float*)smem + wid * 16 * (DP + 4);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        f32x4 x = o[d] * sc;
        *(f32x4*)(os + r * (DP + 4) + 16 * d + 4 * g) = x;
    }
    __syncthreads();
    const float* ob = (const float*)smem;
    for (int i = tid; i < 16 * (DP / 8); i += DEC_W * 64) {
        const int rr = i / (DP / 8), d0 = (i % (DP / 8)) * 8;
        if (rr >= rows || d0 >= c.dim) continue;
        float x[8] = {};
#pragma unroll
        for (int w = 0; w < DEC_W; ++w)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] += ob[(w * 16 + rr) * (DP + 4) + d0 + e];
        const int row2 = tile * 16 + rr, pl = a.by_group.div(row2);
        const int hd = hk * a.group + row2 - pl * a.group, n = first + pl;
        float lsum = 0.f, mr = -INFINITY;
#pragma unroll
        for (int w = 0; w < DEC_W; ++w) mr = fmaxf(mr, ml[w][rr][0]);
        const float mu = mr == -INFINITY ? 0.f : mr;
#pragma unroll
        for (int w = 0; w < DEC_W; ++w) lsum += ml[w][rr][1] * __builtin_amdgcn_exp2f(ml[w][rr][0] - mu);
        if (parts == 1) {
            const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
            Vec8<T> y;
#pragma unroll
            for (int e = 0; e < 8; ++e) y.x[e] = from_f<T>(lsum == 0.f ? 0.f : x[e] * inv);
            store8<T>(a.o.p + ((long long)n * a.o.ts + (long long)hd * a.o.hs) * E + d0 * E, y);
        } else {
            const PagedParts& w = a.rows_part;
            const long long pr = split * w.rows + (w.by_tile ? blockIdx.x * 16ll + rr : (long long)n * a.q_heads + hd);
            float *dst = a.ws + pr * c.dim + d0, *dst_ml = a.ws + a.splits * w.rows * c.dim + 2 * pr;
            *(f32x4*)dst = f32x4{x[0], x[1], x[2], x[3]};
            *(f32x4*)(dst + 4) = f32x4{x[4], x[5], x[6], x[7]};
            if (d0 == 0) { dst_ml[0] = mr; dst_ml[1] = lsum; }
        }
    }
}

// ---- chunks: row tiles that share their keys through LDS
// 8 waves of 32 query rows (from 129 dims on, two waves share 32 rows, each with half of the dims of V). K and V
// tiles go from memory straight to LDS, three tiles ahead, in rings of four; a piece's place in its row is
// exclusive-ored with the row, so that no read meets a bank twice as often as it must. The scores of the next tile are
// computed under the exponentials of this one, and o is rescaled only where a maximum has grown by more than 2^LATE: p then
// stays under 2^8 (f16, with LOWER: 2^15). 2 prompts of 4096 tokens over 8192 and 6125 keys, 32 heads on 8 of
// 128 dims in 16 bits: 686 GFLOP in 752 .. 805 us, 852 .. 912 TFLOP/s, where a product of 8192^3 makes 1118. The chip lowers
// its clock to 2.0 GHz under it, and exponentials, maxima and conversions hold the vector units as long as the products
// hold the matrix units: leaving out any one of them saves its own share alone.
//
// The same swapped products on 32 x 32 tiles: a wave owns 32 query rows (row = lane & 31, h = lane >> 5), register e of
// a score tile is key kappa(e) + 4 h, and registers 8 s .. 8 s + 7 are the probabilities of the second product's s-th
// 16 keys in the order key 16 s + 4 h + j, 16 s + 8 + 4 h + j - 4.
__device__ __forceinline__ int kappa(int e) { return (e & 3) + 8 * (e >> 2); }
__device__ __forceinline__ float xor32_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor32_add(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <typename T> struct Mma32;
template <> struct Mma32<bf16> {
    static __device__ __forceinline__ f32x16 mul(bf16x8 a, bf16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct Mma32<f16> {
    static __device__ __forceinline__ f32x16 mul(f16x8 a, f16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void gbl_void;

template <typename T, int DP> struct TileGeom {
    static constexpr int E = sizeof(T);
    static constexpr int NW = 8;
    static constexpr int HALVES = DP > 128 ? 2 : 1;        // 256 registers hold the sums of 128 dims: two waves share 32 rows
    static constexpr int ROWS = NW * 32 / HALVES;
    static constexpr int KT = E == 2 && DP <= 128 ? 64 : 32;   // keys of a tile
    static constexpr int PITCH = DP * E;                   // a row of K or V
    static constexpr int CPR = PITCH / 16;                 // its 16-byte pieces
    static constexpr int TILE = KT * PITCH;
    static constexpr int RING = 4;                         // tiles of K, and of V, in LDS
    static constexpr int LDS = 2 * RING * TILE;
    static constexpr int PER = KT * CPR / (NW * 64);       // pieces of K, and of V, that a thread brings
    // Piece c of row r lies at place c ^ swizzle(r), so that a read meets each bank as often as it must: of K, one piece
    // column of 16 rows; of V, four pieces of 8 rows (transposing reads) or 8 pieces of the rows r and r + 4.
    static __device__ __forceinline__ int kswizzle(int r) { return CPR == 8 ? (r >> 1) & 7 : r & 15; }
    static __device__ __forceinline__ int vswizzle(int r) {
        if (E == 4) return ((r >> 2) & 1) << 3;
        return CPR == 8 ? ((r >> 1) & 1) << 2 : ((r & 3) << 2) | ((r >> 2) & 3);
    }
};

template <typename T, int DP>
__global__ __launch_bounds__((TileGeom<T, DP>::NW * 64), 2) void paged_tile_kernel(PagedAttnArgs a) {
    using G = TileGeom<T, DP>;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int E = sizeof(T), KT = G::KT, NB = KT / 32, ND = DP / 32 / G::HALVES, NT = G::NW * 64;
    constexpr int NQ = DP * E / 32;                          // 16-byte pieces of a query row that a lane holds
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ unsigned char there[G::RING][KT];                 // a tile's keys that exist
    __shared__ int odd[2];                                   // the last tile of a buffer with a value that is not finite
    const PagedKv& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wid = uniform(tid >> 6), fr = lane & 31, h = lane >> 5;
    const int hk = blockIdx.x % c.heads;
    int b, tile;
    if (!find_longest(c, a.group, G::ROWS, a.rows_upto, blockIdx.x / c.heads, lane, b, tile)) return;
    b = uniform(b);
    tile = uniform(tile);
    int first, end;
    c.rows(b, first, end);
    first = uniform(first);
    const int nq = uniform(end) - first, len = uniform(c.len(b)), nrows = nq * a.group, base = len - nq;
    const int row0 = tile * G::ROWS, row1 = min(row0 + G::ROWS, nrows) - 1;
    const int pmin = base + a.by_group.div(row0), pmax = base + a.by_group.div(row1);
    // this wave's rows; -1 rows: none
    const int w0 = row0 + wid / G::HALVES * 32, w1 = min(w0 + 32, nrows) - 1, dim0 = wid % G::HALVES * ND * 32;
    const bool idle = w0 >= nrows;
    const int wmin = idle ? 0 : base + a.by_group.div(w0), wmax = idle ? -1 : base + a.by_group.div(w1);
    const int row = min(w0 + fr, nrows - 1), place = a.by_group.div(row), head = hk * a.group + row - place * a.group;
    const int pos = base + place;
    const int hi = a.causal ? min(len, pmax + 1) : len;
    const int lo = a.window ? max(0, pmin - a.window + 1) : 0;
    const int tile0 = lo / KT, ntile = hi > lo ? (hi + KT - 1) / KT - tile0 : 0;
    const int split = blockIdx.y;
    const int t0 = tile0 + (int)((long long)ntile * split / a.tile_splits);
    const int t1 = tile0 + (int)((long long)ntile * (split + 1) / a.tile_splits);

    float4 qf[NQ];   // 16-bit: dims 16 k + 8 h ..; 32-bit: dims 8 k + 4 h ..
    {
        const char* qp = a.q.p + ((long long)(first + place) * a.q.ts + (long long)head * a.q.hs) * E + 16 * h;
#pragma unroll
        for (int k = 0; k < NQ; ++k)
            qf[k] = (2 * k + h) * 16 < c.dim * E ? *(const float4*)(qp + 32 * k) : make_float4(0.f, 0.f, 0.f, 0.f);
        if (a.q_sign != 1) {
#pragma unroll
            for (int k = 0; k < NQ; ++k) {
                Pack16<T> x = *(Pack16<T>*)&qf[k];
#pragma unroll
                for (int e = 0; e < 16 / E; ++e) x.x[e] = times(x.x[e], a.q_sign);
                qf[k] = *(float4*)&x;
            }
        }
    }
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m = -INFINITY, l = 0.f;

    // Staging: global memory straight to LDS, 1 KiB per instruction of a wave: its pieces lie side by side there, so the
    // lane picks the piece that belongs to its place. The thread's places are piece tid % CPR of the rows tid / CPR +
    // i NT / CPR; what is not there is not loaded, and its V is cleared.
    constexpr int PER = G::PER, RSTEP = NT / G::CPR, RING = G::RING;
    unsigned char *K0 = smem, *V0 = smem + RING * G::TILE;
    const int scol = tid % G::CPR, srow = tid / G::CPR;
    int page[PER];                       // page ids of the tile that comes next; -1: no such key
    auto pages = [&](int t) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int j = t * KT + srow + i * RSTEP, at = min(max(j, lo), hi - 1);
            page[i] = c.table[b * c.table_stride + c.by_page.div(at)];
            if (at != j) page[i] = -1;
        }
    };
    bool full = false;                   // this wave made 2 PER loads for the last tile brought
    auto bring = [&](int t) {
        unsigned char *K = K0 + (t % RING) * G::TILE + wid * 1024, *V = V0 + (t % RING) * G::TILE + wid * 1024;
        full = true;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int r = srow + i * RSTEP, j = t * KT + r, slot = j - c.by_page.div(j) * c.page;
            const int kc = scol ^ G::kswizzle(r), vc = scol ^ G::vswizzle(r);
            const bool is = (unsigned)page[i] < (unsigned)c.pages;
            const char* kp = c.k_head(hk) + c.k_at(page[i], slot) + kc * 16;
            const char* vp = c.v_head(hk) + c.v_at(page[i], slot) + vc * 16;
            const bool kl = is && (DP * E == c.dim * E || kc * 16 < c.dim * E), vl = is && (DP * E == c.dim * E || vc * 16 < c.dim * E);
            if (scol == 0) there[t % RING][r] = is;
            full = full && __any(kl) && __any(vl);      // both loads are made
            if (kl) __builtin_amdgcn_global_load_lds((gbl_void*)kp, (lds_void*)(K + i * NT * 16), 16, 0, 0);
            if (vl) __builtin_amdgcn_global_load_lds((gbl_void*)vp, (lds_void*)(V + i * NT * 16), 16, 0, 0);
            else *(float4*)(V + i * NT * 16 + lane * 16) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    // Before tile t: its V and the K of the next one have come, for all waves. `left`: the tile after that may still come.
    auto arrive = [&](bool left) {
        __builtin_amdgcn_sched_barrier(0);
        if (left) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * PER) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // A tile that some row of the workgroup sees in part: values that are not finite are set aside.
    auto clean = [&](int t) {
        if (!((a.causal && t * KT + KT - 1 > pmin) || (a.window && t * KT <= pmax - a.window))) return;
        unsigned char* V = V0 + (t % RING) * G::TILE + tid * 16;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float4 x = *(const float4*)(V + i * NT * 16);
            *(float4*)(V + i * NT * 16) = make_float4(finite_word<T>(x.x, bad), finite_word<T>(x.y, bad),
                                                      finite_word<T>(x.z, bad), finite_word<T>(x.w, bad));
        }
        if (bad) odd[t & 1] = t;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // where the lane's fragments lie in a tile
    const int tr_row = 4 * h + ((lane & 15) >> 2), tr_piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const int krow = fr * G::PITCH, kx = (h ^ G::kswizzle(fr)) * 16;
    int vx[ND], vy[F32 ? 1 : ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        if constexpr (F32) {
            vx[d] = 4 * h * G::PITCH + (((dim0 / 4 + 8 * d + (fr >> 2)) ^ G::vswizzle(4 * h)) << 4) + (fr & 3) * 4;
        } else {
            vx[d] = tr_row * G::PITCH + (((dim0 / 8 + 4 * d + tr_piece) ^ G::vswizzle(tr_row)) << 4) + (lane & 1) * 8;
            vy[d] = (tr_row + 8) * G::PITCH + (((dim0 / 8 + 4 * d + tr_piece) ^ G::vswizzle(tr_row + 8)) << 4) + (lane & 1) * 8;
        }
    }

    // S^T of tile t
    auto scores = [&](int t, f32x16 (&s)[NB]) {
        const unsigned char* K = K0 + (t % RING) * G::TILE + krow;
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
#pragma unroll
        for (int k = 0; k < NQ; ++k)
#pragma unroll
            for (int kb = 0; kb < NB; ++kb) {
                const float4 kf = *(const float4*)(K + kb * 32 * G::PITCH + (kx ^ (32 * k)));
                if constexpr (F32) {
                    s[kb] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf.x, qf[k].x, s[kb], 0, 0, 0);
                    s[kb] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf.y, qf[k].y, s[kb], 0, 0, 0);
                    s[kb] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf.z, qf[k].z, s[kb], 0, 0, 0);
                    s[kb] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf.w, qf[k].w, s[kb], 0, 0, 0);
                } else {
                    s[kb] = Mma32<T>::mul(*(const typename Mma<T>::frag*)&kf, *(const typename Mma<T>::frag*)&qf[k], s[kb]);
                }
            }
    };
    auto largest = [&](const f32x16 (&s)[NB]) -> float {
        float mt = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[kb][e]);
        return mt;
    };
    // -inf for the keys that the rows do not see; the rows' largest score, in units of the exponents; mt: this lane's
    // largest before. Far scores are brought to these units here, each with the rounding that their maximum has.
    float units = a.scale_log2;
    auto mask = [&](int t, f32x16 (&s)[NB], float mt) -> float {
        const int j0 = t * KT;
        const unsigned long long here = __ballot(lane < KT && there[t % RING][lane & (KT - 1)]);
        const bool some = here != (KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1);
        if (some || (a.causal && j0 + KT - 1 > wmin) || (a.window && j0 <= wmax - a.window)) {
            asm volatile("" ::: "memory");    // a branch of its own: not folded into every tile
#pragma unroll
            for (int kb = 0; kb < NB; ++kb) {
                // bit k: the row sees key j1 + k
                const int j1 = j0 + kb * 32 + 4 * h;
                unsigned bits = (unsigned)(here >> (32 * kb)) >> (4 * h);
                if (a.causal) bits &= pos - j1 >= 31 ? ~0u : pos < j1 ? 0u : (2u << (pos - j1)) - 1;
                if (a.window) {
                    const int n = pos - a.window + 1 - j1;       // so many keys of them are too far back
                    bits &= n <= 0 ? ~0u : n > 31 ? 0u : ~0u << n;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) s[kb][e] = bits & (1u << kappa(e)) ? s[kb][e] : -INFINITY;
            }
            mt = largest(s);
        }
        mt = xor32_max(mt) * a.scale_log2;
        units = a.scale_log2;
        if (__any(fabsf(mt) >= FAR && mt > -INFINITY)) {
            asm volatile("" ::: "memory");
#pragma unroll
            for (int kb = 0; kb < NB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[kb][e] *= units;
            units = 1.f;
        }
        return mt;
    };
    // tiles of which some row of the wave sees some key: [t0, tw)
    const int tw = idle ? t0 : a.causal ? min(t1, wmax < 0 ? t0 : wmax / KT + 1) : t1;

    // A wave's loop is one tile ahead with the scores: the products of tile t + 1 run under the exponentials of tile t. The
    // loads are three tiles ahead, the page ids four; a wave waits for its loads in the order it made them, so the ids go
    // before the loads of the same turn.
    if (tid < 2) odd[tid] = -1;
    if (DP > c.dim)      // places behind the head's dims are not loaded: zeros
        for (int i = tid; i < G::LDS / 16; i += NT) ((float4*)smem)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();
    if (t0 < t1) {
        f32x16 sa[NB], sb[NB];
        float mt = -INFINITY;
        pages(t0);
        bring(t0);
        pages(t0 + 1);
        if (t0 + 1 < t1) bring(t0 + 1);
        pages(t0 + 2);
        if (t0 + 2 < t1) bring(t0 + 2);
        pages(t0 + 3);
        arrive(false);
        if (t0 < tw) {
            scores(t0, sa);
            mt = mask(t0, sa, largest(sa));
        }
        bool ahead = false;              // the last 2 PER loads may still be on their way
        auto next = [&](int t) {
            if (t > t0) arrive(ahead);
            const bool more = t + 3 < t1;
            int now[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) now[i] = page[i];
            pages(t + 4);
            int then[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) { then[i] = page[i]; page[i] = now[i]; }
            if (more) bring(t + 3);
#pragma unroll
            for (int i = 0; i < PER; ++i) page[i] = then[i];
            ahead = more && full;
            clean(t);
        };
        // tile t with the scores s, the next ones into sn
        auto step = [&](int t, f32x16 (&s)[NB], f32x16 (&sn)[NB]) {
            next(t);
            // m is the maximum less LOWER at its last change: a score may pass it by LATE more before all is rescaled
            constexpr float LOW = LOWER<T, true>;
            if (__any(mt - m > LOW + LATE)) {
                asm volatile("" ::: "memory");
                const float mn = fmaxf(m, lowered<T, true>(mt)), corr = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
                l *= corr;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] *= corr;
                m = mn;
            }
            const float mu = m == -INFINITY ? 0.f : m;
            float ma = -INFINITY;
            const unsigned char* V = V0 + (t % RING) * G::TILE;
            if constexpr (F32) {
                scores(t + 1, sn);
                float p[16 * NB];
#pragma unroll
                for (int e = 0; e < 16 * NB; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 4][e & 15], units, -mu));
                    l += p[e];
                }
#pragma unroll
                for (int kb = 0; kb < NB; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const unsigned char* x = V + (kb * 32 + kappa(e)) * G::PITCH;
#pragma unroll
                        for (int d = 0; d < ND; ++d)
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(*(const float*)(x + vx[d]), p[16 * kb + e], o[d], 0, 0, 0);
                    }
                ma = largest(sn);
            } else {
                // in steps that stay in this order: a product of the next scores with its share of the exponentials,
                // then a product with the values and its share of the next maximum; fragments come AK and AV steps ahead
                constexpr int NS = NQ * NB, NP = ND * KT / 16, AK = 2, AV = 2;
                const unsigned char* K = K0 + ((t + 1) % RING) * G::TILE + krow;
                auto kread = [&](int i) {
                    return *(const float4*)(K + (i % NB) * 32 * G::PITCH + (kx ^ (32 * (i / NB))));
                };
                auto vread = [&](int i) {
                    const unsigned char* vp = V + 16 * (i / ND) * G::PITCH;
                    const v4i16 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vp + vx[i % ND]));
                    const v4i16 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vp + vy[i % ND]));
                    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                };
                Vec8<T> pb[2 * NB];
                float4 kf[AK + 1];
                v8i16 vf[AV + 1];
#pragma unroll
                for (int kb = 0; kb < NB; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sn[kb][e] = 0.f;
#pragma unroll
                for (int i = 0; i < AK; ++i) kf[i] = kread(i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    if (i + AK < NS) kf[(i + AK) % (AK + 1)] = kread(i + AK);
                    if (i + AV >= NS) vf[i + AV - NS] = vread(i + AV - NS);
                    sn[i % NB] = Mma32<T>::mul(*(const typename Mma<T>::frag*)&kf[i % (AK + 1)],
                                               *(const typename Mma<T>::frag*)&qf[i / NB], sn[i % NB]);
#pragma unroll
                    for (int e = 16 * NB * i / NS; e < 16 * NB * (i + 1) / NS; ++e) {
                        const float x = __builtin_amdgcn_exp2f(fmaf(s[e >> 4][e & 15], units, -mu));
                        l += x;
                        pb[e >> 3].x[e & 7] = from_f<T>(x);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    if (i + AV < NP) vf[(i + AV) % (AV + 1)] = vread(i + AV);
                    o[i % ND] = Mma32<T>::mul(*(const typename Mma<T>::frag*)&vf[i % (AV + 1)],
                                              *(const typename Mma<T>::frag*)&pb[i / ND], o[i % ND]);
#pragma unroll
                    for (int e = 16 * NB * i / NP; e < 16 * NB * (i + 1) / NP; ++e) ma = fmaxf(ma, sn[e >> 4][e & 15]);
                    asm volatile("" : "+v"(ma));         // here, not where it is used
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (odd[t & 1] == t) {   // values set aside reach the rows that see them (whatever their weight), and no others
                asm volatile("" ::: "memory");
                for (int k = 0; k < KT; ++k) {
                    const int j = t * KT + k;
                    if (!there[t % RING][k] || (a.causal && j > pos) || (a.window && j <= pos - a.window)) continue;
                    const int pi = c.by_page.div(j);
                    const T* x = (const T*)(c.v_head(hk) + c.v_at(page_of(c, b, pi), j - pi * c.page));
                    int d0 = dim0 + 4 * h;
                    asm volatile("" : "+v"(d0));       // nothing of this is kept ready for every tile
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) add_odd<T>(x, d0 + 32 * d + kappa(i), c.dim, o[d], i);
                }
            }
            if (t + 1 < tw) mt = mask(t + 1, sn, ma);
        };
        int t = t0;
        while (t < tw) {
            step(t++, sa, sb);
            if (t >= tw) break;
            step(t++, sb, sa);
        }
        for (; t < t1; ++t) next(t);     // the other waves' tiles
    }
    l = xor32_add(l);
    if (w0 + fr >= nrows) return;
    const int n = first + place;
    if (a.tile_splits == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        char* dst = a.o.p + ((long long)n * a.o.ts + (long long)head * a.o.hs) * E;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int dd = dim0 + 32 * d + kappa(e) + 4 * h;
                if (dd >= c.dim) continue;
                T y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = from_f<T>(l == 0.f ? 0.f : o[d][e + i] * inv);
                if constexpr (F32) *(float4*)(dst + dd * E) = *(const float4*)y;
                else *(float2*)(dst + dd * E) = *(const float2*)y;
            }
    } else {
        const long long pr = split * a.tile_part.rows + (long long)n * a.q_heads + head;
        float *dst = a.ws + pr * c.dim, *dst_ml = a.ws + a.tile_splits * a.tile_part.rows * c.dim + 2 * pr;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int dd = dim0 + 32 * d + kappa(e) + 4 * h;
                if (dd < c.dim) *(f32x4*)(dst + dd) = f32x4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
            }
        if (h == 0 && dim0 == 0) { dst_ml[0] = m; dst_ml[1] = l; }
    }
}

// The parts of a row tile: as the rows kernel takes them (blocks of kb keys), or all `splits` of the tile kernel (kb 0).
__device__ __forceinline__ int parts_in(const PagedAttnArgs& a, int b, int tile, int per, int nq, int splits, int kb) {
    if (!kb) return splits;
    const int row0 = tile * per, row1 = min(row0 + per, nq * a.group) - 1;
    return uniform(parts_of(a, span_of(a, nq, a.c.len(b), row0, row1, kb).nblk, kb));
}

// The parts that the join reads: sums of split 0's first row, maxima and sums, rows of a split.
struct PartsIn {
    const float *sum, *ml;
    long long rows;
    bool by_tile;
};
__device__ __forceinline__ PartsIn parts_at(const PagedAttnArgs& a, int kb) {
    const PagedParts& w = kb ? a.rows_part : a.tile_part;
    return PartsIn{a.ws, a.ws + (kb ? a.splits : a.tile_splits) * w.rows * a.c.dim, w.rows, w.by_tile};
}

// The same for rows of few splits, several rows to a workgroup: a group of lanes holds a row's dims, 4 a lane, and goes
// over its splits, each lane with one split's weight. 64 caches of 4096 keys in 4 parts: attention takes 222 us, 253 with a
// workgroup per row. More parts go to a workgroup per row, whose threads share them (64 parts: 7 us).
constexpr int FEW_SPLITS = 16, JOIN_TURNS = 4;
__host__ __device__ __forceinline__ int join_lanes(int dim) { return dim <= 64 ? 16 : dim <= 128 ? 32 : 64; }
template <typename T>
__global__ __launch_bounds__(256) void paged_join_few_kernel(PagedAttnArgs a, int per, int over, int upto, int splits, int kb) {
    const PagedKv& c = a.c;
    const int lanes = join_lanes(c.dim), at = threadIdx.x % lanes, groups = 256 / lanes, own = JOIN_TURNS * groups;
    const int parts = (per + own - 1) / own;
    const int unit = blockIdx.x / parts, hk = unit % c.heads;
    int b, tile, first, end;
    if (!find_tile(c, a.group, per, over, upto, unit / c.heads, threadIdx.x & 63, b, tile)) return;
    c.rows(b, first, end);
    splits = parts_in(a, b, tile, per, end - first, splits, kb);
    if (splits == 1) return;
    const int in0 = blockIdx.x % parts * own, row1 = min(tile * per + min(per, in0 + own), (end - first) * a.group);
    const PartsIn in = parts_at(a, kb);
    const int d0 = at * 4;
    for (int row = tile * per + in0 + threadIdx.x / lanes; row < row1; row += groups) {
        const int place = a.by_group.div(row), n = first + place, head = hk * a.group + row - place * a.group;
        const long long r0 = in.by_tile ? unit * 16ll + row - tile * per : (long long)n * a.q_heads + head;
        f32x4 x[FEW_SPLITS];
#pragma unroll
        for (int s = 0; s < FEW_SPLITS; ++s) {
            x[s] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (s < splits && d0 < c.dim) x[s] = *(const f32x4*)(in.sum + (s * in.rows + r0) * c.dim + d0);
        }
        float2 ml = make_float2(-INFINITY, 0.f);
        if (at < splits) ml = *(const float2*)(in.ml + 2 * (at * in.rows + r0));
        float m = ml.x;
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 16));
        m = __shfl(m, 0, lanes);
        const float w = __builtin_amdgcn_exp2f(ml.x - (m == -INFINITY ? 0.f : m));
        float l = ml.y * w;
        for (int o = 8; o > 0; o >>= 1) l += __shfl_xor(l, o, 16);
        l = __shfl(l, 0, lanes);
        f32x4 y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < FEW_SPLITS; ++s) y += x[s] * __shfl(w, s, lanes);
        if (d0 >= c.dim) continue;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T out[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = from_f<T>(l == 0.f ? 0.f : y[e] * inv);
        char* dst = a.o.p + ((long long)n * a.o.ts + (long long)head * a.o.hs + d0) * (int)sizeof(T);
        if constexpr (sizeof(T) == 4) *(float4*)dst = *(const float4*)out;
        else *(float2*)dst = *(const float2*)out;
    }
}

// Joins the splits of one query row, one workgroup each: the splits' sums scaled to their common maximum, then divided
// once. Rows are numbered as the kernel that split them did, `per` to a row tile.
template <typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, int per, int over, int upto, int splits, int kb) {
    const PagedKv& c = a.c;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int unit = blockIdx.x / per, hk = unit % c.heads;
    int b, tile, first, end;
    if (!find_tile(c, a.group, per, over, upto, unit / c.heads, lane, b, tile)) return;
    c.rows(b, first, end);
    const int row = tile * per + blockIdx.x % per;
    if (row >= (end - first) * a.group) return;
    splits = parts_in(a, b, tile, per, end - first, splits, kb);
    if (splits == 1) return;
    const int place = a.by_group.div(row), n = first + place, head = hk * a.group + row - place * a.group;
    const PartsIn in = parts_at(a, kb);
    const long long r0 = in.by_tile ? unit * 16ll + row - tile * per : (long long)n * a.q_heads + head;

    // the splits' weights (at most one per thread)
    __shared__ float ws[256], ms[4], ls[4];
    __shared__ f32x4 xs[4][64];
    const int t = threadIdx.x;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (t < splits) ml = *(const float2*)(in.ml + 2 * (t * in.rows + r0));
    const float mw = wave_max(ml.x);
    if (lane == 0) ms[wid] = mw;
    __syncthreads();
    const float m = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    const float w = __builtin_amdgcn_exp2f(ml.x - (m == -INFINITY ? 0.f : m));
    ws[t] = w;
    const float lw = wave_sum(ml.y * w);
    if (lane == 0) ls[wid] = lw;
    __syncthreads();
    // a lane holds 4 dims; the waves, and the parts of a wave that a row of dims does not fill, take splits in turn
    const int lanes = c.dim <= 64 ? 16 : c.dim <= 128 ? 32 : 64, sub = lane / lanes, d0 = (lane % lanes) * 4;
    const int step = 4 * (64 / lanes);
    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = wid * (64 / lanes) + sub; s < splits; s += step)
        if (d0 < c.dim) x += *(const f32x4*)(in.sum + (s * in.rows + r0) * c.dim + d0) * ws[s];
    for (int o = lanes; o < 64; o <<= 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], o, 64);
    }
    xs[wid][lane] = x;
    __syncthreads();
    if (wid || lane >= lanes || d0 >= c.dim) return;
    const float l = ls[0] + ls[1] + ls[2] + ls[3];
    x = xs[0][lane] + xs[1][lane] + xs[2][lane] + xs[3][lane];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = from_f<T>(l == 0.f ? 0.f : x[e] * inv);
    char* dst = a.o.p + ((long long)n * a.o.ts + (long long)head * a.o.hs + d0) * (int)sizeof(T);
    if constexpr (sizeof(T) == 4) *(float4*)dst = *(const float4*)y;
    else *(float2*)dst = *(const float2*)y;
}

template <typename T> hipError_t run_join(const PagedAttnArgs& a, long long tiles, int per, int over, int upto, int splits,
                                          int kb, hipStream_t st) {
    if (splits <= FEW_SPLITS) {
        const int own = JOIN_TURNS * 256 / join_lanes(a.c.dim);
        paged_join_few_kernel<T><<<(unsigned)(tiles * a.c.heads * ((per + own - 1) / own)), 256, 0, st>>>(a, per, over, upto, splits, kb);
    } else {
        paged_join_kernel<T><<<(unsigned)(tiles * a.c.heads * per), 256, 0, st>>>(a, per, over, upto, splits, kb);
    }
    PFM_LAUNCH_CHECK();
    return hipSuccess;
}

template <typename T, int DP, int NTILES> hipError_t run_rows(const PagedAttnArgs& a, hipStream_t st) {
    using R = DecGeom<T, DP, NTILES>;
    static_assert(R::LDS <= 150 * 1024, "LDS of a workgroup");
    const PagedKv& c = a.c;
    hipError_t e = pfm_allow_lds<paged_rows_kernel<T, DP, NTILES>>(R::LDS);
    if (e != hipSuccess) return e;
    paged_rows_kernel<T, DP, NTILES><<<dim3((unsigned)(a.rows_tiles * c.heads), a.splits), DEC_W * 64, R::LDS, st>>>(a);
    PFM_LAUNCH_CHECK();
    if (a.splits == 1) return hipSuccess;
    const int per = c.cu_q ? 16 : std::min(16, a.group);     // a sequence's rows where they are known
    return run_join<T>(a, c.cu_q ? a.rows_tiles : (long long)c.batch * ((a.group + per - 1) / per), per, 0, a.rows_upto,
                       a.splits, R::KB, st);
}
template <typename T, int DP>
hipError_t run_attention(const PagedAttnArgs& a, hipStream_t st) {
    using G = TileGeom<T, DP>;
    constexpr bool TILE = sizeof(T) == 2 || DP <= 128;     // as in pfm_paged_attention_plan
    static_assert(!TILE || G::LDS <= 150 * 1024, "LDS of a workgroup");
    const PagedKv& c = a.c;
    hipError_t e = hipSuccess;
    if (a.rows_tiles) {
        // 32-bit heads: blocks of 32 keys leave a SIMD one wave beyond 64 dims, blocks of 16 two. 34 caches of 8230 keys, 8
        // heads on 2 of 96 dims: 175 us and 115; 256 of 100 keys, 32 heads on 8 of 128, 82 and 48; 64 streams' chunks of 15
        // rows over 70 keys, 4 heads of 128, 12.5 and 11.7. Beyond 128 dims the longer block does not fit the registers.
        e = run_rows<T, DP, (sizeof(T) == 4 && DP > 64) ? 1 : 2>(a, st);
        if (e != hipSuccess) return e;
    }
    if constexpr (TILE) if (a.tiles) {
        if ((e = pfm_allow_lds<paged_tile_kernel<T, DP>>(G::LDS)) != hipSuccess) return e;
        paged_tile_kernel<T, DP><<<dim3((unsigned)(a.tiles * c.heads), a.tile_splits), G::NW * 64, G::LDS, st>>>(a);
        PFM_LAUNCH_CHECK();
        if (a.tile_splits > 1) e = run_join<T>(a, a.tiles, G::ROWS, a.rows_upto, 0x7fffffff, a.tile_splits, 0, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
template <typename T>
hipError_t run_attention(const PagedAttnArgs& a, hipStream_t st) {
    if (a.c.dim <= 64) return run_attention<T, 64>(a, st);
    if (a.c.dim <= 128) return run_attention<T, 128>(a, st);
    return run_attention<T, 256>(a, st);
}

template <typename T>
hipError_t run_append(AppendArgs a, hipStream_t st) {
    const int half = a.inv_freq ? a.rot / 2 : 0;
    constexpr int MOST = 1 << 23;           // a launch has under 2^32 threads
    for (a.row0 = 0; a.row0 < a.c.tokens; a.row0 += MOST) {
        kv_append_kernel<T><<<std::min(a.c.tokens - a.row0, MOST), AP_T, half * sizeof(float2), st>>>(a);
        PFM_LAUNCH_CHECK();
    }
    return hipSuccess;
}

}  // namespace

// Which kernels run, over how many row tiles, and into how many parts each splits a sequence's keys. The sequences'
// own lengths are on the device: sequences of at most 16 query rows (tokens x heads of a group) go to the rows kernel,
// longer ones to the tile kernel, and both are launched where the sizes known here allow both kinds.
void pfm_paged_attention_plan(int dtype, PagedAttnArgs& a) {
    const PagedKv& c = a.c;
    const long long rows = (long long)c.tokens * a.group, max_kv = (long long)c.width * c.page;
    const int tile_rows = c.dim > 128 ? 128 : 256;
    a.rows_upto = 16;
    // Up to 128 dims the rows kernel takes little work whole: row tiles of 16 are that many more workgroups, and a wave's
    // chain is shorter. The work is row tiles x keys x dims (of all the table reaches: the workspace does not know a window).
    // Measured, rows against tile kernel, at 4 10^6 (6 10^6): 12 us and 15 (64 dims), 15 and 17 (128), 31 and 37 (128, f32);
    // at 16 10^6: 22 and 27 (128), 32 and 61 (128, f32); at 23 10^6: 22 and 19 (64); at 47 10^6: 35 and 26 (128).
    const long long fine = (rows + 15ll * std::min<long long>(c.batch, rows)) / 16;
    const bool little = c.dim <= 128 && (double)fine * c.heads * max_kv * c.dim <= 2e7;
    if (!c.cu_q || little || (dtype == DT_F32 && c.dim > 128)) {   // group rows each; or: too many registers for the tile kernel
        a.rows_upto = 0x7fffffff;
        a.rows_tiles = c.cu_q ? fine : (long long)c.batch * ((a.group + 15) / 16);
        a.tiles = 0;
    } else {
        a.rows_tiles = c.batch;
        if (c.batch == 1 && rows > 16) {             // the tile kernel takes it, whatever its length is
            a.rows_upto = 0;
            a.rows_tiles = 0;
        }
        // sequences of more than 16 rows, each with one tile that is not full
        a.tiles = (rows + std::min<long long>(c.batch, rows / 17) * (tile_rows - 1)) / tile_rows;
        if (rows <= 16) a.tiles = 0;
    }
    // keys that one row tile sees at most: with a window its first row's reach and the rows' own span
    auto parts = [&](long long units, long long keys, long long fill, long long least) {
        if (!units) return 1;
        const long long most = keys / least, want = (fill + units * c.heads - 1) / (units * c.heads);
        return (int)std::max(1ll, std::min(std::min(want, most), 256ll));
    };
    auto seen = [&](int rows) {
        return a.window ? std::min<long long>(max_kv, (long long)a.window + rows + (a.causal ? 0 : rows == 16 ? std::min(a.rows_upto, c.tokens) : c.tokens)) : max_kv;
    };
    // (parts of 256 keys at least: 32 caches of 1000 keys take 32 us, 36 in parts of 128; 4 of 2048 16 us, 20 in parts of 512)
    // Few caches in many parts: as many workgroups as the chip holds at once. 2 of 131072 keys, 32 heads on 8, 202 us and 217
    // with twice as many; 8 of up to 32768 167 and 174. Many caches of different lengths: twice as many, for an even
    // end. 64 of up to 16384 keys 441 and 494 with half as many (of 9216 keys each 435 and 423).
    a.fill = parts(a.rows_tiles, seen(16), a.rows_tiles * c.heads <= 128 ? 1024 : 2048, PART_MIN);
    a.splits = a.fill;
    if (a.rows_tiles) {      // for long sequences among short ones; 2^14 workgroups that end at once take 10 us
        const long long units = a.rows_tiles * c.heads, most = (seen(16) + PART_MAX - 1) / PART_MAX;
        a.splits = (int)std::max<long long>(a.fill, std::min({most, (1ll << 14) / units, 256ll}));
    }
    // The tile kernel has one workgroup per CU at a time. Split into n parts, its row tiles take so many turns of the 256
    // CUs, each as long as a part and what a part costs beside its keys; the parts' sums are written and read once more.
    // Past one turn, tiles of several sequences end apart, and the last turn is taken as half full. Measured at 128 dims:
    // 2.3 us a tile of 64 keys in 16 bits, 9 us one of 32 in 32 bits, 3 us beside, 4 us the join. 256 new tokens of 64
    // heads, each with its own cache of 8192 keys: 289 us whole, 182 in 2 parts, 114 in 4, 130 in 8; 8 sequences of 512
    // tokens over themselves, 32 heads on 8: 61 whole, 109 in 2.
    a.tile_splits = 1;
    if (a.tiles) {
        // row tiles that have work: as if all sequences were as long as each other
        const long long per = (rows + c.batch - 1) / c.batch;
        const double units = (double)std::min<long long>(a.tiles, c.batch * ((per + tile_rows - 1) / tile_rows)) * c.heads;
        const double wide = c.dim <= 64 ? 0.5 : c.dim <= 128 ? 1.0 : 1.5;
        const double tile_us = (dtype == DT_F32 ? 9.0 : 2.3) * wide;
        auto best_of = [&](long long keys, int most) {
            const double n_tiles = keys / (dtype == DT_F32 ? 32.0 : 64.0);
            double best = 1e30;
            int parts = 1;
            for (int n = 1; n <= most && n <= n_tiles / 2 + 1; ++n) {
                const double join = n > 1 ? 4.0 + units * tile_rows * c.dim * 8.0 * n / 4e6 : 0.0;
                const double turns = units * n / 256, ends = c.batch > 1 && turns > 1.0 ? turns + 0.5 : ceil(turns);
                const double us = ends * (ceil(n_tiles / n) * tile_us + 3.0) + join;
                if (us < best) { best = us; parts = n; }
            }
            return parts;
        };
        // Beyond 8 turns of all parts there is nothing left to fill up, and their sums would take gigabytes behind a table that
        // reaches far: 64 single tokens and a chunk of 2048 tokens over 8192 keys, a table of 131072, 641 us in 8 parts and 568
        // in 3; one prompt of 8800 tokens over 17000 keys 2100 us in 2, 2081 whole. (No more than 4 turns: 4500 tokens over
        // 40000 keys 3030 us in 3 parts, 3800 whole. From 2^16 tiles on a launch of the join would not hold all rows.)
        const int most = a.tiles * c.heads < 65536 ? (int)std::max(1.0, std::min(64.0, 2048 / units)) : 1;
        a.tile_splits = best_of(max_kv, most);
        if (a.window) a.tile_splits = best_of(seen(tile_rows), a.tile_splits);     // the workspace is that of no window
    }
    // The rows kernel takes few of a call's rows where the tile kernel is there too: numbered by its row tiles they need
    // no more than 16 places for each sequence and kv head.
    a.tile_part = {(long long)c.tokens * a.q_heads, false};
    a.rows_part = a.tile_part;
    if (c.cu_q && a.rows_tiles * c.heads * 16 < a.rows_part.rows) a.rows_part = {a.rows_tiles * c.heads * 16, true};
}
hipError_t pfm_paged_attention(int dtype, const PagedAttnArgs& a, hipStream_t st) {
    if (dtype == DT_F32) return run_attention<float>(a, st);
    if (dtype == DT_BF16) return run_attention<bf16>(a, st);
    return run_attention<f16>(a, st);
}
hipError_t pfm_kv_append(int dtype, const AppendArgs& a, hipStream_t st) {
    if (dtype == DT_F32) return run_append<float>(a, st);
    if (dtype == DT_BF16) return run_append<bf16>(a, st);
    return run_append<f16>(a, st);
}
