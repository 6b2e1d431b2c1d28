// Drawing one token per row of logits with temperature, top-k, top-p and min-p from a given uniform number.
//
// p_i = exp((x_i - max x) / T). Tokens are ordered by logit, the larger first, ties by index, the smaller first. Kept
// are the first top_k of that order, of these the ones before which less than top_p of their mass lies, of these the
// ones with p_i >= min_p: each filter keeps a prefix of the order, so the kept set is one prefix, given by its last
// element (value, index). The answer is the first kept index in the vocabulary's order whose running sum of p exceeds
// u times the kept mass.
//
// Masses are whole numbers, p_i 2^43 rounded to nearest: their sums do not depend on the order of additions, so the
// answer is the same for every split of a row over threads and workgroups, and their error stays under half a step of
// 2^-43 of the largest probability per token. p itself is computed in 64 bits; tokens under 2^-44 of the largest one's
// probability weigh nothing. A row of 2^20 equal logits sums to 2^63.
//
// One read of the logits is what it cannot do without. Short rows take one workgroup and one read; others a chain of
// kernels over chunks of rows, in which a row reads its logits again only where its filters need it: the maxima (memory
// bounds them), then sums, few candidates or a histogram of masses (64-bit exponentials and atomics bound it), then one
// workgroup per row on what is left (instructions that a lone workgroup fetches and waits for bound it). 256 rows of 131071
// logits in 32 bits, 134 MB, us: maxima 21, and with top-p 0.9 at temperature 1.4, when the nucleus is wide, histograms 44,
// the nucleus' bin 18, its tokens 17, the cut and the draw 33, 140 in all (a copy's rate would give 25); with top-k 50 and
// top-p 60 in all, without filters 62 (maxima 21, sums 33, the draw 13), the largest logit alone 29. One row of 8404 logits: 9
// (the largest alone) .. 11 (no filter), 12 with top-k 15 or 50, 20 with top-k 196 (more than FEW tokens), 22 with a wide
// nucleus. The likely tokens of a row should lie scattered: with the upper two thirds of the vocabulary at -inf, or logits
// that fall with the index, more candidates pass than the list holds, and one workgroup goes over the whole row again
// (256 x 131071, top-p 0.9: 190 and 451 where scattered ones take 131; 64 x 128000 in 16 bits 141 and 320 for 64).
//
// NaN logits are never drawn. If the largest logit is +inf, the tokens that have it share the mass; a row without any
// logit above -inf has no token: -1 with probability 0.
#include <algorithm>

#include "pfm_serve.h"

namespace {

typedef unsigned long long u64;
constexpr int SW = 16, ST = SW * 64;    // waves and threads of a row's workgroup
constexpr int CW = 4, CT = CW * 64;     // and of a chunk's
constexpr int BINS = 2048;              // equal steps of (max - x) / T over [0, SPAN)
constexpr float SPAN = 31.f;            // 2^-44 is e^-30.5
constexpr int LIST = 2048;              // tokens of one bin that are sorted at once
constexpr int CAND = 6144;              // candidates of a row that are worked on in LDS
constexpr int FEW = 256;                // tokens that are ranked by comparing each with each: 9 us less than sorting
constexpr int SEG = 512;                // of these, as many as one wave of a chunk may find
constexpr int GROUPS = 1024;            // maxima of parts of a row, at most
constexpr int CHUNKS = 64;              // chunks of a row, at most
constexpr int PARTS = CHUNKS * CW;      // and of what their waves go over
constexpr u64 OVER = 1u << 24;          // added to a list's count: a wave found more than SEG

// orders floats as unsigned numbers; -0 is +0's equal, as in a comparison
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ u64 shfl_up_u64(u64 v, int o) {
    return (u64)__shfl_up((long long)v, o, 64);
}
__device__ __forceinline__ u64 shfl_u64(u64 v, int l) { return (u64)__shfl((long long)v, l, 64); }
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += (u64)__shfl_xor((long long)v, o, 64);
    return v;
}
__device__ __forceinline__ u64 wave_scan_u64(u64 v, int lane) {   // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 x = shfl_up_u64(v, o);
        if (lane >= o) v += x;
    }
    return v;
}

struct Row {
    float max;
    double scale;        // EXPS log2(e) / T
    float bin_scale;     // 2 BINS / (SPAN T)
};

constexpr int EXPS = 1024;               // a table of 2^(j / EXPS)
struct ExpTable {
    double x[EXPS];
    constexpr ExpTable() : x() {
        for (int j = 0; j < EXPS; ++j) {
            const double a = 0.69314718055994530942 * j / EXPS;
            double y = 1.0;
            for (int n = 22; n > 0; --n) y = 1.0 + y * a / n;      // the series of e^a, from its small end
            x[j] = y;
        }
    }
};
__device__ constexpr ExpTable EXP_TABLE{};
__device__ __forceinline__ void load_exps(double* table, int tid, int nt) {
    for (int i = tid; i < EXPS / 2; i += nt) ((double2*)table)[i] = ((const double2*)EXP_TABLE.x)[i];
}

// p 2^43 as a whole number, p = 2^(t / EXPS) with t = (x - max) EXPS log2(e) / T = k + f, |f| <= 1/2: the table's
// 2^(k mod EXPS / EXPS) times the series of 2^(f / EXPS) to the third power (the rest is under 6e-16), with k's upper part
// added to the exponent. Rounding to whole numbers is an addition each time: of 1.5 2^52 for k, of 2^9 for p. A NaN or
// what lies far below is raised to where p 2^43 rounds to 0. max is finite.
__device__ __forceinline__ u64 mass(float x, const Row& r, const double* exp_table) {
    constexpr double L = 0.69314718055994530942 / EXPS;
    const double t = __builtin_fmax(((double)x - (double)r.max) * r.scale, -46.0 * EXPS);
    const double kd = t + 6755399441055744.0;
    const int k = (int)__double2loint(kd);
    const double f = t - (kd - 6755399441055744.0);
    const double e = exp_table[k & (EXPS - 1)];
    double q = fma(f, L * L * L / 6, L * L / 2);
    q = fma(q, f, L);
    const double p = fma(q * f, e, e);
    const double w = __hiloint2double(__double2hiint(p) + (int)(((unsigned)k << 10) & 0xfff00000u), __double2loint(p)) + 512.0;
    return (u64)__double_as_longlong(w) & ((1ull << 52) - 1);
}
// (max - x) / T in bins; monotone in x (halves: the difference does not overflow), NaN for NaN
__device__ __forceinline__ float steps(float x, const Row& r) {
    return x == r.max ? 0.f : (0.5f * r.max - 0.5f * x) * r.bin_scale;
}
__device__ __forceinline__ int bin_of(float x, const Row& r) {   // BINS: weighs nothing
    const float d = steps(x, r);
    return d < (float)BINS ? (int)d : BINS;
}

// a value that all tokens with steps(x) < d reach, and little more
__device__ __forceinline__ float value_at(float d, const Row& r) {
    return r.max - 2.f * (d / r.bin_scale) * 1.000001f - (fabsf(r.max) * 2e-6f + 1e-37f);
}

// a value that no token with steps(x) >= d passes, and little more
__device__ __forceinline__ float value_below(float d, const Row& r) {
    return r.max + ((fabsf(r.max) * 2e-6f + 1e-37f) - 2.f * (d / r.bin_scale) * 0.999999f);
}

template <typename T> struct Pack { static constexpr int N = 16 / sizeof(T); T x[N]; };

// f(index, value) for the elements [e0, e1) of a row, by `waves` waves of which this is number `wave`; wide loads, U under
// way, where they lie inside. All lanes of a wave call f together; those without an element give it a NaN.
template <int U, typename T, typename F>
__device__ __forceinline__ void each(const T* x, int e0, int e1, int wave, int waves, F f) {
    constexpr int N = Pack<T>::N;
    const int lane = threadIdx.x & 63;
    const float none = __uint_as_float(0x7fc00000u);
    const int skew = (int)(((uintptr_t)x / sizeof(T)) % N);   // elements of x's first 16 bytes that lie before it
    const int v0 = (e0 + skew + N - 1) / N, v1 = (e1 + skew) / N;
    if (v1 <= v0) {
        for (int i = e0 + wave * 64; i < e1; i += waves * 64) f(i + lane, i + lane < e1 ? to_f(x[i + lane]) : none);
        return;
    }
    const int head = v0 * N - skew, tail = v1 * N - skew;     // [e0, head) and [tail, e1): fewer than N each
    if (wave == 0) {
        if (e0 < head) f(e0 + lane, e0 + lane < head ? to_f(x[e0 + lane]) : none);
        if (tail < e1) f(tail + lane, tail + lane < e1 ? to_f(x[tail + lane]) : none);
    }
    const Pack<T>* p = (const Pack<T>*)__builtin_assume_aligned(x - skew, 16);
    int v = v0 + wave * 64;
    for (; v + (U - 1) * waves * 64 + 64 <= v1; v += U * waves * 64) {
        Pack<T> q[U];
#pragma unroll
        for (int k = 0; k < U; ++k) q[k] = p[v + lane + k * waves * 64];
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                f((v + lane + k * waves * 64) * N - skew + j, to_f(q[k].x[j]));
                if (j % 2) __builtin_amdgcn_sched_barrier(0);     // two at a time: more do not fit the registers
            }
    }
    for (; v < v1; v += waves * 64) {
        const bool in = v + lane < v1;
        Pack<T> q;
        if (in) q = p[v + lane];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            f((v + lane) * N - skew + j, in ? to_f(q.x[j]) : none);
            if (j % 2) __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// The same by single elements, four under way: for workgroups that are alone with a row, where the time goes into fetching
// the code of long unrolled loops.
template <typename T, typename F>
__device__ __forceinline__ void each_one(const T* x, int e0, int e1, int wave, int waves, F f) {
    const int lane = threadIdx.x & 63, step = waves * 64;
    for (int i = e0 + wave * 64; i < e1; i += 4 * step) {
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int j = i + k * step + lane;
            v[k] = j < e1 ? to_f(x[j]) : __uint_as_float(0x7fc00000u);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) f(i + k * step + lane, v[k]);
    }
}

struct Lds {
    double exp_table[EXPS];
    u64 hist_w[BINS];
    unsigned hist_n[BINS];
    u64 list[LIST];          // ~key << 32 | index: ascending is the order of tokens
    u64 cand[CAND];          // the same
    ulonglong2 few[FEW];     // entries with their masses
    u64 wsum[SW], part[PARTS];
    unsigned n_list;
    u64 b0, b1;              // broadcasts
    int i0, i1;
};
__device__ __forceinline__ u64 entry(int i, float f) { return (u64)~order_key(f) << 32 | (uint32_t)i; }
__device__ __forceinline__ int entry_index(u64 e) { return (int)(uint32_t)e; }
__device__ __forceinline__ float entry_value(u64 e) { return key_value(~(uint32_t)(e >> 32)); }

// Appends the entries of the lanes that have one to a list in LDS; n counts on past the list's end.
__device__ __forceinline__ void push(u64* list, unsigned& n, unsigned cap, bool have, int i, float f) {
    const unsigned long long who = __ballot(have);
    if (!have) return;
    const int lane = threadIdx.x & 63, leader = __ffsll((long long)who) - 1;
    unsigned at = 0;
    if (lane == leader) at = atomicAdd(&n, (unsigned)__popcll(who));
    at = __shfl(at, leader, 64) + __popcll(who & ((1ull << lane) - 1));
    if (at < cap) list[at] = entry(i, f);
}

// The last kept token of the order: every token with a larger key is kept, of the equal ones those up to `index`.
struct Cut {
    uint32_t key;
    int index;
};
__device__ __forceinline__ bool kept(float x, int i, const Cut& c) {
    const uint32_t k = order_key(x);
    return k > c.key || (k == c.key && i <= c.index);
}

// block-wide inclusive scan of one value per thread; wsum: a place per wave
template <int W>
__device__ __forceinline__ u64 block_scan(u64 v, u64* wsum, int tid, u64& total) {
    const int lane = tid & 63, wid = tid >> 6;
    u64 x = wave_scan_u64(v, lane);
    __syncthreads();
    if (lane == 63) wsum[wid] = x;
    __syncthreads();
    u64 before = 0, t = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const u64 y = wsum[w];
        if (w < wid) before += y;
        t += y;
    }
    total = t;
    return x + before;
}

// The first bin in which the running count reaches `want` >= 1; what lies before it. BINS: none does, and all lies before.
template <int W, typename H>
__device__ int find_bin(const H* hist, u64* wsum, int* i0, u64* b0, int tid, u64 want, u64& before) {
    constexpr int PER = BINS / (W * 64);
    u64 n = 0, total;
#pragma unroll
    for (int j = 0; j < PER; ++j) n += hist[tid * PER + j];
    u64 at = block_scan<W>(n, wsum, tid, total) - n;
    if (tid == 0) { *i0 = BINS; *b0 = total; }
    __syncthreads();
    if (at < want && at + n >= want) {
        int j = 0;
        for (; j < PER - 1 && at + hist[tid * PER + j] < want; ++j) at += hist[tid * PER + j];
        *i0 = tid * PER + j;
        *b0 = at;
    }
    __syncthreads();
    const int bin = *i0;
    before = *b0;
    __syncthreads();
    return bin;
}
// By counts, with the masses before the bin as well.
__device__ int find_bin_n(Lds& s, int tid, u64 want, u64& n_before, u64& w_before) {
    const int bin = find_bin<SW>(s.hist_n, s.wsum, &s.i0, &s.b0, tid, want, n_before);
    u64 w = 0;
    for (int i = tid; i < bin; i += ST) w += s.hist_w[i];
    block_scan<SW>(w, s.wsum, tid, w_before);
    return bin;
}
__device__ int find_bin_w(Lds& s, int tid, u64 want, u64& w_before) {
    return find_bin<SW>(s.hist_w, s.wsum, &s.i0, &s.b0, tid, want, w_before);
}

// ascending, n a power of two <= LIST. A thread has one pair; pairs up to 64 apart stay within its wave's 128 elements.
__device__ void sort_list(u64* a, int n, int tid) {
    static_assert(LIST <= 2 * ST, "one pair per thread");
    bool wide = true;
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (wide || j > 64) __syncthreads();
            else __builtin_amdgcn_wave_barrier();
            wide = j > 64;
            if (tid < n / 2) {
                const int lo = 2 * tid - (tid & (j - 1)), hi = lo + j;
                const u64 x = a[lo], y = a[hi];
                if ((x > y) == ((lo & k) == 0)) { a[lo] = y; a[hi] = x; }
            }
        }
    __syncthreads();
}
// s.list's n entries in ascending order
__device__ void sort_entries(Lds& s, int n, int tid) {
    int p2 = 2;
    while (p2 < n) p2 <<= 1;
    for (int i = n + tid; i < p2; i += ST) s.list[i] = ~0ull;
    sort_list(s.list, p2, tid);
}

// Sums over s.few's n entries, `sum`med by the four threads of entry tid / 4 and known to each of them afterwards.
template <typename F> __device__ __forceinline__ void over_few(Lds& s, int n, int tid, F sum) {
    for (int j = tid & 3; j < n; j += 16) {
        ulonglong2 o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = s.few[min(j + 4 * k, FEW - 1)];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (j + 4 * k < n) sum(o[k]);
    }
}
__device__ __forceinline__ u64 four_sum(u64 v) {
    v += (u64)__shfl_xor((long long)v, 1, 64);
    return v + (u64)__shfl_xor((long long)v, 2, 64);
}
// n <= FEW entries get(i) and their masses into s.few; entry tid / 4 (tid < 4 n), the number of entries before it and their
// mass
template <typename G>
__device__ u64 rank_few(Lds& s, int n, int tid, const Row& r, G get, u64& rank, u64& before) {
    static_assert(4 * FEW <= ST, "four threads per entry");
    if (tid < n) {
        const u64 e = get(tid);
        s.few[tid] = make_ulonglong2(e, mass(entry_value(e), r, s.exp_table));
    }
    __syncthreads();
    const u64 e = tid < 4 * n ? s.few[tid >> 2].x : 0;
    u64 c = 0, w = 0;
    if (tid < 4 * n) over_few(s, n, tid, [&](const ulonglong2& o) {
        const bool ahead = o.x < e;
        c += ahead;
        w += ahead ? o.y : 0;
    });
    rank = four_sum(c);
    before = four_sum(w);
    return e;
}

// The token of bin `bin` at which the running count (or mass), *_before ahead of the bin, reaches `want`; and the mass of
// all tokens up to it. s.list holds the bin's s.n_list tokens if they fit; all(f) goes over a set that has the bin's.
template <typename All>
__device__ Cut find_cut(All all, int V, const Row& r, Lds& s, int tid, int bin, bool by_mass, u64 n_before,
                        u64 w_before, u64 want, u64& mass_to) {
    const int n = (int)s.n_list;
    __syncthreads();
    if (n <= FEW) {
        u64 rank, before;
        const u64 e = rank_few(s, n, tid, r, [&](int i) { return s.list[i]; }, rank, before);
        const u64 w = tid < 4 * n ? s.few[tid >> 2].y : 0;
        const u64 at = by_mass ? before + w_before : rank + n_before, after = at + (by_mass ? w : 1);
        if (tid < 4 * n && !(tid & 3) && at < want && after >= want) { s.b0 = e; s.b1 = before + w + w_before; }
        __syncthreads();
        const u64 last = s.b0;
        mass_to = s.b1;
        __syncthreads();
        return Cut{~(uint32_t)(last >> 32), entry_index(last)};
    }
    if (n <= LIST) {
        sort_entries(s, n, tid);
        u64 base_n = n_before, base_w = w_before, total;
        for (int i0 = 0; i0 < n; i0 += ST) {
            const int i = i0 + tid;
            const u64 w = i < n ? mass(entry_value(s.list[i]), r, s.exp_table) : 0;
            const u64 to = block_scan<SW>(w, s.wsum, tid, total) + base_w;
            const u64 at = by_mass ? to - w : base_n + tid, after = by_mass ? to : base_n + tid + 1;
            if (i < n && at < want && after >= want) { s.i0 = i; s.b1 = to; }
            base_w += total;
            base_n += ST;
        }
        __syncthreads();
        const u64 at = s.list[s.i0];
        mass_to = s.b1;
        __syncthreads();
        return Cut{~(uint32_t)(at >> 32), entry_index(at)};
    }
    // too many to sort: the bin's keys digit by digit, then the equal ones by index
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        u64* dw = s.list;                  // [256] masses, [256] counts
        u64* dn = s.list + 256;
        for (int i = tid; i < 512; i += ST) s.list[i] = 0;
        __syncthreads();
        const uint32_t above = shift == 24 ? 0u : ~0u << (shift + 8);
        all([&](int i, float f) {
            const uint32_t k = order_key(f);
            if ((k & above) == prefix && bin_of(f, r) == bin) {
                atomicAdd(&dw[(k >> shift) & 255], mass(f, r, s.exp_table));
                atomicAdd(&dn[(k >> shift) & 255], 1ull);
            }
        });
        __syncthreads();
        u64 w = 0, c = 0, t;
        const int digit = 255 - tid;       // the larger first
        if (tid < 256) { w = dw[digit]; c = dn[digit]; }
        const u64 w1 = block_scan<SW>(w, s.wsum, tid, t) + w_before, c1 = block_scan<SW>(c, s.wsum, tid, t) + n_before;
        __syncthreads();
        const u64 to = by_mass ? w1 : c1, mine = by_mass ? w : c;
        if (tid < 256 && to - mine < want && to >= want) {
            s.i0 = digit;
            s.b0 = c1 - c;
            s.b1 = w1 - w;
        }
        __syncthreads();
        prefix |= (uint32_t)s.i0 << shift;
        n_before = s.b0;
        w_before = s.b1;
        __syncthreads();
    }
    const u64 each_w = mass(key_value(prefix), r, s.exp_table);
    // of the equal ones the first `take` are kept: the index of the last, in parts of the vocabulary that get smaller
    const u64 take = by_mass ? (want - w_before + each_w - 1) / each_w : want - n_before;
    mass_to = w_before + take * each_w;
    int e0 = 0, e1 = V;
    u64 left = take;
    while (e1 - e0 > 1) {
        const int part = (e1 - e0 + 511) / 512;
        for (int i = tid; i < 512; i += ST) s.list[i] = 0;
        __syncthreads();
        all([&](int i, float f) {
            if (i >= e0 && i < e1 && order_key(f) == prefix) atomicAdd(&s.list[(i - e0) / part], 1ull);
        });
        __syncthreads();
        u64 t;
        const u64 c = tid < 512 ? s.list[tid] : 0, to = block_scan<SW>(c, s.wsum, tid, t);
        __syncthreads();
        if (tid < 512 && to - c < left && to >= left) { s.i0 = tid; s.b0 = to - c; }
        __syncthreads();
        e0 += s.i0 * part;
        e1 = min(e0 + part, e1);
        left -= s.b0;
        __syncthreads();
    }
    return Cut{prefix, e0};
}

// ---- a row's settings and what the kernels leave for each other
struct Setting {
    Row r;
    float u, top_p, min_p;
    int top_k;
    bool greedy, by_k, by_p, by_min;
    u64 least;            // min-p in masses: p_i >= min_p  <=>  mass >= min_p 2^43, to the rounding of a mass
};
__device__ __forceinline__ bool is_greedy(const SampleArgs& a, int b) {
    return a.temperature && !(a.temperature[b] > 0.f);
}
__device__ __forceinline__ Setting setting(const SampleArgs& a, int b, float top) {
    Setting g;
    const double T = a.temperature ? fmin(fmax((double)a.temperature[b], 1e-30), 1e30) : 1.0;   // the bins' steps stay finite
    g.greedy = is_greedy(a, b);
    g.r = Row{top, EXPS * 1.4426950408889634074 / T, (float)(2.0 * BINS / (SPAN * T))};
    g.u = a.u[b];
    g.top_k = a.top_k ? a.top_k[b] : 0;
    g.top_p = a.top_p ? a.top_p[b] : 1.f;
    g.min_p = a.min_p ? a.min_p[b] : 0.f;
    g.by_k = g.top_k > 0 && g.top_k < a.vocab;
    g.by_p = g.top_p < 1.f;                           // a NaN is off
    g.by_min = g.min_p > 0.f;
    g.top_p = fmaxf(g.top_p, 0.f);
    g.least = g.by_min ? max((u64)1, (u64)ceil(fmin((double)g.min_p, 1.0) * 8796093022208.0)) : 1;
    return g;
}
// the answer is the first token whose running sum is larger
__device__ __forceinline__ u64 aim(const Setting& g, u64 total) {
    const double t = floor((g.u > 0.f ? (double)g.u : 0.0) * (double)total);
    return t >= (double)total ? total - 1 : (u64)t;
}
// the mass at which top-p ends; the first token is kept in any case
__device__ __forceinline__ u64 nucleus(const Setting& g, u64 total) {
    const double want = ceil((double)g.top_p * (double)total);
    return want < 1.0 ? 1 : want >= (double)total ? total : (u64)want;
}

// The step below which the tokens are that may be kept (a bin or two more than the bound, for the steps' own rounding).
// kth_bin: the bin that the k-th largest of some tokens is in.
__device__ __forceinline__ float candidate_limit(const Setting& g, int V, int kth_bin) {
    float limit = (float)BINS;
    if (g.by_k) limit = fminf(limit, kth_bin + 1.f);
    else if (g.by_p) limit = fminf(limit, logf((float)V / (1.f - g.top_p)) * (1.0001f * BINS / SPAN) + 2.f);
    if (g.by_min && !(g.by_k && g.by_p)) limit = fminf(limit, -logf(fminf(g.min_p, 1.f)) * (1.0001f * BINS / SPAN) + 2.f);
    return limit;
}

enum { DONE, SUMS, NARROW, WIDE, FULL, INFS };  // how a row is done; DONE: by its maxima alone
struct RowWs {                           // one per row
    u64 list[CAND];
    u64 part[PARTS];                     // masses: SUMS, INFS: of the waves' parts; others: of the chunks
    float groups[GROUPS];                // maxima of parts of the row
    float top[CHUNKS];                   // maxima of the chunks
    int top_at[CHUNKS];                  // their first index, for the largest logit alone
    u64 n_list;
    u64 total, want, before;             // WIDE: all mass, the nucleus' mass, the mass ahead of `bin`
    int kind, bin;
};
struct Plan {
    int chunks, chunk;                   // chunks of a row and elements of a chunk, a multiple of CW
    int groups;                          // maxima that a chunk leaves
    RowWs* rows;
    u64* hist;                           // [batch][chunks][BINS]
};

__device__ __forceinline__ float row_max(const RowWs& w, int chunks, int lane) {
    return wave_max(lane < chunks ? w.top[lane] : -INFINITY);
}

// First: the maxima of each chunk and of its parts.
template <typename T>
__global__ __launch_bounds__(CT) void sample_max_kernel(SampleArgs a, Plan p) {
    __shared__ float wmax[CW];
    __shared__ int wat[CW];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, c = blockIdx.y, b = blockIdx.x;
    const T* x = (const T*)a.x + (long long)b * a.ld;
    const int e0 = min(c * p.chunk, a.vocab), e1 = min(e0 + p.chunk, a.vocab);
    RowWs& w = p.rows[b];
    float mine = -INFINITY;
    int at = 0x7fffffff;
    if (is_greedy(a, b)) {
        each<2>(x, e0, e1, wid, CW, [&](int i, float f) {
            if (f > mine || (f == mine && i < at && f > -INFINITY)) { mine = f; at = i; }
        });
    } else {
        each<4>(x, e0, e1, wid, CW, [&](int i, float f) { mine = fmaxf(mine, f); });
    }
    float m = mine;
    const int per = CT / p.groups;          // lanes of a part: a power of two up to 16
    for (int o = 1; o < 64; o <<= 1) {
        if (o == per && lane % per == 0) w.groups[c * p.groups + tid / per] = m;
        m = fmaxf(m, __shfl_xor(m, o, 64));
    }
    int first = mine == m ? at : 0x7fffffff;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
    if (lane == 0) { wmax[wid] = m; wat[wid] = first; }
    __syncthreads();
    if (tid) return;
    for (int k = 1; k < CW; ++k) {
        if (wmax[k] > m || (wmax[k] == m && wat[k] < first)) { m = wmax[k]; first = wat[k]; }
    }
    w.top[c] = m;
    w.top_at[c] = first;
    if (c == 0) { w.n_list = 0; w.kind = DONE; }
}

struct ChunkLds {
    double exp_table[EXPS];
    u64 data[CW * SEG > BINS ? CW * SEG : BINS];      // the waves' candidates, or a histogram
    u64 wsum[CW];
    u64 b0;
    int i0;
};
// the waves' candidates to the row's list
__device__ __forceinline__ void hand_over(RowWs& w, const u64* own, int n, int lane) {
    u64 at = 0;
    if (lane == 0 && n) at = atomicAdd(&w.n_list, n > SEG ? OVER : (u64)n);
    at = shfl_u64(at, 0);
    for (int i = lane; i < min(n, SEG); i += 64)
        if (at + i < CAND) w.list[at + i] = own[i];
}

// Second: what each row needs of its chunks.
//   SUMS    no filter but min-p: the masses of the chunks
//   NARROW  the tokens that may be kept, few, into the row's list. What bounds them from the maxima:
//             top-k  the GROUPS maxima are as many tokens; what lies under the k-th of them is not among the k largest
//             top-p  a token with less than (1 - top_p) / V of the largest one's probability has, with all that are smaller
//                    still, less than 1 - top_p of the mass: it lies behind the nucleus (its mass counts, it does not)
//             min-p  by definition (with both others the nucleus is of all k: no bound)
//   WIDE    top-p alone, where nearly every part's maximum may be kept: a histogram of the masses of each chunk
//   INFS    the largest logit is +inf
template <typename T>
__global__ __launch_bounds__(CT, 4) void sample_scan_kernel(SampleArgs a, Plan p) {
    __shared__ ChunkLds s;
    constexpr int U = sizeof(T);             // loads of 16 logits under way where each becomes a mass: what the registers hold
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, c = blockIdx.y, b = blockIdx.x;
    const T* x = (const T*)a.x + (long long)b * a.ld;
    const int e0 = min(c * p.chunk, a.vocab), e1 = min(e0 + p.chunk, a.vocab);
    const int q0 = min(e0 + wid * (p.chunk / CW), e1), q1 = min(q0 + p.chunk / CW, e1);    // this wave's part
    RowWs& w = p.rows[b];
    const float mx = row_max(w, p.chunks, lane);
    if (mx == -INFINITY || is_greedy(a, b)) return;
    if (mx == INFINITY) {                 // the tokens at +inf share the mass: their number
        u64 sum = 0;
        each<4>(x, q0, q1, 0, 1, [&](int i, float f) { sum += f == INFINITY; });
        sum = wave_sum_u64(sum);
        if (lane == 0) w.part[c * CW + wid] = sum;
        if (c == 0 && tid == 0) w.kind = INFS;
        return;
    }
    const Setting g = setting(a, b, mx);
    const Row r = g.r;
    load_exps(s.exp_table, tid, CT);

    const int parts = p.chunks * p.groups;
    int kth = BINS;
    if (g.by_k) {
        unsigned* n = (unsigned*)s.data;
        for (int i = tid; i < BINS; i += CT) n[i] = 0;
        __syncthreads();
        for (int i = tid; i < parts; i += CT) {
            const int bin = bin_of(w.groups[i], r);
            if (bin < BINS) atomicAdd(&n[bin], 1u);
        }
        __syncthreads();
        u64 before;
        kth = find_bin<CW>(n, s.wsum, &s.i0, &s.b0, tid, g.top_k, before);
    }
    const float limit = candidate_limit(g, a.vocab, kth);
    int kind = g.by_k ? NARROW : SUMS;
    if (g.by_p && !g.by_k) {
        int pass = 0;
        for (int i = tid; i < parts; i += CT) pass += steps(w.groups[i], r) < limit;
        u64 all;
        block_scan<CW>(pass, s.wsum, tid, all);
        kind = (int)all < parts - parts / 64 ? NARROW : WIDE;
    }
    if (c == 0 && tid == 0) w.kind = kind;
    __syncthreads();

    u64 sum = 0, total;
    if (kind == SUMS && !g.by_min) {
        each<U>(x, q0, q1, 0, 1, [&](int i, float f) { sum += mass(f, r, s.exp_table); });
    } else if (kind == SUMS) {
        each<U>(x, q0, q1, 0, 1, [&](int i, float f) {
            const u64 y = mass(f, r, s.exp_table);
            sum += y >= g.least ? y : 0;
        });
    } else if (kind == NARROW) {
        int n = 0;                        // of this wave
        u64* own = s.data + wid * SEG;
        const float from = value_at(limit, r);
        auto take = [&](int i, float f) {
            const unsigned long long who = __ballot(f >= from);
            if (!who) return;
            const int to = n + __popcll(who & ((1ull << lane) - 1));
            if (f >= from && to < SEG) own[to] = entry(i, f);
            n += __popcll(who);
        };
        if (g.by_p && !g.by_k) {
            each<U>(x, e0, e1, wid, CW, [&](int i, float f) {
                take(i, f);
                sum += mass(f, r, s.exp_table);
            });
        } else {
            each<4>(x, e0, e1, wid, CW, take);
        }
        hand_over(w, own, n, lane);
    } else {
        for (int i = tid; i < BINS; i += CT) s.data[i] = 0;
        __syncthreads();
        each<U>(x, e0, e1, wid, CW, [&](int i, float f) {
            const int bin = bin_of(f, r);
            if (bin < BINS) atomicAdd(&s.data[bin], mass(f, r, s.exp_table));
        });
        __syncthreads();
        u64* h = p.hist + ((long long)b * p.chunks + c) * BINS;
        for (int i = tid; i < BINS; i += CT) h[i] = s.data[i];
    }
    if (kind == SUMS) {
        sum = wave_sum_u64(sum);
        if (lane == 0) w.part[c * CW + wid] = sum;
        return;
    }
    block_scan<CW>(sum, s.wsum, tid, total);
    if (tid == 0) w.part[c] = total;
}

// Fourth, for the WIDE rows: the tokens of the bin where the nucleus ends, and the masses ahead of it by chunk.
template <typename T>
__global__ __launch_bounds__(CT, 4) void sample_edge_kernel(SampleArgs a, Plan p) {
    __shared__ ChunkLds s;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, c = blockIdx.y, b = blockIdx.x;
    RowWs& w = p.rows[b];
    if (w.kind != WIDE) return;
    const float mx = row_max(w, p.chunks, lane);
    const T* x = (const T*)a.x + (long long)b * a.ld;
    const int e0 = min(c * p.chunk, a.vocab), e1 = min(e0 + p.chunk, a.vocab);
    const Setting g = setting(a, b, mx);
    const Row r = g.r;
    load_exps(s.exp_table, tid, CT);
    __syncthreads();
    const int bin = w.bin;
    int n = 0;
    u64 sum = 0, total;
    u64* own = s.data + wid * SEG;
    const float from = value_at(bin + 1.f, r), upto = value_below((float)bin, r);
    auto take = [&](int i, float f) {
        if (!__any(f >= from && f <= upto)) return;
        const bool have = bin_of(f, r) == bin;
        const unsigned long long who = __ballot(have);
        const int to = n + __popcll(who & ((1ull << lane) - 1));
        if (have && to < SEG) own[to] = entry(i, f);
        n += __popcll(who);
    };
    if (g.by_min) {
        each<2>(x, e0, e1, wid, CW, [&](int i, float f) {
            take(i, f);
            const u64 y = mass(f, r, s.exp_table);
            sum += steps(f, r) < (float)bin && y >= g.least ? y : 0;
        });
    } else {                              // the histogram has them
        each<4>(x, e0, e1, wid, CW, take);
        const u64* h = p.hist + ((long long)b * p.chunks + c) * BINS;
#pragma unroll 8
        for (int i = tid; i < bin; i += CT) sum += h[i];
    }
    hand_over(w, own, n, lane);
    block_scan<CW>(sum, s.wsum, tid, total);
    if (tid == 0) w.part[c] = total;
}

// The token at which the running sum over [0, V) passes the aim, `total` in all: the part by s.part (`parts` of
// `size` elements), while it is long a part of it by the waves, and the last 8 ST elements at once.
template <typename T, typename W>
__device__ void draw(const SampleArgs& a, int parts, int size, const T* x, Lds& s, int tid, int b, const Setting& g,
                     u64 total, W weight) {
    const int lane = tid & 63, wid = tid >> 6;
    u64 t;
    const u64 w0 = tid < parts ? s.part[tid] : 0, to0 = block_scan<SW>(w0, s.wsum, tid, t);
    u64 target = aim(g, total);
    if (tid < parts && to0 - w0 <= target && to0 > target) { s.i0 = tid; s.b0 = to0 - w0; }
    __syncthreads();
    int e0 = s.i0 * size, e1 = min(e0 + size, a.vocab);
    target -= s.b0;
    while (e1 - e0 > 8 * ST) {
        __syncthreads();
        const int each_w = (e1 - e0 + SW - 1) / SW, q0 = min(e0 + wid * each_w, e1), q1 = min(q0 + each_w, e1);
        u64 w = 0;
        each_one(x, q0, q1, 0, 1, [&](int i, float f) { w += weight(i, f); });
        w = wave_sum_u64(w);
        const u64 to = block_scan<SW>(lane == 63 ? w : 0, s.wsum, tid, t);
        if (lane == 63 && to - w <= target && to > target) {
            s.i0 = q0;
            s.i1 = q1;
            s.b0 = to - w;
        }
        __syncthreads();
        e0 = s.i0;
        e1 = s.i1;
        target -= s.b0;
    }
    const int per = (e1 - e0 + ST - 1) / ST;       // up to 8 neighbours of each thread
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int i = e0 + tid * per + j;
        f[j] = j < per && i < e1 ? to_f(x[i]) : -INFINITY;
    }
    u64 mine = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < per) mine += f[j] > -INFINITY ? weight(e0 + tid * per + j, f[j]) : 0;
    u64 at = block_scan<SW>(mine, s.wsum, tid, t) - mine;
    if (at <= target && at + mine > target) {
        for (int i = e0 + tid * per;; ++i) {
            const u64 w = weight(i, to_f(x[i]));
            if (at + w > target) {
                a.token[b] = i;
                if (a.prob) a.prob[b] = (float)((double)w / (double)total);
                return;
            }
            at += w;
        }
    }
}

// The same from the candidates in s.cand: masses by index in BINS steps, then the tokens of the step.
template <typename A, typename W>
__device__ void draw_from(const SampleArgs& a, A all, Lds& s, int tid, int b, const Setting& g, W weight) {
    for (int i = tid; i < BINS; i += ST) s.hist_w[i] = 0;
    if (tid == 0) s.n_list = 0;
    __syncthreads();
    const int per = (a.vocab + BINS - 1) / BINS;
    u64 mine = 0, total, wb, t;
    all([&](int i, float f) {
        const u64 w = weight(i, f);
        if (w) atomicAdd(&s.hist_w[i / per], w);
        mine += w;
    });
    block_scan<SW>(mine, s.wsum, tid, total);
    const u64 target = aim(g, total);
    const int bin = find_bin_w(s, tid, target + 1, wb);
    all([&](int i, float f) {
        if (i / per == bin && weight(i, f)) {
            const u64 e = entry(i, f);
            s.list[atomicAdd(&s.n_list, 1u)] = e << 32 | e >> 32;      // at most `per` <= 512 of them, to go by index
        }
    });
    __syncthreads();
    const int m = (int)s.n_list;
    __syncthreads();
    sort_entries(s, m, tid);
    const u64 e = tid < m ? s.list[tid] : 0;
    const u64 w = tid < m ? mass(key_value(~(uint32_t)e), g.r, s.exp_table) : 0;
    const u64 to = block_scan<SW>(w, s.wsum, tid, t) + wb;
    if (tid < m && to - w <= target && to > target) {
        a.token[b] = (int)(e >> 32);
        if (a.prob) a.prob[b] = (float)((double)w / (double)total);
    }
}

// The cuts of top-k and of top-p, the earlier of both: each the end of a bin of the histograms in s.hist_n and s.hist_w,
// found among the bin's tokens, which all(f) goes over. total: all mass; with top-k that of its tokens afterwards. edge: the
// bin of top-p is known (WIDE), with its tokens in s.list.
template <typename A>
__device__ __forceinline__ Cut cuts(A all, int V, const Setting& g, Lds& s, int tid, const RowWs* edge, u64& total) {
    Cut cut{0, V};                        // everything
#pragma unroll 1
    for (int by_mass = edge ? 1 : 0; by_mass < 2; ++by_mass) {
        if (!(by_mass ? g.by_p : g.by_k)) continue;
        u64 nb = 0, wb, want, to;
        int bin;
        if (edge) {
            bin = edge->bin;
            want = edge->want;
            wb = edge->before;
        } else {
            want = by_mass ? nucleus(g, total) : (u64)g.top_k;
            bin = by_mass ? find_bin_w(s, tid, want, wb) : find_bin_n(s, tid, want, nb, wb);
            if (!by_mass) total = wb;     // of all, unless the cut lies before
            if (bin >= BINS) continue;    // fewer than k, or min-p ends before
            if (tid == 0) s.n_list = 0;
            __syncthreads();
            all([&](int i, float f) { push(s.list, s.n_list, LIST, bin_of(f, g.r) == bin, i, f); });
            __syncthreads();
        }
        const Cut c = find_cut(all, V, g.r, s, tid, bin, by_mass, nb, wb, want, to);
        if (!by_mass) total = to;
        if (c.key > cut.key || (c.key == cut.key && c.index < cut.index)) cut = c;
    }
    return cut;
}

// The end of a row whose n <= CAND candidates are in s.cand; total: all mass where top-p stands alone.
__device__ __forceinline__ void draw_narrow(const SampleArgs& a, Lds& s, int tid, int b, const Setting& g, int n, u64 total) {
    if (n <= FEW) {
        // few: each token's place in the order and the mass ahead of it say whether it is kept
        u64 rank, before, t;
        const u64 e = rank_few(s, n, tid, g.r, [&](int i) { return s.cand[i]; }, rank, before);
        const bool own = tid < 4 * n && !(tid & 3);
        const u64 y = own ? s.few[tid >> 2].y : 0;
        bool keep = own && (!g.by_k || rank < (u64)g.top_k);
        if (g.by_k) block_scan<SW>(keep ? y : 0, s.wsum, tid, total);
        keep = keep && (!g.by_p || before < nucleus(g, total)) && y >= g.least;
        block_scan<SW>(keep ? y : 0, s.wsum, tid, total);
        if (own) s.few[tid >> 2] = make_ulonglong2(e & 0xffffffff, keep ? y : 0);     // index and what is kept
        __syncthreads();
        const u64 target = aim(g, total);
        t = 0;
        if (tid < 4 * n) over_few(s, n, tid, [&](const ulonglong2& o) { t += o.x < (e & 0xffffffff) ? o.y : 0; });
        t = four_sum(t);
        if (keep && t <= target && t + y > target) {
            a.token[b] = entry_index(e);
            if (a.prob) a.prob[b] = (float)((double)y / (double)total);
        }
        return;
    }
    for (int i = tid; i < BINS; i += ST) { s.hist_w[i] = 0; s.hist_n[i] = 0; }
    __syncthreads();
    auto all = [&](auto f) {
        for (int i = tid; i < n; i += ST) f(entry_index(s.cand[i]), entry_value(s.cand[i]));
    };
    all([&](int i, float f) {
        const int bin = bin_of(f, g.r);
        if (bin >= BINS) return;
        if (g.by_k) atomicAdd(&s.hist_n[bin], 1u);
        if (g.by_p) atomicAdd(&s.hist_w[bin], mass(f, g.r, s.exp_table));
    });
    __syncthreads();
    const Cut cut = cuts(all, a.vocab, g, s, tid, nullptr, total);
    draw_from(a, all, s, tid, b, g, [&](int i, float f) -> u64 {
        if (!kept(f, i, cut)) return 0;
        const u64 y = mass(f, g.r, s.exp_table);
        return y >= g.least ? y : 0;
    });
}

// Third, one workgroup per row: the rows that are done, and the WIDE rows' bin.
template <typename T>
__global__ __launch_bounds__(ST) void sample_pick_kernel(SampleArgs a, Plan p) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    Lds& s = *(Lds*)smem;
    const int tid = threadIdx.x, lane = tid & 63, b = blockIdx.x;
    const T* x = (const T*)a.x + (long long)b * a.ld;
    RowWs& w = p.rows[b];
    const float mx = row_max(w, p.chunks, lane);
    if (mx == -INFINITY || is_greedy(a, b)) {
        int first = lane < p.chunks && w.top[lane] == mx ? w.top_at[lane] : 0x7fffffff;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
        if (tid == 0) {
            a.token[b] = mx == -INFINITY ? -1 : first;
            if (a.prob) a.prob[b] = mx == -INFINITY ? 0.f : 1.f;
        }
        return;
    }
    const Setting g = setting(a, b, mx);
    const int kind = w.kind;
    load_exps(s.exp_table, tid, ST);
    const int parts = kind == SUMS || kind == INFS ? p.chunks * CW : p.chunks, size = p.chunk / CW;
    u64 total;                            // SUMS: what is kept; top-p alone: all mass
    {
        const u64 mine = tid < parts ? w.part[tid] : 0;
        if (tid < parts) s.part[tid] = mine;
        block_scan<SW>(mine, s.wsum, tid, total);
    }
    if (kind == INFS) {
        if (g.by_k) total = min(total, (u64)g.top_k);
        if (g.by_p) total = max((u64)1, min(total, (u64)ceil((double)g.top_p * (double)total)));
        draw(a, parts, size, x, s, tid, b, g, total, [&](int i, float f) -> u64 { return f == INFINITY; });
        return;
    }
    if (kind == SUMS) {
        draw(a, parts, size, x, s, tid, b, g, total, [&](int i, float f) -> u64 {
            const u64 y = mass(f, g.r, s.exp_table);
            return y >= g.least ? y : 0;
        });
        return;
    }
    if (kind == WIDE) {
        const u64* h = p.hist + (long long)b * p.chunks * BINS;
        for (int i = tid; i < BINS; i += ST) {
            u64 y = 0;
#pragma unroll 8
            for (int c = 0; c < p.chunks; ++c) y += h[(long long)c * BINS + i];
            s.hist_w[i] = y;
        }
        __syncthreads();
        u64 before;
        find_bin_w(s, tid, ~0ull, total);           // all that weighs is in a bin
        const u64 want = nucleus(g, total);
        const int bin = find_bin_w(s, tid, want, before);
        if (tid == 0) { w.total = total; w.want = want; w.before = before; w.bin = bin; }
        return;
    }
    const u64 n64 = w.n_list;
    if (n64 > CAND) {
        if (tid == 0) w.kind = FULL;
        return;
    }
    const int n = (int)n64;
    for (int i = tid; i < n; i += ST) s.cand[i] = w.list[i];
    __syncthreads();
    draw_narrow(a, s, tid, b, g, n, total);
}

// Last, one workgroup per row: the WIDE rows' end, and the rows whose candidates did not fit (FULL) from the logits alone.
template <typename T>
__global__ __launch_bounds__(ST) void sample_rest_kernel(SampleArgs a, Plan p) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    Lds& s = *(Lds*)smem;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, b = blockIdx.x, V = a.vocab;
    RowWs& w = p.rows[b];
    const int kind = w.kind;
    if (kind != WIDE && kind != FULL) return;
    const float mx = row_max(w, p.chunks, lane);
    const T* x = (const T*)a.x + (long long)b * a.ld;
    const Setting g = setting(a, b, mx);
    const Row r = g.r;
    load_exps(s.exp_table, tid, ST);
    if (tid < PARTS) s.part[tid] = kind == WIDE && tid < p.chunks ? w.part[tid] : 0;
    auto row = [&](auto f) { each_one(x, 0, V, wid, SW, f); };
    u64 total = 0;
    int n = 0;
    if (kind == WIDE) {
        n = (int)min(w.n_list, (u64)LIST + 1);
        for (int i = tid; i < min(n, LIST); i += ST) s.list[i] = w.list[i];
        if (tid == 0) s.n_list = n;
    } else {
        for (int i = tid; i < BINS; i += ST) { s.hist_w[i] = 0; s.hist_n[i] = 0; }
        __syncthreads();
        row([&](int i, float f) {
            const int bin = bin_of(f, r);
            if (bin >= BINS) return;
            atomicAdd(&s.hist_n[bin], 1u);
            atomicAdd(&s.hist_w[bin], mass(f, r, s.exp_table));
        });
        __syncthreads();
        find_bin_w(s, tid, ~0ull, total);           // all that weighs is in a bin
    }
    __syncthreads();
    const Cut cut = cuts(row, V, g, s, tid, kind == WIDE ? &w : nullptr, total);
    auto weight = [&](int i, float f) -> u64 {
        if (!kept(f, i, cut)) return 0;
        const u64 y = mass(f, r, s.exp_table);
        return y >= g.least ? y : 0;
    };
    // WIDE: the masses ahead of the bin are there, its own tokens up to the cut come to them
    if (kind == WIDE && n <= LIST) {
        for (int i = tid; i < n; i += ST) {
            const u64 y = weight(entry_index(s.list[i]), entry_value(s.list[i]));
            if (y) atomicAdd(&s.part[entry_index(s.list[i]) / p.chunk], y);
        }
    } else {
        const int bin = kind == WIDE ? w.bin : -1;
        row([&](int i, float f) {
            const u64 y = bin < 0 || bin_of(f, r) == bin ? weight(i, f) : 0;
            if (y) atomicAdd(&s.part[i / p.chunk], y);
        });
    }
    __syncthreads();
    block_scan<SW>(tid < p.chunks ? s.part[tid] : 0, s.wsum, tid, total);
    draw(a, p.chunks, p.chunk, x, s, tid, b, g, total, weight);
}

// Rows of at most SHORT logits, one workgroup each and nothing else: a thread keeps neighbouring logits. Against the chain
// of kernels, us: one row of 8404 11 and 16 (no filter), 12 and 22 (top-k 50, top-p), 22 and 29 (top-p on a wide nucleus); of
// 12288 14 and 16, 14 and 22, 25 and 36; of 16000, in 16 logits a thread, 21 and 16, 18 and 22, 34 and 38; 512 rows of 8404
// 24 and 23, 25 and 31, 59 and 83.
constexpr int OWN = 12, SHORT = OWN * ST;
template <typename T>
__global__ __launch_bounds__(ST) void sample_short_kernel(SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    Lds& s = *(Lds*)smem;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, b = blockIdx.x, V = a.vocab;
    const T* x = (const T*)a.x + (long long)b * a.ld;
    const int per = (V + ST - 1) / ST, i0 = tid * per;
    float v[OWN], mine = -INFINITY;
#pragma unroll
    for (int j = 0; j < OWN; ++j) v[j] = j < per && i0 + j < V ? to_f(x[i0 + j]) : -INFINITY;
    load_exps(s.exp_table, tid, ST);
    for (int i = tid; i < BINS; i += ST) { s.hist_w[i] = 0; s.hist_n[i] = 0; }
    int at = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < OWN; ++j)
        if (v[j] > mine) { mine = v[j]; at = i0 + j; }
    const float m = wave_max(mine);
    float* wmax = (float*)s.wsum;
    if (lane == 0) wmax[wid] = m;
    __syncthreads();
    float mx = m;
#pragma unroll
    for (int w = 0; w < SW; ++w) mx = fmaxf(mx, wmax[w]);
    if (mx == -INFINITY || is_greedy(a, b)) {
        // threads are in the vocabulary's order: the first that has the maximum
        if (tid == 0) s.i0 = 0x7fffffff;
        __syncthreads();
        if (mine == mx) atomicMin(&s.i0, at);
        __syncthreads();
        if (tid == 0) {
            a.token[b] = mx == -INFINITY ? -1 : s.i0;
            if (a.prob) a.prob[b] = mx == -INFINITY ? 0.f : 1.f;
        }
        return;
    }
    const Setting g = setting(a, b, mx);
    // Short loops that pick a logit from the registers by the loop's count: one row of 8404 with top-k 50 and top-p takes 12
    // us. Unrolled, each loop is code that a lone workgroup fetches once: 5 us more.
    auto all = [&](auto f) {
#pragma unroll 1
        for (int j = 0; j < per; ++j)
            if (v[j] > -INFINITY) f(i0 + j, v[j]);
    };
    u64 total, t;
    const bool inf = mx == INFINITY;      // its tokens share the mass
    if (!inf && (g.by_k || g.by_p)) {
        int kth = BINS;
        if (g.by_k) {
            if (bin_of(mine, g.r) < BINS) atomicAdd(&s.hist_n[bin_of(mine, g.r)], 1u);
            __syncthreads();
            u64 before;
            kth = find_bin<SW>(s.hist_n, s.wsum, &s.i0, &s.b0, tid, g.top_k, before);
        }
        const float from = value_at(candidate_limit(g, V, kth), g.r);
        if (tid == 0) s.n_list = 0;
        __syncthreads();
        u64 z = 0;
        all([&](int i, float f) { push(s.cand, s.n_list, CAND, f >= from, i, f); });
        if (g.by_p && !g.by_k) all([&](int i, float f) { z += mass(f, g.r, s.exp_table); });
        block_scan<SW>(z, s.wsum, tid, total);
        const int n = (int)s.n_list;
        __syncthreads();
        if (n <= CAND) {
            draw_narrow(a, s, tid, b, g, n, total);
            return;
        }
        for (int i = tid; i < BINS; i += ST) s.hist_n[i] = 0;
        __syncthreads();
    }
    Cut cut{0, V};
    if (inf) {
        u64 n = 0;
        all([&](int i, float f) { n += f == INFINITY; });
        block_scan<SW>(n, s.wsum, tid, total);
        if (g.by_k) total = min(total, (u64)g.top_k);
        if (g.by_p) total = max((u64)1, min(total, (u64)ceil((double)g.top_p * (double)total)));
    } else if (g.by_k || g.by_p) {
        u64 z = 0;
        all([&](int i, float f) {
            const int bin = bin_of(f, g.r);
            if (bin >= BINS) return;
            if (g.by_k) atomicAdd(&s.hist_n[bin], 1u);
            if (g.by_p) {
                const u64 y = mass(f, g.r, s.exp_table);
                atomicAdd(&s.hist_w[bin], y);
                z += y;
            }
        });
        block_scan<SW>(z, s.wsum, tid, total);
        cut = cuts(all, V, g, s, tid, nullptr, total);
    }
    auto weight = [&](int i, float f) -> u64 {
        if (inf) return f == INFINITY;
        if (!kept(f, i, cut)) return 0;
        const u64 y = mass(f, g.r, s.exp_table);
        return y >= g.least ? y : 0;
    };
    u64 w = 0;
    all([&](int i, float f) { w += weight(i, f); });
    const u64 to = block_scan<SW>(w, s.wsum, tid, t);
    if (!inf) total = t;
    const u64 target = aim(g, total);
    u64 run = to - w;
    if (run <= target && to > target) {
        bool done = false;
        all([&](int i, float f) {
            const u64 y = weight(i, f);
            if (!done && run + y > target) {
                done = true;
                a.token[b] = i;
                if (a.prob) a.prob[b] = (float)((double)y / (double)total);
            }
            run += y;
        });
    }
}

// Chunks of at least 2048 elements, as many as give the chip four workgroups per CU, or one more than that (64 rows of
// 128000, top-p: 65 us; 68 with two per CU, 77 with eight; 256 of 131071 140, 148 and 142).
Plan plan(int batch, int vocab) {
    Plan p{};
    const int want = std::max(1, std::min(CHUNKS, (1024 + batch - 1) / batch));
    const int most = std::max(1, vocab / 2048);
    p.chunks = std::min(want, most);
    p.chunk = (vocab + p.chunks * CW - 1) / (p.chunks * CW) * CW;
    p.groups = CT;
    while (p.groups * p.chunks > GROUPS && p.groups > GROUPS / CHUNKS) p.groups /= 2;
    return p;
}

template <typename T> hipError_t run(const SampleArgs& a, hipStream_t st) {
    static_assert(sizeof(Lds) <= 150 * 1024 && BINS % ST == 0 && BINS % CT == 0 && CHUNKS <= 64, "sizes");
    if (a.vocab <= SHORT) {
        const hipError_t e = pfm_allow_lds<sample_short_kernel<T>>(sizeof(Lds));
        if (e != hipSuccess) return e;
        sample_short_kernel<T><<<a.batch, ST, sizeof(Lds), st>>>(a);
        PFM_LAUNCH_CHECK();
        return hipSuccess;
    }
    Plan p = plan(a.batch, a.vocab);
    p.rows = (RowWs*)a.ws;
    p.hist = (u64*)(p.rows + a.batch);
    hipError_t e = pfm_allow_lds<sample_pick_kernel<T>>(sizeof(Lds));
    if (e == hipSuccess) e = pfm_allow_lds<sample_rest_kernel<T>>(sizeof(Lds));
    if (e != hipSuccess) return e;
    const dim3 grid(a.batch, p.chunks);
    sample_max_kernel<T><<<grid, CT, 0, st>>>(a, p);
    sample_scan_kernel<T><<<grid, CT, 0, st>>>(a, p);
    sample_pick_kernel<T><<<a.batch, ST, sizeof(Lds), st>>>(a, p);
    if (a.top_k || a.top_p) {
        if (a.top_p) sample_edge_kernel<T><<<grid, CT, 0, st>>>(a, p);
        sample_rest_kernel<T><<<a.batch, ST, sizeof(Lds), st>>>(a, p);
    }
    PFM_LAUNCH_CHECK();
    return hipSuccess;
}

}  // namespace

long long pfm_sample_ws_bytes(int batch, int vocab) {
    if (vocab <= SHORT) return 0;
    return (long long)batch * (long long)sizeof(RowWs) + (long long)batch * plan(batch, vocab).chunks * BINS * 8;
}
hipError_t pfm_sample(int dtype, const SampleArgs& a, hipStream_t st) {
    if (dtype == DT_F32) return run<float>(a, st);
    if (dtype == DT_BF16) return run<bf16>(a, st);
    return run<f16>(a, st);
}
