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
// NaN logits are never drawn. If the largest logit is +inf, the tokens that have it share the mass; a row without any
// logit above -inf has no token: -1 with probability 0.
#include "pfm_serve.h"

namespace {

typedef unsigned long long u64;
constexpr int SW = 16, ST = SW * 64;    // waves and threads of a row's workgroup
constexpr int BINS = 2048;              // equal steps of (max - x) / T over [0, SPAN)
constexpr float SPAN = 31.f;            // 2^-44 is e^-30.5
constexpr int LIST = 2048;              // tokens of one bin that are sorted at once

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
    double scale;        // log2(e) / T
    float bin_scale;     // 2 BINS / (SPAN T)
};

// p 2^43 as a whole number: 2^t with t = (x - max) log2(e) / T, t = k / 64 + f, |f| <= 1/128: a table's 2^(k mod 64 / 64)
// times the series of e^(f ln 2) to the fourth power (the rest is under 4e-14)
__device__ __forceinline__ u64 mass(float x, const Row& r, const double* exp_table) {
    if (x == r.max) return 1ull << 43;
    const double t = ((double)x - (double)r.max) * r.scale;
    if (!(t > -44.5)) return 0;
    const double kd = rint(t * 64.0);
    const int k = (int)kd;
    const double f = (t - kd * 0.015625) * 0.69314718055994530942;
    const double e = exp_table[k & 63];
    double p = fma(f, 1.0 / 24, 1.0 / 6);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p * f, e, e);
    return (u64)__double_as_longlong(ldexp(p, (k >> 6) + 43) + 4503599627370496.0) & ((1ull << 52) - 1);
}
// monotone in x (halves: the difference does not overflow); BINS: weighs nothing
__device__ __forceinline__ int bin_of(float x, const Row& r) {
    if (x == r.max) return 0;
    const float d = (0.5f * r.max - 0.5f * x) * r.bin_scale;
    return d < (float)BINS ? (int)d : BINS;      // a NaN's bin: BINS
}

template <typename T> struct Pack { static constexpr int N = 16 / sizeof(T); T x[N]; };

// f(index, value) for the elements [e0, e1) of a row, by the threads tid of nt; wide loads where they lie inside
template <typename T, typename F>
__device__ __forceinline__ void each(const T* x, int e0, int e1, int tid, int nt, F f) {
    constexpr int N = Pack<T>::N;
    const int skew = (int)(((uintptr_t)x / sizeof(T)) % N);   // elements of x's first 16 bytes that lie before it
    for (long long v = (e0 + skew) / N + tid; v * N - skew < e1; v += nt) {
        const int i = (int)(v * N - skew);
        if (i >= e0 && i + N <= e1) {
            const Pack<T> p = *(const Pack<T>*)__builtin_assume_aligned(x + i, 16);
#pragma unroll
            for (int j = 0; j < N; ++j) f(i + j, to_f(p.x[j]));
        } else {
            for (int j = 0; j < N; ++j)
                if (i + j >= e0 && i + j < e1) f(i + j, to_f(x[i + j]));
        }
    }
}

struct Lds {
    double exp_table[64];
    u64 hist_w[BINS];
    unsigned hist_n[BINS + 1];
    u64 list[LIST];          // ~key << 32 | index: ascending is the order of tokens
    u64 wsum[SW];
    float wmax[SW];
    unsigned wn[SW];
    unsigned n_list;
    u64 b0, b1;              // broadcasts
    int i0, i1;
};

// The last kept token of the order: every token with a larger key is kept, of the equal ones those up to `index`.
struct Cut {
    uint32_t key;
    int index;
};
__device__ __forceinline__ bool kept(float x, int i, const Cut& c) {
    const uint32_t k = order_key(x);
    return k > c.key || (k == c.key && i <= c.index);
}

// block-wide inclusive scans of one value per thread
__device__ __forceinline__ u64 block_scan(u64 v, Lds& s, int tid, u64& total) {
    const int lane = tid & 63, wid = tid >> 6;
    u64 x = wave_scan_u64(v, lane);
    __syncthreads();
    if (lane == 63) s.wsum[wid] = x;
    __syncthreads();
    u64 before = 0, t = 0;
#pragma unroll
    for (int w = 0; w < SW; ++w) {
        const u64 y = s.wsum[w];
        if (w < wid) before += y;
        t += y;
    }
    total = t;
    return x + before;
}

// The first bin in which the running count (or mass) reaches `want` >= 1; what lies before it and in it. BINS: none does.
__device__ int find_bin(Lds& s, int tid, bool by_mass, u64 want, u64& n_before, u64& w_before) {
    constexpr int PER = BINS / ST;
    u64 n = 0, w = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) { n += s.hist_n[tid * PER + j]; w += s.hist_w[tid * PER + j]; }
    u64 nt, wt;
    u64 n0 = block_scan(n, s, tid, nt) - n, w0 = block_scan(w, s, tid, wt) - w;
    __syncthreads();
    if (tid == 0) { s.i0 = BINS; s.b0 = nt; s.b1 = wt; }
    __syncthreads();
    const u64 at = by_mass ? w0 : n0, mine = by_mass ? w : n;
    if (at < want && at + mine >= want) {
        int j = 0;
        for (; j < PER - 1; ++j) {
            const u64 add = by_mass ? s.hist_w[tid * PER + j] : s.hist_n[tid * PER + j];
            if ((by_mass ? w0 : n0) + add >= want) break;
            n0 += s.hist_n[tid * PER + j];
            w0 += s.hist_w[tid * PER + j];
        }
        s.i0 = tid * PER + j;
        s.b0 = n0;
        s.b1 = w0;
    }
    __syncthreads();
    const int bin = s.i0;
    n_before = s.b0;
    w_before = s.b1;
    __syncthreads();
    return bin;
}

__device__ void sort_list(u64* a, int n, int tid) {   // ascending, n a power of two <= LIST
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int i = tid; i < n / 2; i += ST) {
                const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                const u64 x = a[lo], y = a[hi];
                if ((x > y) == ((lo & k) == 0)) { a[lo] = y; a[hi] = x; }
            }
        }
    __syncthreads();
}

// The token of bin `bin` at which the running count (or mass), `before` ahead of the bin, reaches `want`; and the mass
// of all tokens up to it.
template <typename T>
__device__ Cut find_cut(const T* x, int V, const Row& r, Lds& s, int tid, int bin, bool by_mass, u64 n_before,
                        u64 w_before, u64 want, u64& mass_to) {
    const int n = (int)s.hist_n[bin];
    if (n <= LIST) {
        if (tid == 0) s.n_list = 0;
        __syncthreads();
        each(x, 0, V, tid, ST, [&](int i, float f) {
            if (bin_of(f, r) == bin) s.list[atomicAdd(&s.n_list, 1u)] = ((u64)~order_key(f) << 32) | (uint32_t)i;
        });
        int p2 = 2;
        while (p2 < n) p2 <<= 1;
        __syncthreads();
        for (int i = n + tid; i < p2; i += ST) s.list[i] = ~0ull;
        sort_list(s.list, p2, tid);
        u64 base_n = n_before, base_w = w_before, total;
        if (tid == 0) { s.i0 = -1; s.b1 = 0; }
        for (int i0 = 0; i0 < n; i0 += ST) {
            const int i = i0 + tid;
            const u64 w = i < n ? mass(key_value(~(uint32_t)(s.list[i] >> 32)), r, s.exp_table) : 0;
            const u64 to = block_scan(w, s, tid, total) + base_w;
            const u64 at = by_mass ? to - w : base_n + tid, after = by_mass ? to : base_n + tid + 1;
            if (i < n && at < want && after >= want) { s.i0 = i; s.b1 = to; }
            base_w += total;
            base_n += ST;
        }
        __syncthreads();
        const u64 at = s.list[s.i0];
        mass_to = s.b1;
        __syncthreads();
        return Cut{~(uint32_t)(at >> 32), (int)(uint32_t)at};
    }
    // too many to sort: the bin's keys digit by digit, then the equal ones by index
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        u64* dw = s.list;                  // [256] masses, [256] counts
        u64* dn = s.list + 256;
        for (int i = tid; i < 512; i += ST) s.list[i] = 0;
        __syncthreads();
        const uint32_t above = shift == 24 ? 0u : ~0u << (shift + 8);
        each(x, 0, V, tid, ST, [&](int i, float f) {
            const uint32_t k = order_key(f);
            if (bin_of(f, r) == bin && (k & above) == prefix) {
                atomicAdd(&dw[(k >> shift) & 255], mass(f, r, s.exp_table));
                atomicAdd(&dn[(k >> shift) & 255], 1ull);
            }
        });
        __syncthreads();
        u64 w = 0, c = 0, t;
        const int digit = 255 - tid;       // the larger first
        if (tid < 256) { w = dw[digit]; c = dn[digit]; }
        const u64 w1 = block_scan(w, s, tid, t) + w_before, c1 = block_scan(c, s, tid, t) + n_before;
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
    const float v = key_value(prefix);
    const u64 each_w = mass(v, r, s.exp_table);
    // of the equal ones the first `take` are kept
    const u64 take = by_mass ? (want - w_before + each_w - 1) / each_w : want - n_before;
    mass_to = w_before + take * each_w;
    int e0 = 0, e1 = V;
    u64 left = take;
    while (e1 - e0 > 1) {                  // into the SW-th part that holds the take-th one
        const int part = (e1 - e0 + SW - 1) / SW, wid = tid >> 6, lane = tid & 63;
        const int p0 = min(e0 + wid * part, e1), p1 = min(p0 + part, e1);
        u64 c = 0, t;
        each(x, p0, p1, lane, 64, [&](int i, float f) { c += order_key(f) == prefix; });
        const u64 all = wave_sum_u64(c), to = block_scan(lane == 63 ? all : 0, s, tid, t);
        __syncthreads();
        if (lane == 63 && to - all < left && to >= left) {
            s.i0 = p0;
            s.i1 = p1;
            s.b0 = to - all;
        }
        __syncthreads();
        e0 = s.i0;
        e1 = s.i1;
        left -= s.b0;
        __syncthreads();
    }
    return Cut{prefix, e0};
}

// One workgroup per row: the row's maximum; a histogram of counts and masses; the cuts; then the token, by parts that
// get smaller by the number of waves.
template <typename T>
__global__ __launch_bounds__(ST) void sample_rows_kernel(SampleArgs a) {
    __shared__ Lds s;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, b = blockIdx.x, V = a.vocab;
    const T* x = (const T*)a.x + (long long)b * a.ld;

    float mx = -INFINITY;
    each(x, 0, V, tid, ST, [&](int i, float f) { mx = fmaxf(mx, f); });
    mx = wave_max(mx);
    if (lane == 0) s.wmax[wid] = mx;
    if (tid < 64) s.exp_table[tid] = exp2((double)tid / 64);
    for (int i = tid; i < BINS; i += ST) { s.hist_w[i] = 0; s.hist_n[i] = 0; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SW; ++w) mx = fmaxf(mx, s.wmax[w]);
    if (mx == -INFINITY) {
        if (tid == 0) { a.token[b] = -1; if (a.prob) a.prob[b] = 0.f; }
        return;
    }
    const float T0 = a.temperature ? a.temperature[b] : 1.f;
    const bool greedy = !(T0 > 0.f);
    const float u = a.u[b];
    int top_k = a.top_k ? a.top_k[b] : 0;
    if (top_k <= 0 || top_k > V) top_k = V;
    float top_p = a.top_p ? a.top_p[b] : 1.f, min_p = a.min_p ? a.min_p[b] : 0.f;
    if (greedy) top_k = 1;
    Row r;
    r.max = mx;
    const double T1 = greedy ? 1.0 : fmax((double)T0, 1e-30);   // the bins' steps stay finite
    r.scale = 1.4426950408889634074 / T1;
    r.bin_scale = (float)(2.0 * BINS / (SPAN * T1));
    const bool by_k = top_k < V, by_p = top_p < 1.f && !greedy;   // NaN: off

    Cut cut{0, V};                        // everything
    if (by_k || by_p) {
        each(x, 0, V, tid, ST, [&](int i, float f) {
            const int bin = bin_of(f, r);
            if (bin < BINS) {
                atomicAdd(&s.hist_n[bin], 1u);
                atomicAdd(&s.hist_w[bin], mass(f, r, s.exp_table));
            }
        });
        __syncthreads();
        u64 nb, wb, total;
        bool cut_k = false;
        if (by_k) {
            const int bin = find_bin(s, tid, false, top_k, nb, wb);
            total = wb;                   // all of it, unless the cut lies before
            if (bin < BINS) {
                cut = find_cut(x, V, r, s, tid, bin, false, nb, wb, top_k, total);
                cut_k = true;
            }
        } else {
            find_bin(s, tid, true, ~0ull, nb, total);
        }
        if (by_p) {
            // the first token is kept in any case
            const double want = ceil(fmax((double)top_p, 0.0) * (double)total);
            const u64 w = want < 1.0 ? 1 : want >= (double)total ? total : (u64)want;
            const int bin = find_bin(s, tid, true, w, nb, wb);
            u64 to;
            const Cut c = find_cut(x, V, r, s, tid, bin, true, nb, wb, w, to);
            if (!cut_k || c.key > cut.key || (c.key == cut.key && c.index < cut.index)) cut = c;
        }
    }
    // min-p in masses: p_i >= min_p  <=>  mass >= min_p 2^43, to the rounding of a mass
    const double floor_w = min_p > 0.f && !greedy ? fmin((double)min_p, 1.0) * 8796093022208.0 : 0.0;
    const u64 least = floor_w > 1.0 ? (u64)ceil(floor_w) : 1;
    auto weight = [&](int i, float f) -> u64 {
        if (!kept(f, i, cut)) return 0;
        const u64 w = mass(f, r, s.exp_table);
        return w >= least ? w : 0;
    };
    int e0 = 0, e1 = V;
    u64 target = 0, total = 0;
    bool known = false;
    while (e1 - e0 > 1) {
        const int part = (e1 - e0 + SW - 1) / SW;
        const int p0 = min(e0 + wid * part, e1), p1 = min(p0 + part, e1);
        u64 w = 0, t;
        each(x, p0, p1, lane, 64, [&](int i, float f) { w += weight(i, f); });
        w = wave_sum_u64(w);
        const u64 to = block_scan(lane == 63 ? w : 0, s, tid, t);
        if (!known) {
            total = t;
            const double at = floor((u > 0.f ? (double)u : 0.0) * (double)t);
            target = at >= (double)t ? t - 1 : (u64)at;
            known = true;
        }
        __syncthreads();
        if (lane == 63 && to - w <= target && to > target) {
            s.i0 = p0;
            s.i1 = p1;
            s.b0 = to - w;
        }
        __syncthreads();
        e0 = s.i0;
        e1 = s.i1;
        target -= s.b0;
        __syncthreads();
    }
    if (tid == 0) {
        a.token[b] = e0;
        if (a.prob) a.prob[b] = known ? (float)((double)weight(e0, to_f(x[e0])) / (double)total) : 1.f;
    }
}

template <typename T> hipError_t run(const SampleArgs& a, hipStream_t st) {
    sample_rows_kernel<T><<<a.batch, ST, 0, st>>>(a);
    PFM_LAUNCH_CHECK();
    return hipSuccess;
}

}  // namespace

long long pfm_sample_ws_bytes(int batch, int vocab) { return 0; }
hipError_t pfm_sample(int dtype, const SampleArgs& a, hipStream_t st) {
    if (dtype == DT_F32) return run<float>(a, st);
    if (dtype == DT_BF16) return run<bf16>(a, st);
    return run<f16>(a, st);
}
