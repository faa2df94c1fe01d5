// Sampling (ps_hip_sample): top-k, temperature, top-p, min-p and a draw from a given number, a row of logits each.
//   Every stage takes a beginning of the candidates in descending order, so that none of them needs the order itself, only places in it: the place where a count (top-k), a sum of weights
//   (top-p, the draw) or a weight (min-p) is reached.  Candidates are counted and their weights added in bins of equal width of z = (largest - logit) / temperature, 1/32 wide up to z = 40 and
//   one for the rest (weight 0); a place's bin follows from sums over bins, and only that bin's candidates are collected and sorted.  A bin with more of them than LDS takes
//   (equal logits, a high temperature) is walked digit by digit of the logit instead.
//   Weights e^-z are computed in 64 bits -- e^-(bin / 32) from a table times a polynomial of what is left, below 1/32 -- and added as whole multiples of 2^-scale of the largest one: any
//   order of work gives the same sums, and they are within 2^-44 or so of the true ones, where 32-bit sums would move one draw in some thousands to a neighbour.
//   sample_top_kernel    the largest logit of a part of a row; clears the bins
//   sample_bins_kernel   counts and weights of a part, in LDS, added to the row's bins
//   sample_pick_kernel   the stages; with few parts of a row (many rows) it makes the bins itself
#include "ps_serve.h"

#include <algorithm>
#include <cmath>

namespace {
typedef unsigned long long u64;
constexpr int NB = 1280, LIST = 4096, PICK = 1024; // bins below z = 40; candidates of a sorted list; threads of a pick
constexpr double WIDTH = 1.0 / 32;

struct smp_args {
    const void *logits;
    long long n, rows, stride;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *ids;
    float *prob;
    int parts, scale;
    float *top;    // [row][part]
    unsigned *cnt; // [row][NB + 1]
    u64 *sum;      // [row][NB + 1]
};
struct F16 { typedef _Float16 T; };
struct BF16 { typedef __bf16 T; };
struct F32 { typedef float T; };
template <class E> __device__ __forceinline__ float logit(const typename E::T *row, long long i) { return (float)row[i]; }
__device__ __forceinline__ bool candidate(float l) { return l > -INFINITY; } // (NaN is none)
// f(logit, index) for the numbers lo .. hi of a row, 16 bytes at a time where they are aligned
template <class E, int THREADS, class F>
__device__ __forceinline__ void each(const typename E::T *row, long long lo, long long hi, F f) {
    constexpr int PER = 16 / sizeof(typename E::T);
    const long long mis = ((uintptr_t)(row + lo) & 15) / sizeof(typename E::T), head = min(hi, lo + (mis ? PER - mis : 0)), body = (hi - head) / PER;
    if ((long long)threadIdx.x < head - lo) f(logit<E>(row, lo + threadIdx.x), lo + threadIdx.x);
    const pv_u4 *p = (const pv_u4 *)(row + head);
    auto unpack = [&](const pv_u4 &v, long long i) {
        typename E::T x[PER];
        __builtin_memcpy(x, &v, 16);
#pragma unroll
        for (int e = 0; e < PER; e++) f((float)x[e], head + i * PER + e);
    };
    long long i = threadIdx.x;
    for (; i + 3 * THREADS < body; i += 4 * THREADS) { // four loads in flight
        const pv_u4 a = p[i], b = p[i + THREADS], c = p[i + 2 * THREADS], d = p[i + 3 * THREADS];
        unpack(a, i);
        unpack(b, i + THREADS);
        unpack(c, i + 2 * THREADS);
        unpack(d, i + 3 * THREADS);
    }
    for (; i < body; i += THREADS) unpack(p[i], i);
    const long long tail = head + body * PER;
    if ((long long)threadIdx.x < hi - tail) f(logit<E>(row, tail + threadIdx.x), tail + threadIdx.x);
}
// logits as whole numbers of the same order, and back
__device__ __forceinline__ unsigned order_of(float l) {
    const unsigned u = __float_as_uint(l == 0.f ? 0.f : l); // (the two zeros are equal)
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order(unsigned o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }

struct row_of { // what a row's weights go by
    double top, inv; // largest logit, 1 / temperature
    int k;           // candidates at most (0: all)
    int scale;       // weights are multiples of 2^-scale
};
__device__ __forceinline__ row_of row_settings(const smp_args &a, long long r, float top) {
    row_of w;
    const float t = a.temperature ? a.temperature[r] : 1.f;
    w.top = top;
    w.k = a.top_k ? max(a.top_k[r], 0) : 0;
    w.inv = 1.0;
    if (t > 0.f) w.inv = 1.0 / (double)t;
    else w.k = 1; // the first candidate
    w.scale = a.scale;
    return w;
}
__device__ __forceinline__ double z_of(const row_of &w, float l) { return (double)l == w.top ? 0.0 : (w.top - (double)l) * w.inv; }
__device__ __forceinline__ int bin_of(double z) { return z < NB * WIDTH ? (int)(z * (1 / WIDTH)) : NB; } // (NaN: the rest)
__device__ __forceinline__ double weight_of(double z, int bin, const double *table) { // bin < NB
    const double f = bin * WIDTH - z; // -1/32 .. 0
    double e = 1.0 / 40320;
    e = fma(e, f, 1.0 / 5040);
    e = fma(e, f, 1.0 / 720);
    e = fma(e, f, 1.0 / 120);
    e = fma(e, f, 1.0 / 24);
    e = fma(e, f, 1.0 / 6);
    e = fma(e, f, 0.5);
    e = fma(e, f, 1.0);
    e = fma(e, f, 1.0);
    return table[bin] * e;
}
__device__ __forceinline__ u64 whole(double w, int scale) { return (u64)__double2ull_rn(ldexp(w, scale)); }
__device__ __forceinline__ void make_table(double *table, int threads) {
    for (int b = threadIdx.x; b < NB; b += threads) table[b] = exp(-b * WIDTH);
}
template <int THREADS> __device__ __forceinline__ float block_max(float v, float *sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
    for (int i = 1; i < THREADS / 64; i++) v = fmaxf(v, sh[i]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ void part_of(const smp_args &a, int part, long long &lo, long long &hi) {
    const long long per = ((a.n + a.parts - 1) / a.parts + 63) / 64 * 64;
    lo = min(a.n, part * per);
    hi = min(a.n, lo + per);
}

template <class E>
__global__ __launch_bounds__(256) void sample_top_kernel(const smp_args a) {
    __shared__ float sh[4];
    const long long r = blockIdx.y;
    const typename E::T *row = (const typename E::T *)a.logits + r * a.stride;
    for (int b = blockIdx.x * 256 + threadIdx.x; b <= NB; b += 256 * a.parts) { a.cnt[r * (NB + 1) + b] = 0; a.sum[r * (NB + 1) + b] = 0; }
    long long lo, hi;
    part_of(a, blockIdx.x, lo, hi);
    float m = -INFINITY;
    each<E, 256>(row, lo, hi, [&](float l, long long) { m = fmaxf(m, l); });
    m = block_max<256>(m, sh);
    if (threadIdx.x == 0) a.top[r * a.parts + blockIdx.x] = m;
}
__device__ __forceinline__ void add_to_bins(const row_of &w, float l, unsigned *cnt, u64 *sum, const double *table) {
    if (!candidate(l)) return;
    const double z = z_of(w, l);
    const int b = bin_of(z);
    atomicAdd(&cnt[b], 1u);
    if (b < NB) atomicAdd(&sum[b], whole(weight_of(z, b, table), w.scale));
}
__device__ __forceinline__ float row_top(const smp_args &a, long long r) {
    float m = -INFINITY;
    for (int i = 0; i < a.parts; i++) m = fmaxf(m, a.top[r * a.parts + i]);
    return m;
}
template <class E>
__global__ __launch_bounds__(256) void sample_bins_kernel(const smp_args a) {
    __shared__ unsigned cnt[NB + 1];
    __shared__ u64 sum[NB + 1];
    __shared__ double table[NB];
    const long long r = blockIdx.y;
    const typename E::T *row = (const typename E::T *)a.logits + r * a.stride;
    for (int b = threadIdx.x; b <= NB; b += 256) { cnt[b] = 0; sum[b] = 0; }
    make_table(table, 256);
    const row_of w = row_settings(a, r, row_top(a, r));
    __syncthreads();
    long long lo, hi;
    part_of(a, blockIdx.x, lo, hi);
    each<E, 256>(row, lo, hi, [&](float l, long long) { add_to_bins(w, l, cnt, sum, table); });
    __syncthreads();
    for (int b = threadIdx.x; b <= NB; b += 256)
        if (cnt[b]) { atomicAdd(&a.cnt[r * (NB + 1) + b], cnt[b]); if (sum[b]) atomicAdd(&a.sum[r * (NB + 1) + b], sum[b]); }
}

// What a pick holds.  cx / wx: candidates and weights before a bin.  The list: candidates of the bins la .. lb - 1 in order, lw the weights up to and with each.
struct pick_lds {
    unsigned cx[NB + 2];
    u64 wx[NB + 2];
    double table[NB];
    u64 list[LIST], lw[LIST];
    u64 sh[32];
    float shf[32];
    unsigned dcnt[256];
    u64 dsum[256];
    int n_list, la, lb;
    u64 out[4];
};
__device__ __forceinline__ u64 scan64(u64 v, u64 *sh, u64 *total) { // sum over the threads before this one
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) sh[wave] = x;
    __syncthreads();
    u64 before = 0, all = 0;
    for (int i = 0; i < PICK / 64; i++) { if (i < wave) before += sh[i]; all += sh[i]; }
    __syncthreads();
    *total = all;
    return before + x - v;
}
template <class E>
struct picker {
    const smp_args &a;
    const typename E::T *row;
    row_of w;
    pick_lds &s;

    __device__ __forceinline__ u64 weight(unsigned order) const {
        const double z = z_of(w, from_order(order));
        const int b = bin_of(z);
        return b < NB ? whole(weight_of(z, b, s.table), w.scale) : 0;
    }
    // the candidates of bin b in a list, or false where they are too many for one; from the first bin on where they all fit
    __device__ bool collect(int b) {
        if (s.la <= b && b < s.lb) return true;
        const int la = s.cx[b + 1] <= LIST ? 0 : b, lb = b + 1, n = (int)(s.cx[lb] - s.cx[la]);
        if (n > LIST) return false;
        __syncthreads();
        if (threadIdx.x == 0) { s.n_list = 0; s.la = la; s.lb = lb; }
        __syncthreads();
        // a bin's logits lie between two of its neighbours' -- the exact bin decides
        each<E, PICK>(row, 0, a.n, [&](float l, long long i) {
            if (!candidate(l)) return;
            const int x = bin_of(z_of(w, l));
            if (x >= la && x < lb) s.list[atomicAdd(&s.n_list, 1)] = (u64)~order_of(l) << 32 | (unsigned)i;
        });
        __syncthreads();
        int P = 1;
        while (P < n) P <<= 1;
        for (int i = n + threadIdx.x; i < P; i += PICK) s.list[i] = ~0ull;
        __syncthreads();
        for (int k = 2; k <= P; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int i = threadIdx.x; i < P / 2; i += PICK) {
                    const int x = (i & ~(j - 1)) * 2 + (i & (j - 1)), y = x + j;
                    const u64 p = s.list[x], q = s.list[y];
                    if ((p > q) == ((x & k) == 0)) { s.list[x] = q; s.list[y] = p; }
                }
                __syncthreads();
            }
        // weights up to and with each: a thread has four in a row
        u64 v[LIST / PICK], own = 0, all;
#pragma unroll
        for (int e = 0; e < LIST / PICK; e++) {
            const int i = threadIdx.x * (LIST / PICK) + e;
            v[e] = i < n ? weight(~(unsigned)(s.list[i] >> 32)) : 0;
            own += v[e];
        }
        u64 before = scan64(own, s.sh, &all);
#pragma unroll
        for (int e = 0; e < LIST / PICK; e++) {
            const int i = threadIdx.x * (LIST / PICK) + e;
            before += v[e];
            if (i < n) s.lw[i] = before;
        }
        __syncthreads();
        return true;
    }
    // A bin that is too large for a list: the candidate at which a count (by_weight: a sum of weights) within the bin is reached, digit by digit.  -> its order, the candidates and weights before
    // those that are equal to it, and how many equal ones up to it
    __device__ void descend(int b, bool by_weight, u64 goal, unsigned &order, u64 &c_before, u64 &w_before, u64 &nth) {
        unsigned found = 0, mask = 0;
        c_before = w_before = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = threadIdx.x; i < 256; i += PICK) { s.dcnt[i] = 0; s.dsum[i] = 0; }
            __syncthreads();
            each<E, PICK>(row, 0, a.n, [&](float l, long long) {
                if (!candidate(l)) return;
                const double z = z_of(w, l);
                const unsigned o = ~order_of(l); // ascending: from the largest on
                if (bin_of(z) != b || (o & mask) != found) return;
                atomicAdd(&s.dcnt[o >> shift & 255], 1u);
                if (b < NB) atomicAdd(&s.dsum[o >> shift & 255], whole(weight_of(z, b, s.table), w.scale));
            });
            __syncthreads();
            if (threadIdx.x == 0) {
                u64 c = c_before, x = w_before;
                int d = 0;
                for (; d < 255; d++) {
                    if ((by_weight ? x + s.dsum[d] : c + s.dcnt[d]) >= goal) break;
                    c += s.dcnt[d];
                    x += s.dsum[d];
                }
                s.out[0] = d; s.out[1] = c; s.out[2] = x;
            }
            __syncthreads();
            found |= (unsigned)s.out[0] << shift;
            mask |= 255u << shift;
            c_before = s.out[1];
            w_before = s.out[2];
            __syncthreads();
        }
        order = ~found;
        const u64 each_w = weight(order);
        nth = by_weight ? (each_w ? (goal - w_before + each_w - 1) / each_w : 1) : goal - c_before;
        if (nth < 1) nth = 1;
    }
    // weights of the first c candidates of bin b
    __device__ u64 weight_of_first(int b, u64 c) {
        if (c == 0) return 0;
        if (c == s.cx[b + 1] - s.cx[b]) return s.wx[b + 1] - s.wx[b];
        if (collect(b)) return s.lw[s.cx[b] - s.cx[s.la] + c - 1] - (s.wx[b] - s.wx[s.la]);
        unsigned o;
        u64 cb, wb, nth;
        descend(b, false, c, o, cb, wb, nth);
        return wb + nth * weight(o);
    }
    // the first place of bin b whose weights, added up to and with it, reach goal >= 1 -> how many that are
    __device__ u64 place_of(int b, u64 goal) {
        if (collect(b)) {
            const u64 off = s.wx[b] - s.wx[s.la];
            int lo = (int)(s.cx[b] - s.cx[s.la]), hi = (int)(s.cx[b + 1] - s.cx[s.la]) - 1;
            const int first = lo;
            while (lo < hi) {
                const int m = (lo + hi) / 2;
                if (s.lw[m] - off >= goal) hi = m;
                else lo = m + 1;
            }
            return lo - first + 1;
        }
        unsigned o;
        u64 cb, wb, nth;
        descend(b, true, goal, o, cb, wb, nth);
        return cb + nth;
    }
    // candidates of bin b with a weight of at least `least`
    __device__ u64 at_least(int b, double least) {
        u64 mine = 0, all;
        each<E, PICK>(row, 0, a.n, [&](float l, long long) {
            if (!candidate(l)) return;
            const double z = z_of(w, l);
            if (bin_of(z) == b && weight_of(z, b, s.table) >= least) mine++;
        });
        scan64(mine, s.sh, &all);
        return all;
    }
    // the c-th candidate of bin b: its index, and its weight
    __device__ int candidate_at(int b, u64 c, u64 &wt) {
        if (collect(b)) {
            const u64 x = s.list[s.cx[b] - s.cx[s.la] + c - 1];
            wt = weight(~(unsigned)(x >> 32));
            return (int)(unsigned)x;
        }
        unsigned o;
        u64 cb, wb, nth;
        descend(b, false, c, o, cb, wb, nth);
        wt = weight(o);
        // the nth of the equal ones by index: a thread looks through a stretch of the row
        const long long per = (a.n + PICK - 1) / PICK, lo = min(a.n, threadIdx.x * per), hi = min(a.n, lo + per);
        u64 mine = 0, all;
        auto equal = [&](long long i) { const float l = logit<E>(row, i); return candidate(l) && order_of(l) == o; };
        for (long long i = lo; i < hi; i++) mine += equal(i);
        const u64 before = scan64(mine, s.sh, &all);
        if (before < nth && nth <= before + mine) {
            u64 k = before;
            for (long long i = lo; i < hi; i++)
                if (equal(i) && ++k == nth) { s.out[0] = (u64)i; break; }
        }
        __syncthreads();
        const int id = (int)s.out[0];
        __syncthreads();
        return id;
    }
    // the first bin behind whose end a count or a sum has reached goal (goal <= the whole)
    template <class X> __device__ __forceinline__ int bin_reaching(const X *before, u64 goal) const {
        int lo = 0, hi = NB;
        while (lo < hi) {
            const int m = (lo + hi) / 2;
            if (before[m + 1] >= goal) hi = m;
            else lo = m + 1;
        }
        return lo;
    }
    __device__ void pick(long long r) {
        if (s.cx[NB + 1] == 0) { // no candidate
            if (threadIdx.x == 0) { a.ids[r] = -1; if (a.prob) a.prob[r] = 0.f; }
            return;
        }
        int bl = NB; // what stays: the bins before bl and the first cl of bin bl (the last bin's weights are 0)
        u64 cl = 0;
        if (w.k > 0 && (unsigned)w.k < s.cx[NB]) {
            bl = bin_reaching(s.cx, (u64)w.k);
            cl = (u64)w.k - s.cx[bl];
        }
        u64 total = s.wx[bl] + weight_of_first(bl, cl);
        const float p = a.top_p ? a.top_p[r] : 1.f, m = a.min_p ? a.min_p[r] : 0.f;
        int bp = bl;
        u64 cp = cl;
        if (p < 1.f) {
            const double goal = ceil((double)fmaxf(p, 0.f) * (double)total);
            const u64 g = max((u64)1, min(total, (u64)goal));
            bp = min(bl, bin_reaching(s.wx, g));
            cp = place_of(bp, g - s.wx[bp]);
        }
        if (m > 0.f) {
            const double least = fmin((double)m, 1.0);
            int lo = 0, hi = NB - 1; // the last bin whose largest weight is `least` or more
            while (lo < hi) {
                const int x = (lo + hi + 1) / 2;
                if (s.table[x] >= least) lo = x;
                else hi = x - 1;
            }
            if (lo < bp || (lo == bp && cp > 0)) {
                const u64 c = at_least(lo, least);
                if (lo < bp || c < cp) { bp = lo; cp = c; }
            }
        }
        if (bp != bl || cp != cl) total = s.wx[bp] + weight_of_first(bp, cp);
        const float uf = a.u[r];
        const double at = uf > 0.f ? floor((double)uf * (double)total) : 0.0;
        const u64 g = at >= (double)total ? total : min(total, (u64)at + 1); // the first sum that is above u * total
        int b = min(bp, bin_reaching(s.wx, g));
        u64 wt;
        const u64 c = place_of(b, g - s.wx[b]);
        const int id = candidate_at(b, c, wt);
        if (threadIdx.x == 0) {
            a.ids[r] = id;
            if (a.prob) a.prob[r] = (float)((double)wt / (double)total);
        }
    }
};

template <class E, bool OWN>
__global__ __launch_bounds__(PICK) void sample_pick_kernel(const smp_args a) {
    extern __shared__ __attribute__((aligned(16))) char raw[];
    pick_lds &s = *(pick_lds *)raw;
    const long long r = blockIdx.x;
    const typename E::T *row = (const typename E::T *)a.logits + r * a.stride;
    make_table(s.table, PICK);
    float top;
    unsigned *cnt = (unsigned *)s.list; // (before there is a list)
    u64 *sum = s.lw;
    if (threadIdx.x == 0) { s.la = s.lb = 0; }
    if constexpr (OWN) {
        for (int b = threadIdx.x; b <= NB; b += PICK) { cnt[b] = 0; sum[b] = 0; }
        float m = -INFINITY;
        each<E, PICK>(row, 0, a.n, [&](float l, long long) { m = fmaxf(m, l); });
        top = block_max<PICK>(m, s.shf);
    } else top = row_top(a, r);
    picker<E> pk{a, row, row_settings(a, r, top), s};
    if constexpr (OWN) {
        __syncthreads();
        each<E, PICK>(row, 0, a.n, [&](float l, long long) { add_to_bins(pk.w, l, cnt, sum, s.table); });
    } else {
        for (int b = threadIdx.x; b <= NB; b += PICK) { cnt[b] = a.cnt[r * (NB + 1) + b]; sum[b] = a.sum[r * (NB + 1) + b]; }
    }
    __syncthreads();
    // sums before each bin: a thread has two bins
    u64 all;
    const int b0 = 2 * threadIdx.x, b1 = b0 + 1;
    const u64 c0 = b0 <= NB ? cnt[b0] : 0, c1 = b1 <= NB ? cnt[b1] : 0, w0 = b0 <= NB ? sum[b0] : 0, w1 = b1 <= NB ? sum[b1] : 0;
    const u64 cb = scan64(c0 + c1, s.sh, &all), wb = scan64(w0 + w1, s.sh, &all);
    if (b0 <= NB + 1) { s.cx[b0] = (unsigned)cb; s.wx[b0] = wb; }
    if (b1 <= NB + 1) { s.cx[b1] = (unsigned)(cb + c0); s.wx[b1] = wb + w0; }
    __syncthreads();
    pk.pick(r);
}

template <class E>
void launch(const smp_args &a, hipStream_t st) {
    const size_t lds = sizeof(pick_lds);
    static unsigned long long seen[2] = {0, 0};
    if (a.parts == 1) {
        if (ps_first_on_device(&seen[0])) (void)hipFuncSetAttribute((const void *)sample_pick_kernel<E, true>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        hipLaunchKernelGGL((sample_pick_kernel<E, true>), dim3((unsigned)a.rows), dim3(PICK), lds, st, a);
        return;
    }
    if (ps_first_on_device(&seen[1])) (void)hipFuncSetAttribute((const void *)sample_pick_kernel<E, false>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL((sample_top_kernel<E>), dim3((unsigned)a.parts, (unsigned)a.rows), dim3(256), 0, st, a);
    hipLaunchKernelGGL((sample_bins_kernel<E>), dim3((unsigned)a.parts, (unsigned)a.rows), dim3(256), 0, st, a);
    hipLaunchKernelGGL((sample_pick_kernel<E, false>), dim3((unsigned)a.rows), dim3(PICK), lds, st, a);
}
} // namespace

size_t psv_sample_space(int n_cu, int dtype, const void *logits, int64_t n, int64_t rows, int64_t stride, const ps_sample_params *p, int32_t *ids, float *prob, void *base, bool launch_, hipStream_t st) {
    smp_args a{};
    // a row alone where there is a row for half the CUs; else parts of at least 2048 logits, as many as fill the chip twice
    a.parts = rows * 2 > n_cu ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({(2 * n_cu + rows - 1) / std::max<int64_t>(rows, 1), (n + 2047) / 2048, 128}));
    ps_carve ws{(char *)base};
    if (a.parts > 1) {
        a.top = ws.take<float>((size_t)(rows * a.parts));
        a.cnt = ws.take<unsigned>((size_t)rows * (NB + 1));
        a.sum = ws.take<u64>((size_t)rows * (NB + 1));
    }
    if (!launch_) return ws.at;
    a.logits = logits; a.n = n; a.rows = rows; a.stride = stride;
    a.temperature = p->temperature; a.top_k = p->top_k; a.top_p = p->top_p; a.min_p = p->min_p; a.u = p->u;
    a.ids = ids; a.prob = prob;
    int bits = 0;
    while (((int64_t)1 << bits) < n) bits++;
    a.scale = 62 - bits; // a row's weights add up to at most 2^62
    if (dtype == PS_F32) launch<F32>(a, st);
    else if (dtype == PS_F16) launch<F16>(a, st);
    else launch<BF16>(a, st);
    return ws.at;
}
