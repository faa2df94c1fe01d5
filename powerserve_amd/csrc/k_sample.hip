// Sampling (ps_hip_sample): top-k, temperature, top-p, min-p and a draw from a given number, a row of logits each.
//   Every stage takes a beginning of the candidates in descending order, so that none of them needs the order itself, only places in it: the place where a count (top-k), a sum of weights
//   (top-p, the draw) or a weight (min-p) is reached.
//   First pass: the largest logit of each of 1024 groups of a row.  The k-th largest of those is a bound that at least k candidates reach (any k up to 1024), and few more than that do.
//   Second pass: the candidates at or above the bound -- the k-th for a count, else the 1014th, some 5000 of a large vocabulary -- go into a list, the head; where no count makes the others
//   irrelevant, all are counted and their weights added in bins of equal width of z = (largest - logit) / temperature, 1/32 wide up to z = 40 and one for the rest (weight 0).
//   A place's bin follows from sums over bins, and only that bin's candidates are collected -- from the head in LDS, or, where a place lies behind it, in one more
//   pass over the row -- and walked digit by digit of (logit, index), with counts and weights of a digit's values, until one is left.  Where they are more than LDS takes (equal logits, a
//   high temperature) every digit is a pass over the row.
//   Weights e^-z -- of z in 64 bits, e^-(bin / 32) from a table times a polynomial of what is left, below 1/32 -- are added as whole multiples of 2^-scale of the largest one: any order of
//   work gives the same sums, and what a weight is off by, 2^-28 of it to either side alike, moves one draw in millions to a neighbour, where 32-bit sums would move one in some thousands.
// Measured: one row of 128256 in fp32, 3 + 7 + 10 us, the latency of the passes and of a stage's steps; 33 rows of 151936 in bf16, 4 + 21 + 17, the second pass's 64-bit arithmetic and its additions to the LDS; 256
// such rows of fp32 in one launch, 116 us: 15 the first pass (131 MB), 30 the second where the head alone counts and 55 where all do, 14 for each place that lies behind the head, 1 for one in it (vector units 49 % busy; waves wait 64 % of
// their time, for the row, for LDS and for each other).
//   sample_top_kernel   the first pass over a part of a row
//   sample_head_kernel  the second pass over a part
//   sample_pick_kernel  the stages; with few parts of a row (many rows) it makes both passes itself
#include "ps_serve.h"

#include <algorithm>
#include <cmath>

namespace {
typedef unsigned long long u64;
constexpr int NB = 1280, LIST = 2048, HEAD = 8192, PICK = 1024; // bins below z = 40; candidates of a bin's list, of the head; threads of a pick
constexpr int PART_HEAD = 2048; // of a part
constexpr int QUANTILE = 1014; // of the 1024 groups' largest logits: the head's bound where no count gives one
constexpr double WIDTH = 1.0 / 32;

struct smp_args {
    const void *logits;
    long long rows, stride;
    int n; // up to 2^24
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *ids;
    float *prob;
    int parts, scale;
    float *top;     // [row][1024] the groups' largest logits
    float *bound;   // [row][2] the bound, the largest logit
    unsigned *cnt;  // [row][part][NB + 1]
    u64 *sum;       // [row][part][NB + 1]
    u64 *head;      // [row][part][PART_HEAD]
    unsigned *held; // [row][part] candidates in it
};
struct F16 { typedef _Float16 T; };
struct BF16 { typedef __bf16 T; };
struct F32 { typedef float T; };
// One of a few registers.  (A chain of choices among the l[i] would be made a load of an array in memory: 33 rows of 151936 bf16 numbers, the second pass 31 us, 21 so.)
template <int N> __device__ __forceinline__ float at(const float (&l)[N], int e) {
    unsigned v = 0;
#pragma unroll
    for (int i = 0; i < N; i++) v |= e == i ? __float_as_uint(l[i]) : 0u;
    return __uint_as_float(v);
}
__device__ __forceinline__ bool candidate(float l) { return l > -INFINITY; } // (NaN is none)
// f(numbers, index of the first) for the pieces of 16 bytes of the numbers lo .. hi of a row: a piece is worked on with the next three and the one that takes its place on their way.  What lies before
// the first whole piece and behind the last goes in a piece each, filled up with minus infinity.
template <class E, int THREADS, class F>
__device__ __forceinline__ void each(const typename E::T *row, int lo, int hi, F f) {
    typedef typename E::T T;
    constexpr int PER = 16 / sizeof(T);
    const int mis = (int)(((uintptr_t)(row + lo) & 15) / sizeof(T)), tid = threadIdx.x;
    const int head = min(hi, lo + (mis ? PER - mis : 0)), body = (hi - head) / PER, tail = head + body * PER;
    auto give = [&](const T (&x)[PER], int first) {
        float l[PER];
#pragma unroll
        for (int e = 0; e < PER; e++) l[e] = (float)x[e];
        f(l, first);
    };
    const pv_u4 *p = (const pv_u4 *)(row + head);
    auto piece = [&](const pv_u4 &v, int u) {
        T x[PER];
        __builtin_memcpy(x, &v, 16);
        give(x, head + u * PER);
    };
    if (tid < body) {
        pv_u4 v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = p[min(tid + j * THREADS, body - 1)];
        for (int i = tid; i < body; i += 4 * THREADS) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const pv_u4 x = v[j];
                v[j] = p[min(i + (j + 4) * THREADS, body - 1)];
                if (j == 0 || i + j * THREADS < body) piece(x, i + j * THREADS);
            }
        }
    }
    const int n = tid == 0 ? head - lo : tid == 64 ? hi - tail : 0, first = tid == 0 ? lo : tail;
    if (n > 0) {
        T x[PER];
#pragma unroll
        for (int e = 0; e < PER; e++) x[e] = e < n ? row[first + e] : (T)-INFINITY;
        give(x, first);
    }
}
// sums over a wave's lanes up to and with each
template <int CTRL, int ROWS> __device__ __forceinline__ u64 moved(u64 v) {
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 15, false), hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 15, false);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_sums(u64 v) {
    v += moved<0x111, 15>(v); // row_shr: 1, 2, 4, 8
    v += moved<0x112, 15>(v);
    v += moved<0x114, 15>(v);
    v += moved<0x118, 15>(v);
    v += moved<0x142, 10>(v); // row_bcast: 15 into rows 1 and 3, 31 into rows 2 and 3
    v += moved<0x143, 12>(v);
    return v;
}
// logits as whole numbers of the same order, and back
__device__ __forceinline__ unsigned order_of(float l) {
    const unsigned u = __float_as_uint(l == 0.f ? 0.f : l); // (the two zeros are equal)
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order(unsigned o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }

struct row_of { // what a row's weights go by
    double top, inv; // largest logit, 32 / temperature
    int k;           // candidates at most (0: all)
};
__device__ __forceinline__ row_of row_settings(const smp_args &a, long long r, float top) {
    row_of w;
    const float t = a.temperature ? a.temperature[r] : 1.f;
    w.top = top;
    w.k = a.top_k ? max(a.top_k[r], 0) : 0;
    w.inv = 1 / WIDTH;
    if (t > 0.f) w.inv = 1 / WIDTH / (double)t;
    else w.k = 1; // the first candidate
    return w;
}
// z in widths of a bin
__device__ __forceinline__ double z_of(const row_of &w, float l) { return (double)l == w.top ? 0.0 : (w.top - (double)l) * w.inv; }
__device__ __forceinline__ int bin_of(double z) { return z < (double)NB ? (int)z : NB; } // (NaN: the rest)
// The weight as a multiple of 2^-scale (the table holds them so), bin < NB: e^-(bin / 32) in 64 bits times e^-f, f < 1/32, whose difference from 1 is a polynomial in 32 bits: 2^-28 of the weight
// off, to either side alike.  Half the instructions of a polynomial in 64 bits, in the loop over a whole vocabulary; wherever a weight is asked for it is this one.
__device__ __forceinline__ u64 weight_of(double z, int bin, const double *table) {
    const float f = (float)(z - (double)bin) * -(float)WIDTH; // -1/32 .. 0
    float e = 1.f / 120;
    e = fmaf(e, f, 1.f / 24);
    e = fmaf(e, f, 1.f / 6);
    e = fmaf(e, f, 0.5f);
    e = fmaf(e, f, 1.f) * f;
    const double w = fma(table[bin], (double)e, table[bin]);
    return __double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull; // 2^52 + w: w rounded to a whole number, below 2^52
}
// e^-(b / 32) 2^scale, as a product of two of 72 numbers (sh: 72; barriers inside)
__device__ __forceinline__ void make_table(double *table, double *sh, int threads, int scale) {
    const int t = threadIdx.x;
    if (t < 72) sh[t] = t < 40 ? ldexp(exp(-(double)t), scale) : exp(-(t - 40) * WIDTH);
    __syncthreads();
    for (int b = t; b < NB; b += threads) table[b] = sh[b >> 5] * sh[40 + (b & 31)];
    __syncthreads();
}
__device__ __forceinline__ void part_of(const smp_args &a, int part, int &lo, int &hi) {
    const int per = ((a.n + a.parts - 1) / a.parts + 7) / 8 * 8;
    lo = min(a.n, part * per);
    hi = min(a.n, lo + per);
}

// What a row's passes go by.  tail: the candidates below the bound count too; counts: so does their number
struct passes {
    float bound;
    bool tail, counts;
};
__device__ __forceinline__ u64 entry(float l, int i) { return (u64)~order_of(l) << 32 | (unsigned)i; } // ascending: from the largest on, equal ones by index
__device__ __forceinline__ passes passes_of(int k, float bound) { return passes{bound, k < 1 || k > QUANTILE, k > 0}; }
struct digit_lds { // 256 values of a digit: candidates and weights, and where a count or a sum is reached
    unsigned cnt[256];
    u64 sum[256];
    u64 out[4];
};
// The digit at which a count (by_weight: a sum) reaches goal, which c and x, what lies before, are raised to; one wave.  Lane l has digits 4 l .. 4 l + 3.
__device__ __forceinline__ void find_digit(digit_lds &d, bool by_weight, u64 goal, u64 c, u64 x) {
    const int lane = threadIdx.x & 63;
    u64 cs[4], ss[4], ct = 0, st = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) { cs[e] = d.cnt[4 * lane + e]; ss[e] = d.sum[4 * lane + e]; ct += cs[e]; st += ss[e]; }
    c += wave_sums(ct) - ct;
    x += wave_sums(st) - st;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const u64 before = by_weight ? x : c, with = before + (by_weight ? ss[e] : cs[e]);
        if (before < goal && with >= goal) { d.out[0] = (u64)(4 * lane + e); d.out[1] = c; d.out[2] = x; d.out[3] = cs[e]; }
        c += cs[e];
        x += ss[e];
    }
}
// The bound of a row from its groups' largest logits, a thread each; top: the largest of all.  From the first bit on in which they differ 16 bits, digit by digit; what differs behind them lets a
// few more into the head.
__device__ __forceinline__ void row_bound(const smp_args &a, long long r, float mine, digit_lds &d, float &top, passes &ps) {
    const unsigned o = ~order_of(mine); // ascending: from the largest on
    unsigned lo = o, hi = o;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) { lo = min(lo, (unsigned)__shfl_xor((int)lo, x, 64)); hi = max(hi, (unsigned)__shfl_xor((int)hi, x, 64)); }
    if (threadIdx.x < 256) { d.cnt[threadIdx.x] = 0; d.sum[threadIdx.x] = 0; }
    if (threadIdx.x == 0) { d.out[0] = ~0ull; d.out[1] = 0; }
    const int some = __syncthreads_count(mine > -INFINITY); // groups with a candidate: short parts and masked stretches leave others empty
    if ((threadIdx.x & 63) == 0) { atomicMin(&d.out[0], (u64)lo); atomicMax(&d.out[1], (u64)hi); }
    __syncthreads();
    lo = (unsigned)d.out[0];
    hi = (unsigned)d.out[1];
    top = from_order(~lo);
    const int k = row_settings(a, r, top).k, first = 31 - __clz(lo ^ hi); // (-1: all are equal)
    ps = passes_of(k, 0.f);
    const u64 goal = (u64)(ps.tail ? max(1, min(QUANTILE, some - (1024 - QUANTILE))) : k);
    unsigned mask = first >= 31 ? 0 : ~0u << (first + 1), found = lo & mask;
    u64 before = 0;
    int shift = max(0, first - 7);
#pragma unroll 1
    for (int i = 0; i < 2; i++) {
        __syncthreads();
        if ((o & mask) == found) atomicAdd(&d.cnt[o >> shift & 255], 1u);
        __syncthreads();
        if (threadIdx.x < 64) find_digit(d, false, goal, before, 0);
        __syncthreads();
        mask |= 255u << shift;
        found = (found & ~(255u << shift)) | (unsigned)d.out[0] << shift;
        before = d.out[1];
        if (threadIdx.x < 256) d.cnt[threadIdx.x] = 0;
        if (shift == 0) break;
        shift = max(0, shift - 8);
    }
    ps.bound = from_order(~min(found | ~mask, ~order_of(-INFINITY)));
    __syncthreads();
}
__device__ __forceinline__ void add_to_bins(const row_of &w, float l, unsigned *cnt, u64 *sum, const double *table, bool counts) {
    const double z = z_of(w, l);
    const int b = bin_of(z);
    if (counts && candidate(l)) atomicAdd(&cnt[b], 1u);
    if (b < NB) atomicAdd(&sum[b], weight_of(z, b, table));
}

template <class E>
__global__ __launch_bounds__(256) void sample_top_kernel(const smp_args a) {
    const long long r = blockIdx.y;
    const typename E::T *row = (const typename E::T *)a.logits + r * a.stride;
    int lo, hi;
    part_of(a, blockIdx.x, lo, hi);
    float m = -INFINITY;
    each<E, 256>(row, lo, hi, [&](const auto &l, int) {
#pragma unroll
        for (float x : l) m = fmaxf(m, x);
    });
    // 1024 groups a row: of parts / 4 lanes each
    const int lanes = a.parts / 4;
    for (int o = 1; o < lanes; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if (threadIdx.x % lanes == 0) a.top[r * 1024 + blockIdx.x * (256 / lanes) + threadIdx.x / lanes] = m;
}
// the second pass over lo .. hi: at or above the bound into the head (room for `most`; n counts on); where the others count, all into the bins
template <class E>
__device__ __forceinline__ void second_pass(const typename E::T *row, int lo, int hi, const row_of &w, const passes &ps, u64 *head, int *n, int most, unsigned *cnt, u64 *sum, const double *table) {
    each<E, PICK>(row, lo, hi, [&](const auto &l, int first) {
        constexpr int PER = sizeof(l) / 4;
        float m = l[0];
#pragma unroll
        for (int e = 1; e < PER; e++) m = fmaxf(m, l[e]);
        if (m >= ps.bound && candidate(m)) {
            unsigned high = 0;
#pragma unroll
            for (int e = 0; e < PER; e++) high |= (l[e] >= ps.bound && candidate(l[e]) ? 1u : 0u) << e;
            int k = atomicAdd(n, __popc(high));
            while (high) {
                const int e = __ffs(high) - 1;
                high &= high - 1;
                if (k < most) head[k] = entry(at(l, e), first + e);
                k++;
            }
        }
        if (ps.tail)
#pragma unroll
            for (int e = 0; e < PER; e++) add_to_bins(w, l[e], cnt, sum, table, ps.counts);
    });
}
template <class E>
__global__ __launch_bounds__(PICK) void sample_head_kernel(const smp_args a) {
    __shared__ unsigned cnt[NB + 1];
    __shared__ u64 sum[NB + 1];
    __shared__ double table[NB];
    __shared__ u64 list[PART_HEAD];
    __shared__ int n_list;
    const long long r = blockIdx.y;
    const typename E::T *row = (const typename E::T *)a.logits + r * a.stride;
    float top;
    passes ps;
    row_bound(a, r, a.top[r * 1024 + threadIdx.x], *(digit_lds *)list, top, ps);
    __syncthreads();
    const row_of w = row_settings(a, r, top);
    if (ps.tail) {
        for (int b = threadIdx.x; b <= NB; b += PICK) { cnt[b] = 0; sum[b] = 0; }
        make_table(table, (double *)list, PICK, a.scale);
    }
    if (threadIdx.x == 0) n_list = 0;
    __syncthreads();
    int lo, hi;
    part_of(a, blockIdx.x, lo, hi);
    second_pass<E>(row, lo, hi, w, ps, list, &n_list, PART_HEAD, cnt, sum, table);
    __syncthreads();
    // side by side with the other parts': sums between work-groups of different XCDs would be atomics at the memory (33 rows of 16 parts: 35 us of 47)
    const long long part = r * a.parts + blockIdx.x;
    if (threadIdx.x == 0) {
        a.held[part] = (unsigned)n_list;
        if (blockIdx.x == 0) { a.bound[2 * r] = ps.bound; a.bound[2 * r + 1] = top; }
    }
    if (ps.tail)
        for (int b = threadIdx.x; b <= NB; b += PICK) {
            if (ps.counts) a.cnt[part * (NB + 1) + b] = cnt[b];
            a.sum[part * (NB + 1) + b] = sum[b];
        }
    for (int i = threadIdx.x; i < min(n_list, PART_HEAD); i += PICK) a.head[part * PART_HEAD + i] = list[i];
}

// What a pick holds.  cx / wx: candidates and weights before a bin.  The list: the candidates of a bin (where they fit).
struct pick_lds {
    unsigned cx[NB + 2];
    u64 wx[NB + 2];
    double table[NB];
    u64 head[HEAD];
    union {
        u64 list[LIST];
        struct {
            u64 sum[NB + 1]; // (while the bins are made)
            unsigned cnt[NB + 1];
        } bins;
    };
    digit_lds d;
    int n_head, n[4], place[4]; // a stage each
    u64 both[2], sh[16], few[64];
    int n_few;
};
template <class E>
struct picker {
    const smp_args &a;
    const typename E::T *row;
    row_of w;
    pick_lds &s;
    int in_head; // the bins before this one are in the head whole
    int bin = -1, n_list = 0; // what was collected last

    __device__ __forceinline__ u64 weight(u64 v) const { // of an entry
        const double z = z_of(w, from_order(~(unsigned)(v >> 32)));
        const int b = bin_of(z);
        return b < NB ? weight_of(z, b, s.table) : 0;
    }
    // the logits of bin b lie between these two, a little widened: most others are passed by without arithmetic in 64 bits
    __device__ __forceinline__ void range_of(int b, float &lo, float &hi) const {
        const double zl = b / w.inv, zh = (b + 1) / w.inv, size = fabs(w.top);
        const bool known = size < INFINITY;
        hi = known && zl < 1e30 ? (float)(w.top - zl + 1e-5 * (size + zl)) : INFINITY;
        lo = known && zh < 1e30 && b < NB ? (float)(w.top - zh - 1e-5 * (size + zh)) : -INFINITY;
    }
    // f(entry, weight) for the candidates of bin b in the row
    template <class F> __device__ __forceinline__ void each_of_bin(int b, F f) {
        float lo, hi;
        range_of(b, lo, hi);
        each<E, PICK>(row, 0, a.n, [&](const auto &l, int first) {
            unsigned some = 0;
#pragma unroll
            for (int e = 0; e < (int)(sizeof(l) / 4); e++) some |= (l[e] >= lo && l[e] <= hi ? 1u : 0u) << e;
            while (some) {
                const int e = __ffs(some) - 1;
                some &= some - 1;
                const float v = at(l, e);
                const double z = z_of(w, v);
                if (bin_of(z) == b && candidate(v)) f(entry(v, first + e), b < NB ? weight_of(z, b, s.table) : (u64)0);
            }
        });
    }
    // the candidates of bin b into the list; false where they are too many.  (The stages that ask count in places of their own, so that none waits to clear one.)
    __device__ __forceinline__ bool collect(int b, int stage) {
        if (bin == b) return n_list <= LIST;
        bin = b;
        auto put = [&](u64 v, u64) {
            const int k = atomicAdd(&s.n[stage], 1);
            if (k < LIST) s.list[k] = v;
        };
        if (b < in_head) {
            for (int i = threadIdx.x; i < s.n_head; i += PICK) {
                const u64 v = s.head[i];
                if (bin_of(z_of(w, from_order(~(unsigned)(v >> 32)))) == b) put(v, 0);
            }
        } else each_of_bin(b, put);
        __syncthreads();
        n_list = s.n[stage];
        return n_list <= LIST;
    }
    // f(entry, weight) for the candidates of the bin that was collected last
    template <class F> __device__ __forceinline__ void each_collected(bool listed, F f) {
        if (listed) {
            for (int i = threadIdx.x; i < n_list; i += PICK) f(s.list[i], weight(s.list[i]));
        } else each_of_bin(bin, f);
    }
    // The candidate of bin b at which a count (by_weight: a sum of weights) within the bin reaches goal >= 1, digit by digit of its entry -> its entry, its place within the bin, the weights up to it
    __device__ __forceinline__ void select(bool listed, bool by_weight, u64 goal, u64 &found, u64 &place, u64 &sum) {
        place = sum = 0;
        if (listed && n_list <= 64) return of_few(s.list, n_list, by_weight, goal, found, place, sum);
        // from the first bit on in which logits of the bin can differ
        float lo, hi;
        range_of(bin, lo, hi);
        const unsigned from = ~order_of(hi), to = ~order_of(lo);
        const int bits = 64 - __clz(from ^ to); // (32: index alone)
        u64 mask = bits >= 64 ? 0 : ~0ull << bits;
        found = (u64)from << 32 & mask;
        int shift = bits - 8;
        if (threadIdx.x < 256) { s.d.cnt[threadIdx.x] = 0; s.d.sum[threadIdx.x] = 0; }
        __syncthreads();
#pragma unroll 1
        for (;; shift = max(0, shift - 8)) {
            each_collected(listed, [&](u64 v, u64 x) {
                if ((v & mask) != found) return;
                const int k = (int)(v >> shift & 255);
                atomicAdd(&s.d.cnt[k], 1u);
                atomicAdd(&s.d.sum[k], x);
            });
            __syncthreads();
            if (threadIdx.x < 64) find_digit(s.d, by_weight, goal, place, sum);
            __syncthreads();
            // (the lowest digits may overlap the ones before them: those bits are the same in all that are left)
            mask |= 255ull << shift;
            found = (found & ~(255ull << shift)) | s.d.out[0] << shift;
            place = s.d.out[1];
            sum = s.d.out[2];
            const u64 left = s.d.out[3];
            __syncthreads();
            if (threadIdx.x < 256) { s.d.cnt[threadIdx.x] = 0; s.d.sum[threadIdx.x] = 0; }
            if (left <= 64) break; // (the last digit leaves one)
            __syncthreads();
        }
        each_collected(listed, [&](u64 v, u64) {
            if ((v & mask) == found) s.few[atomicAdd(&s.n_few, 1)] = v;
        });
        __syncthreads();
        const u64 c = place, x = sum;
        of_few(s.few, s.n_few, by_weight, goal - (by_weight ? x : c), found, place, sum);
        place += c;
        sum += x;
    }
    // the same among at most 64 entries: a wave, each lane against all
    __device__ __forceinline__ void of_few(const u64 *few, int n, bool by_weight, u64 goal, u64 &found, u64 &place, u64 &sum) {
        if (threadIdx.x < 64) {
            const u64 v = (int)threadIdx.x < n ? few[threadIdx.x] : ~0ull, x = (int)threadIdx.x < n ? weight(v) : 0; // (no index is that large)
            u64 c = 0, upto = 0;
#pragma unroll 4
            for (int i = 0; i < n; i++) {
                const u64 o = (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32 | (unsigned)__builtin_amdgcn_readlane((int)v, i);
                const u64 y = (u64)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32 | (unsigned)__builtin_amdgcn_readlane((int)x, i);
                if (o <= v) { c++; upto += y; }
            }
            if (v != ~0ull && (by_weight ? upto - x < goal && upto >= goal : c == goal)) { s.d.out[0] = v; s.d.out[1] = c; s.d.out[2] = upto; }
        }
        __syncthreads();
        found = s.d.out[0];
        place = s.d.out[1];
        sum = s.d.out[2];
        if (threadIdx.x == 0) s.n_few = 0;
        __syncthreads();
    }
    // the bin in which sums before each of them (and behind the last) reach goal >= 1
    template <class X> __device__ __forceinline__ int reaching(const X *before, u64 goal, int stage) {
        for (int i = threadIdx.x; i < NB; i += PICK)
            if (before[i] < goal && before[i + 1] >= goal) s.place[stage] = i;
        __syncthreads();
        return s.place[stage];
    }
    __device__ __forceinline__ void pick(long long r, float p, float m, float uf) {
        // what stays: the bins before b and the first c of bin b (the last bin's weights are 0)
        int b = NB;
        u64 c = 0, total = s.wx[NB];
        enum { COUNT, SUM, LEAST, DRAW };
#pragma unroll 1
        for (int stage = COUNT; stage <= DRAW; stage++) {
            int x = 0; // the bin that the stage's place is in, and what it asks for there
            u64 goal = 0;
            u64 least = 0;
            if (stage == LEAST) {
                if (!(m > 0.f)) continue;
                least = (u64)__double2ull_rn(ldexp(fmin((double)m, 1.0), a.scale));
                // the last bin whose largest weight is `least` or more
                for (int i = threadIdx.x; i < NB; i += PICK)
                    if (s.table[i] >= (double)least && (i == NB - 1 || s.table[i + 1] < (double)least)) s.place[stage] = i;
                __syncthreads();
                x = s.place[stage];
                if (x > b || (x == b && c == 0)) continue;
            } else {
                if (stage == COUNT) {
                    if (!(w.k > 0 && (unsigned)w.k < s.cx[NB])) continue;
                    goal = (u64)w.k;
                    x = reaching(s.cx, goal, stage);
                    goal -= s.cx[x];
                } else {
                    if (stage == SUM) {
                        if (!(p < 1.f)) continue;
                        goal = max((u64)1, min(total, (u64)ceil((double)fmaxf(p, 0.f) * (double)total)));
                    } else { // the first sum that is above u * total
                        const double at = uf > 0.f ? floor((double)uf * (double)total) : 0.0;
                        goal = at >= (double)total ? total : min(total, (u64)at + 1);
                    }
                    x = min(b, reaching(s.wx, goal, stage));
                    goal -= s.wx[x];
                }
            }
            const bool listed = collect(x, stage);
            u64 found = 0, n = 0, sum = 0; // the place within the bin, and the weights up to it
            if (stage == LEAST) {
                if (threadIdx.x == 0) s.both[0] = s.both[1] = 0;
                __syncthreads();
                each_collected(listed, [&](u64, u64 wt) {
                    if (wt >= least) { atomicAdd(&s.both[0], (u64)1); atomicAdd(&s.both[1], wt); }
                });
                __syncthreads();
                n = s.both[0];
                sum = s.both[1];
                __syncthreads();
            } else select(listed, stage != COUNT, goal, found, n, sum);
            if (stage == DRAW) {
                if (threadIdx.x == 0) {
                    a.ids[r] = (int)(unsigned)found;
                    if (a.prob) a.prob[r] = (float)((double)weight(found) / (double)total);
                }
            } else if (x < b || c == 0 || n < c) { // (c == 0: bin b was not cut)
                b = x;
                c = n;
                total = s.wx[x] + sum;
            }
        }
    }
};

template <class E, bool OWN>
__global__ __launch_bounds__(PICK) void sample_pick_kernel(const smp_args a) {
    extern __shared__ __attribute__((aligned(16))) char raw[];
    pick_lds &s = *(pick_lds *)raw;
    const long long r = blockIdx.x;
    const typename E::T *row = (const typename E::T *)a.logits + r * a.stride;
    unsigned *cnt = s.bins.cnt;
    u64 *sum = s.bins.sum;
    const float p = a.top_p ? a.top_p[r] : 1.f, m = a.min_p ? a.min_p[r] : 0.f, uf = a.u[r];
    float mine = -INFINITY, top;
    passes ps;
    if constexpr (OWN)
        each<E, PICK>(row, 0, a.n, [&](const auto &l, int) {
#pragma unroll
            for (float x : l) mine = fmaxf(mine, x);
        });
    make_table(s.table, (double *)s.head, PICK, a.scale);
    if constexpr (OWN) row_bound(a, r, mine, s.d, top, ps);
    else {
        top = a.bound[2 * r + 1];
        ps = passes_of(row_settings(a, r, top).k, a.bound[2 * r]);
    }
    if (!candidate(top)) {
        if (threadIdx.x == 0) { a.ids[r] = -1; if (a.prob) a.prob[r] = 0.f; }
        return;
    }
    const row_of w = row_settings(a, r, top);
    for (int b = threadIdx.x; b <= NB; b += PICK) {
        unsigned c = 0;
        u64 x = 0;
        if (!OWN && ps.tail) {
#pragma unroll 8
            for (int q = 0; q < a.parts; q++) x += a.sum[(r * a.parts + q) * (NB + 1) + b];
            if (ps.counts) // (loops of their own: a condition between the loads would wait for each)
#pragma unroll 8
                for (int q = 0; q < a.parts; q++) c += a.cnt[(r * a.parts + q) * (NB + 1) + b];
        }
        cnt[b] = c;
        sum[b] = x;
    }
    if (threadIdx.x < 4) { s.n[threadIdx.x] = 0; s.place[threadIdx.x] = NB; s.n_head = s.n_few = 0; }
    __syncthreads();
    if constexpr (OWN) {
        second_pass<E>(row, 0, a.n, w, ps, s.head, &s.n_head, HEAD, cnt, sum, s.table);
        __syncthreads();
    } else { // the parts' heads one behind the other, a wave a part
        const int lane = threadIdx.x & 63;
        const unsigned n = lane < a.parts ? a.held[r * a.parts + lane] : 0;
        unsigned before = n > PART_HEAD ? HEAD + 1 : n; // (too many anywhere: no head)
        const unsigned own = before;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned y = __shfl_up(before, o, 64);
            if (lane >= o) before += y;
        }
        const unsigned all = __shfl(before, 63, 64);
        before -= own;
        if (all <= HEAD)
            for (int q = threadIdx.x >> 6; q < a.parts; q += PICK / 64) {
                const unsigned at = __shfl(before, q, 64), m = __shfl(own, q, 64);
                for (unsigned i = lane; i < m; i += 64) s.head[at + i] = a.head[(r * a.parts + q) * PART_HEAD + i];
            }
        if (threadIdx.x == 0) s.n_head = (int)all;
        __syncthreads();
    }
    int in_head = ps.tail ? bin_of(z_of(w, ps.bound)) : NB + 1;
    if (s.n_head > HEAD) { // no head, and every candidate in the bins
        in_head = 0;
        if (!ps.tail) {
            const passes all{NAN, true, true}; // (nothing is at or above it)
            second_pass<E>(row, 0, a.n, w, all, s.head, &s.n[0], 0, cnt, sum, s.table);
        }
    } else if (!ps.tail) {
        for (int i = threadIdx.x; i < s.n_head; i += PICK) add_to_bins(w, from_order(~(unsigned)(s.head[i] >> 32)), cnt, sum, s.table, true);
    }
    __syncthreads();
    // sums before each bin: a thread of four waves has six bins
    constexpr int EACH = 6;
    static_assert(256 * EACH >= NB + 2, "");
    const int t = threadIdx.x, lane = t & 63;
    unsigned c[EACH], cs = 0, cp = 0;
    u64 x[EACH], xs = 0, xp = 0;
    if (t < 256) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int b = t * EACH + e;
            c[e] = b <= NB ? cnt[b] : 0;
            x[e] = b <= NB ? sum[b] : 0;
            cs += c[e];
            xs += x[e];
        }
        cp = (unsigned)wave_sums(cs);
        xp = wave_sums(xs);
        if (lane == 63) { s.sh[t >> 6] = xp; s.sh[4 + (t >> 6)] = cp; }
    }
    __syncthreads();
    if (t < 256) {
        cp -= cs;
        xp -= xs;
        for (int i = 0; i < t >> 6; i++) { xp += s.sh[i]; cp += (unsigned)s.sh[4 + i]; }
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int b = t * EACH + e;
            if (b <= NB + 1) { s.cx[b] = cp; s.wx[b] = xp; }
            cp += c[e];
            xp += x[e];
        }
    }
    __syncthreads();
    picker<E> pk{a, row, w, s, in_head};
    pk.pick(r, p, m, uf);
}

template <class E>
void launch(const smp_args &a, hipStream_t st) {
    const size_t lds = sizeof(pick_lds);
    static std::atomic<unsigned long long> done[2];
    if (a.parts == 1) {
        ps_allow_lds((const void *)sample_pick_kernel<E, true>, lds, done[0]);
        hipLaunchKernelGGL((sample_pick_kernel<E, true>), dim3((unsigned)a.rows), dim3(PICK), lds, st, a);
        return;
    }
    ps_allow_lds((const void *)sample_pick_kernel<E, false>, lds, done[1]);
    hipLaunchKernelGGL((sample_top_kernel<E>), dim3((unsigned)a.parts, (unsigned)a.rows), dim3(256), 0, st, a);
    hipLaunchKernelGGL((sample_head_kernel<E>), dim3((unsigned)a.parts, (unsigned)a.rows), dim3(PICK), 0, st, a);
    hipLaunchKernelGGL((sample_pick_kernel<E, false>), dim3((unsigned)a.rows), dim3(PICK), lds, st, a);
}
} // namespace

// the pieces of the scratch memory of `rows` rows in `all` parts together
static void sample_carve(smp_args &a, ps_carve &ws, size_t rows, size_t all) {
    a.top = ws.take<float>(rows * 1024);
    a.bound = ws.take<float>(rows * 2);
    a.cnt = ws.take<unsigned>(all * (NB + 1));
    a.sum = ws.take<u64>(all * (NB + 1));
    a.head = ws.take<u64>(all * PART_HEAD);
    a.held = ws.take<unsigned>(all);
}
// The most that any call of up to n logits and up to `rows` rows takes: the rows that have parts are up to half the CUs, and their parts up to two a CU.
size_t psv_sample_most(int n_cu, int64_t n, int64_t rows) {
    const int64_t least = 1024, r = std::min<int64_t>(rows, n_cu / 2);
    if (r < 1 || n < 4 * least) return 0;
    int parts = 4;
    while (parts < 64 && parts * 2 * least <= n) parts *= 2;
    smp_args a{};
    ps_carve ws{nullptr};
    sample_carve(a, ws, (size_t)r, (size_t)std::min<int64_t>(r * parts, 2 * n_cu));
    return ws.at;
}
size_t psv_sample_space(int n_cu, int dtype, const void *logits, int64_t n, int64_t rows, int64_t stride, const ps_sample_params *p, int32_t *ids, float *prob, void *base, bool launch_, hipStream_t st) {
    smp_args a{};
    // a row alone where there is a row for half the CUs; else 4, 8 .. 64 parts (1024 groups of a row in all) of at least a piece of 16 bytes a thread, as many as the chip takes at once
    const int64_t least = dtype == PS_F32 ? 1024 : 2048;
    a.parts = 1;
    if (rows * 2 <= n_cu && n >= 4 * least)
        for (a.parts = 4; a.parts < 64 && a.parts * 2 * rows <= 2 * n_cu && a.parts * 2 * least <= n;) a.parts *= 2;
    ps_carve ws{(char *)base};
    if (a.parts > 1) sample_carve(a, ws, (size_t)rows, (size_t)rows * a.parts);
    if (!launch_) return ws.at;
    a.logits = logits; a.n = (int)n; a.rows = rows; a.stride = stride;
    a.temperature = p->temperature; a.top_k = p->top_k; a.top_p = p->top_p; a.min_p = p->min_p; a.u = p->u;
    a.ids = ids; a.prob = prob;
    int bits = 0;
    while (((int64_t)1 << bits) < n) bits++;
    a.scale = std::min(51, 62 - bits); // a row's weights add up to at most 2^62, one is below 2^52
    if (dtype == PS_F32) launch<F32>(a, st);
    else if (dtype == PS_F16) launch<F16>(a, st);
    else launch<BF16>(a, st);
    return ws.at;
}
