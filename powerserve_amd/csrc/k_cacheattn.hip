// Attention of the newest tokens of many sequences over their caches (ps_hip_cache_attn), with the attention weight every slot receives, and taking an accepted path (ps_hip_cache_advance).
//   O = softmax(scale Q K^T + mask) V per kv head; its rows are the new tokens times the query heads that share the head (row t R + r: token t, query head r of R), its keys the held slots and the
//   new tokens.  Weight of a slot = the sum over rows of its soft-max weights.
//   cache_attn_kernel     16 RT rows of one kv head against a part of its keys; the waves of a work-group share the part (blocks of 32 keys in turn), join in LDS, and leave sum, maximum and
//                         unnormed result of the part -- or the result itself where there is one part.  New rows go into the cache on the way.
//   cache_join_kernel     the parts of a row together; up to 32 rows, beside that: a slot's weights from the scores, which cache_attn_kernel leaves beside its result
//   cache_append_kernel, cache_rows_kernel, cache_receive_kernel, cache_gather_kernel   the same for more rows of a 16-bit cache, cache_weight_kernel of an fp32 one: the scores are made again for the
//                         weights
// S^T = K Q^T, so that a lane has one row and maximum and sum run over its own registers and two lane moves; the second product O^T = V^T P^T takes its 32 keys in any order that both operands
// share, so a lane's weights are its piece of the operand as they are.  16-bit values pass through LDS, a wave's own stretch, and come back transposed (ds_read_b64_tr_b16: 4 keys x 16 numbers).
// Lengths are read on the device; a part is ceil(length / parts) keys, so that a fixed grid serves any length.
// Measured, dim 128, 32 query heads of 8, bf16: one token of 32 sequences that hold 17 to 8191 slots, with weights, 54 + 10 us, 187 MB of keys and values at 3.5 TB/s (the library's sum over 1 GiB 4.0, this
// repository's mat-vec 4.8) -- memory, and short work-groups whose plan and first block's loads nothing hides; 2048 tokens behind 2047, 175 + 90 us for 103 and 52 GFLOP, 590 and 580 TFLOP/s (the library's product of
// 8192^3: 1130) -- the soft-max on the vector units and the products on the matrix units, busy 55 and 51 % of the CUs' time in the first and 47 and 30 % in the second: they hardly run at the same time; one
// token behind 100 in fp32 (14 heads of 2, dim 64), 9 + 4 us: latency of lengths, keys, sums and two launches.
#include "ps_serve.h"

#include <algorithm>
#include <cmath>

namespace {
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
struct F16 { static constexpr int SIZE = 2; };
struct BF16 { static constexpr int SIZE = 2; };
struct F32 { static constexpr int SIZE = 4; };

struct ca_args {
    char *k, *v, *out;
    const char *q, *k_new, *v_new;
    long long seq, slot, head, q_seq, q_row, o_seq, o_row, new_seq, new_row; // strides in bytes
    int n_seqs, n_ctx, G, dim, R, T;
    unsigned by_R; // 2^32 / R, rounded up: what a row of fewer than 2^32 / R is divided with (R 1: 0)
    float sc2; // scale, times log2(e) where scores are held in units of log 2
    const int32_t *n_kv, *count, *pos_new;
    int32_t *pos;
    const uint8_t *tree;
    const float *weight;
    float *weight_out;
    float *part; // [seq][kv head][16 rows][part]: 16 x dim results, the 16 scores that their weights are taken against, 16 sums
    float *score; // [seq][kv head][slot][score_rows]: scores of few rows for the weights, or NULL
    float *lse;  // [seq][kv head][T R] logarithm, in the scores' units, of the sum of weights (+inf: no weights)
    int parts, tiles, score_rows; // tiles of 16 rows
    int share, *chunks; // 2 to 256 sequences in parts: work-groups that all their keys are shared out to, and keys of a part of each sequence; else 0, NULL
    int plain; // offsets within 32 slots fit 32 bits
    int near;  // offsets within a sequence's q do
    int scorers;      // few rows: work-groups of a kv head that make its weights from scores
    int wgroups;      // many rows: work-groups of a kv head that the weights' work is shared out to (0: one each 256 slots)
    float *wpart;     // [seq][kv head][work-group + block of 256 slots][256]: sums of a work-group's rows of a block
};
struct ca_lens { int n0, cnt, len; };
__device__ __forceinline__ int token_of(const ca_args &a, int row) { return a.by_R ? (int)__umulhi((unsigned)row, a.by_R) : row; }
__device__ __forceinline__ ca_lens lens_of(const ca_args &a, int s) {
    ca_lens l;
    l.n0 = min(max(a.n_kv[s], 0), a.n_ctx);
    l.cnt = min(max(a.count ? a.count[s] : a.T, 0), min(a.T, a.n_ctx - l.n0));
    l.len = l.n0 + l.cnt;
    return l;
}
// keys of a part of sequence s
__device__ __forceinline__ int chunk_of(const ca_args &a, int s, int len) {
    if (a.chunks) return a.chunks[s];
    return max(128, ((len + a.parts - 1) / a.parts + 127) / 128 * 128);
}
__device__ __forceinline__ bool sees(const ca_args &a, int s, int t, int u) { return a.tree ? a.tree[((long long)s * a.T + t) * a.T + u] != 0 : u <= t; }
// Which of the new tokens x .. x + 3 (below 0: held slots, which all see) token t sees, a bit each.  A tree's four bytes are one load, whatever their alignment, moved so that it stays in the row: a
// byte after the other would be as many waits for the L2 in the last block of every sequence.
__device__ __forceinline__ unsigned sees4(const ca_args &a, const ca_lens &L, int s, int t, int x) {
    auto ones = [](int n) { return (1u << min(max(n, 0), 4)) - 1; };
    if (!a.tree) return ones(min(t, L.cnt - 1) - x + 1);
    const uint8_t *row = a.tree + ((long long)s * a.T + t) * a.T;
    const int at = min(max(x, 0), max(a.T - 4, 0)), d = x - at;
    unsigned v = 0;
    if (a.T >= 4) __builtin_memcpy(&v, row + at, 4);
    else
        for (int i = 0; i < a.T; i++) v |= (unsigned)row[i] << 8 * i;
    v = ((((v & 0x7f7f7f7fu) + 0x7f7f7f7fu) | v) & 0x80808080u) >> 7; // a byte that is not 0: 1
    v = v * 0x10204080u >> 28;
    v = d >= 0 ? v >> min(d, 4) : v << min(-d, 4) | ones(-d);
    return v & ones(L.cnt - x);
}

template <class E> __device__ __forceinline__ pv_f4 mfma(const pv_u4 &x, const pv_u4 &y, const pv_f4 &c);
template <> __device__ __forceinline__ pv_f4 mfma<BF16>(const pv_u4 &x, const pv_u4 &y, const pv_f4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
}
template <> __device__ __forceinline__ pv_f4 mfma<F16>(const pv_u4 &x, const pv_u4 &y, const pv_f4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0, 0);
}
// two numbers to 16 bits, to nearest even, and what that leaves
template <class E> __device__ __forceinline__ unsigned round2(float a, float b) {
    if constexpr (sizeof(E) && __is_same(E, BF16)) return __builtin_bit_cast(unsigned, __builtin_convertvector((pv_f2){a, b}, b2));
    else return __builtin_bit_cast(unsigned, __builtin_convertvector((pv_f2){a, b}, h2));
}
template <class E> __device__ __forceinline__ pv_f2 wide2(unsigned u) {
    if constexpr (__is_same(E, BF16)) return (pv_f2){__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)};
    else { const h2 h = __builtin_bit_cast(h2, u); return (pv_f2){(float)h[0], (float)h[1]}; }
}
template <class E> __device__ __forceinline__ unsigned odd_bits(unsigned u) { // not 0: infinities or NaN among the numbers of 32 bits (an exponent of ones and one more is the sign's bit)
    if constexpr (E::SIZE == 4) return ((u & 0x7f800000u) + 0x00800000u) & 0x80000000u;
    constexpr unsigned m = __is_same(E, BF16) ? 0x7f807f80u : 0x7c007c00u, one = __is_same(E, BF16) ? 0x00800080u : 0x04000400u;
    return ((u & m) + one) & 0x80008000u;
}
// the others of them alone
template <class E> __device__ __forceinline__ unsigned without_odd(unsigned u) {
    if constexpr (E::SIZE == 4) return odd_bits<E>(u) ? 0u : u;
    constexpr unsigned m = __is_same(E, BF16) ? 0x7f80u : 0x7c00u;
    return ((u & m) == m ? 0u : u & 0xffffu) | ((u >> 16 & m) == m ? 0u : u & 0xffff0000u);
}
// Scores of 16-bit caches are held in units of log 2, and 2^x is the instruction's.  Those of fp32 caches are as they are, and e^x is 2^(x log2 e) with what the product rounds off put back: 2^-23 of
// it, where the instruction alone would have 2^-24 of the exponent.
template <class E> __device__ __forceinline__ float ex(float x) {
    if constexpr (E::SIZE == 2) return __builtin_amdgcn_exp2f(x);
    else {
        const float y = x * 1.44269504f, lo = fmaf(x, 1.44269504f, -y) + x * 1.92596299e-8f, e = __builtin_amdgcn_exp2f(y);
        return x < -104.f ? 0.f : fmaf(e, lo * 0.693147181f, e);
    }
}
// The score that a row's weights are taken against, from its largest: e^(score - this).  It cancels in the result and in the sums' logarithm.  fp16 weights are up to 2^15 instead of 1 (65504 is the largest
// number), so that one keeps its 11 bits down to 2^-29 of the largest, and its second number to 2^-40 of it: thousands of small weights beside an attention sink are the result where the sink's value is
// small.  From 2^20 on, where a float's steps are an eighth and more, the largest itself.
template <class E> __device__ __forceinline__ float against(float top) {
    if constexpr (__is_same(E, F16)) return fabsf(top) < 1048576.f ? top - 15.f : top;
    else return top;
}
template <class E> __device__ __forceinline__ float lg(float x) { return E::SIZE == 2 ? log2f(x) : logf(x); }
__device__ __forceinline__ bool odd32(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }
template <class E> __device__ __forceinline__ float number(const char *p) {
    if constexpr (E::SIZE == 4) return *(const float *)p;
    else return wide2<E>(*(const unsigned short *)p)[0];
}

// The frames of operands.  16-bit: a lane's piece of 16 x 32 numbers is 8 numbers of one row, of k step s 32 s + 8 (l / 16) ..; fp32: four steps' numbers at once, 16 s + 4 (l / 16) ..
template <class E, int DP> constexpr int STEPS = E::SIZE == 2 ? DP / 32 : DP / 16;
template <class E, int DP> using frame = pv_u4[STEPS<E, DP>];
template <class E, int DP>
__device__ __forceinline__ void get_row(frame<E, DP> &f, const char *row, int q, int dim) { // zeros behind dim
#pragma unroll
    for (int s = 0; s < STEPS<E, DP>; s++) {
        const int e = E::SIZE == 2 ? 32 * s + 8 * q : 16 * s + 4 * q;
        f[s] = *(const pv_u4 *)(row + (e < dim ? e * E::SIZE : 0));
        if (e >= dim) f[s] = (pv_u4){0, 0, 0, 0};
    }
}
template <class E, int DP>
__device__ __forceinline__ pv_f4 dot(const frame<E, DP> &k, const frame<E, DP> &q) {
    pv_f4 c = {0.f, 0.f, 0.f, 0.f}, d = c;
#pragma unroll
    for (int s = 0; s < STEPS<E, DP>; s++) {
        if constexpr (E::SIZE == 2) c = mfma<E>(k[s], q[s], c);
        else {
            // two sums of half the products each: what a score is off by is most of what an fp32 result is (one token behind 101 slots: 4.4e-7 with one sum, 2.6e-7 so, 2.5e-7 with four, whose registers cost
            // many rows 8 to 14 % of their time, these two 1 to 2 %)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[s][e]), __uint_as_float(q[s][e]), c, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[s][e + 1]), __uint_as_float(q[s][e + 1]), d, 0, 0, 0);
            }
        }
    }
    if constexpr (E::SIZE == 4) c += d;
    return c;
}

constexpr int VPAD = 16; // numbers behind a value row in LDS: four rows of eight banks side by side

// Parts of a step's work, all of much the same size: the keys of all sequences shared out, so that one long sequence among short ones does not keep a few work-groups busy and none is started for
// slots that nobody holds.  Every work-group of 256 threads finds the same plan from the lengths (a thread a sequence), and what it has of it; false: nothing.
__device__ __forceinline__ bool shared_part(const ca_args &a, int id, int blocks, int &rb, int &g, int &s, int &split, int &chunk) {
    __shared__ int before[257], chunk_at[256], sums[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const ca_lens mine = tid < a.n_seqs ? lens_of(a, tid) : ca_lens{0, 0, 0};
    const int len = mine.cnt ? mine.len : 0;
    int x = len;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    if (lane == 0) sums[wave] = x;
    __syncthreads();
    const long long all = (long long)sums[0] + sums[1] + sums[2] + sums[3], even = (all * a.G * blocks + a.share - 1) / a.share;
    const int keys = max(128, (int)((max(even, (long long)((len + a.parts - 1) / a.parts)) + 127) / 128 * 128));
    chunk_at[tid] = keys;
    if (id == 0 && tid < a.n_seqs) a.chunks[tid] = keys;
    x = len ? (len + keys - 1) / keys : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    for (int i = 0; i < wave; i++) x += sums[i];
    before[tid + 1] = x;
    if (tid == 0) before[0] = 0;
    __syncthreads();
    if (id >= before[256] * a.G * blocks) return false;
    rb = id % blocks; id /= blocks;
    g = id % a.G; id /= a.G;
    int lo = 0, hi = a.n_seqs - 1; // the last sequence whose parts begin at id or before
    while (lo < hi) {
        const int m = (lo + hi + 1) / 2;
        if (before[m] <= id) lo = m;
        else hi = m - 1;
    }
    s = lo;
    split = id - before[s];
    chunk = chunk_at[s];
    return true;
}
// The next block's keys and values are on their way while one is worked on; two work-groups a CU (three or four leave no registers for that: slower).  fp32 runs on v_mfma_f32_16x16x4: 1024 tokens behind
// 1000, dim 64 55 TFLOP/s, dim 128, whose registers leave one work-group a CU, 50 (the library's product: 153).
template <class E, int DP, int RT>
__global__ __launch_bounds__(256, E::SIZE == 4 && DP == 128 ? 1 : 2) void cache_attn_kernel(const ca_args a) {
    constexpr int NS = STEPS<E, DP>, ND = DP / 16, OP = DP + 4, VR = DP + VPAD;
    constexpr int VBYTES = E::SIZE == 2 ? 4 * 32 * VR * 2 : 0, OBYTES = 4 * 16 * OP * 4;
    __shared__ __attribute__((aligned(16))) char lds[VBYTES > OBYTES ? VBYTES : OBYTES];
    __shared__ float lm[4][16], ll[4][16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, q4 = lane >> 4;
    const int blocks = (a.tiles + RT - 1) / RT;
    int rb, g, s, split, chunk;
    if (a.share) {
        if (!shared_part(a, blockIdx.x, blocks, rb, g, s, split, chunk)) return;
    } else {
        int id = blockIdx.x;
        rb = id % blocks; id /= blocks;
        split = id % a.parts; id /= a.parts;
        g = id % a.G;
        s = id / a.G;
    }
    rb = blocks - 1 - rb; // (the rows with the most causal keys first)
    const ca_lens L = lens_of(a, s);
    if (!a.share) chunk = chunk_of(a, s, L.len);
    const int k0 = split * chunk, rows_ = L.cnt * a.R;
    if (L.cnt == 0 || k0 >= L.len || rb * RT * 16 >= rows_) return;
    // row blocks but the last stop where none of their rows sees any key
    const bool last = (rb + 1) * RT * 16 >= rows_;
    const int k1 = min(min(L.len, k0 + chunk), last || a.tree ? L.len : L.n0 + token_of(a, rb * RT * 16 + RT * 16 - 1) + 1);
    const char *kb_ = a.k + s * a.seq + g * a.head, *vb_ = a.v + s * a.seq + g * a.head;
    const char *kn = a.k_new ? a.k_new + s * a.new_seq + (long long)g * a.dim * E::SIZE : nullptr, *vn = a.k_new ? a.v_new + s * a.new_seq + (long long)g * a.dim * E::SIZE : nullptr;
    auto row_at = [&](const char *held, const char *fresh, int j) { return fresh && j >= L.n0 ? fresh + (j - L.n0) * a.new_row : held + j * a.slot; };

    pv_u4 qf[RT][NS];
    int tok[RT];
    pv_f4 o[RT][ND];
    float m[RT], l[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) {
        const int row = min((rb * RT + r) * 16 + c, L.cnt * a.R - 1); // rows behind the last repeat it
        tok[r] = token_of(a, row);
        get_row<E, DP>(qf[r], a.q + s * a.q_seq + tok[r] * a.q_row + (long long)(g * a.R + row - tok[r] * a.R) * a.dim * E::SIZE, q4, a.dim);
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; d++) o[r][d] = (pv_f4){0.f, 0.f, 0.f, 0.f};
    }
    bool odd = false; // a new token's values hold infinities or NaN: they stay out of the products and join those rows that see them
    unsigned short *vl = (unsigned short *)lds + wave * 32 * VR;

    // a block's operands: keys of two tiles of 16; values as rows (16-bit) or as they are multiplied (fp32: keys 4 (l / 16) + i, numbers 64 x + 4 c ..)
    constexpr int LPR = DP / 8, RPI = 64 / LPR, VI = E::SIZE == 2 ? 32 / RPI : 8 * (DP / 64);
    pv_u4 kf[2][NS], vf[VI];
    const int vr = lane / LPR, vc = lane % LPR * 8;
    constexpr int ES = E::SIZE;
    const unsigned ko = c * (unsigned)a.slot + q4 * 16, vo = ES == 2 ? vr * (unsigned)a.slot + vc * 2 : 4 * q4 * (unsigned)a.slot + c * 16;
    auto fetch = [&](int kb) {
        if ((RT == 1 || ES == 4) && kb + 32 <= (kn ? min(L.n0, k1) : k1) && a.plain && a.dim == DP) { // slots of the cache: one place a wave, and an offset a lane
            const char *kt = kb_ + kb * a.slot, *vt = vb_ + kb * a.slot;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int st = 0; st < NS; st++) kf[u][st] = *(const pv_u4 *)(kt + 16 * u * a.slot + 64 * st + ko);
#pragma unroll
            for (int i = 0; i < VI; i++) {
                const int r = ES == 2 ? i * RPI : 16 * (i / (4 * (DP / 64))) + i / (DP / 64) % 4;
                vf[i] = *(const pv_u4 *)(vt + r * a.slot + (ES == 2 ? 0 : 256 * (i % (DP / 64))) + vo);
            }
            return;
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int j = min(kb + 16 * u + c, k1 - 1);
            get_row<E, DP>(kf[u], row_at(kb_, kn, j), q4, a.dim);
        }
#pragma unroll
        for (int i = 0; i < VI; i++) {
            const int r = E::SIZE == 2 ? i * RPI + vr : 16 * (i / (4 * (DP / 64))) + 4 * q4 + i / (DP / 64) % 4, e = E::SIZE == 2 ? vc : 64 * (i % (DP / 64)) + 4 * c;
            const int j = kb + r;
            vf[i] = *(const pv_u4 *)(row_at(vb_, vn, min(j, k1 - 1)) + (e < a.dim ? e * E::SIZE : 0));
            if (j >= k1 || e >= a.dim) vf[i] = (pv_u4){0, 0, 0, 0};
        }
    };
    if (k0 + wave * 32 < k1) fetch(k0 + wave * 32);
    for (int kb = k0 + wave * 32; kb < k1; kb += 128) {
        if (kb + 32 > L.n0) { // new tokens among the keys
            if (kn) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int j = kb + 16 * u + c;
                    if (j >= L.n0 && j < k1) {
#pragma unroll
                        for (int st = 0; st < NS; st++) {
                            const int e = E::SIZE == 2 ? 32 * st + 8 * q4 : 16 * st + 4 * q4;
                            if (e < a.dim) *(pv_u4 *)(a.k + s * a.seq + g * a.head + j * a.slot + e * E::SIZE) = kf[u][st];
                        }
                        if (q4 == 0 && a.pos_new && a.pos) a.pos[((long long)s * a.G + g) * a.n_ctx + j] = a.pos_new[(long long)s * a.T + j - L.n0];
                    }
                }
            }
            unsigned any = 0;
#pragma unroll
            for (int i = 0; i < VI; i++)
#pragma unroll
                for (int x = 0; x < 4; x++) any |= odd_bits<E>(vf[i][x]);
            if (any || vn)
#pragma unroll
                for (int i = 0; i < VI; i++) {
                    const int r = E::SIZE == 2 ? i * RPI + vr : 16 * (i / (4 * (DP / 64))) + 4 * q4 + i / (DP / 64) % 4, e = E::SIZE == 2 ? vc : 64 * (i % (DP / 64)) + 4 * c;
                    const int j = kb + r;
                    if (j < L.n0 || j >= k1 || e >= a.dim) continue;
                    if (vn) *(pv_u4 *)(a.v + s * a.seq + g * a.head + j * a.slot + e * E::SIZE) = vf[i];
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (odd_bits<E>(vf[i][x])) { odd = true; vf[i][x] = without_odd<E>(vf[i][x]); }
                }
        }
        pv_u4 vk[VI];
        if constexpr (E::SIZE == 2) {
#pragma unroll
            for (int i = 0; i < VI; i++) *(pv_u4 *)(vl + (i * RPI + vr) * VR + vc) = vf[i];
        } else {
#pragma unroll
            for (int i = 0; i < VI; i++) vk[i] = vf[i];
        }
        pv_f4 z[RT][2];
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int u = 0; u < 2; u++) z[r][u] = dot<E, DP>(kf[u], qf[r]);
        if (kb + 128 < k1) fetch(kb + 128);
        const bool edge = kb + 32 > min(L.n0, k1);
#pragma unroll
        for (int r = 0; r < RT; r++) {
            unsigned seen = 0;
            if (edge)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int j = kb + 16 * u + 4 * q4;
                    seen |= (sees4(a, L, s, tok[r], j - L.n0) & ((1u << min(max(k1 - j, 0), 4)) - 1)) << 4 * u;
                }
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float v = z[r][u][i] * a.sc2;
                    if (edge && !(seen >> (4 * u + i) & 1)) v = -INFINITY;
                    z[r][u][i] = v;
                    top = fmaxf(top, v);
                }
            if (a.score) {
                float *sc = a.score + (((long long)s * a.G + g) * a.n_ctx + kb + 4 * q4) * a.score_rows + (rb * RT + r) * 16 + c;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if ((rb * RT + r) * 16 + c < L.cnt * a.R && kb + 16 * u + 4 * q4 + i < k1) sc[(16 * u + i) * a.score_rows] = z[r][u][i];
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float mn = fmaxf(m[r], against<E>(top)), ms = mn == -INFINITY ? 0.f : mn, al = ex<E>(m[r] - ms);
            float p[8], sum = 0.f;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    p[4 * u + i] = ex<E>(z[r][u][i] - ms);
                    sum += p[4 * u + i];
                }
            m[r] = mn;
            l[r] = fmaf(l[r], al, sum);
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[r][d][i] *= al;
            if constexpr (E::SIZE == 2) {
                // the weights as two 16-bit numbers each: what the second product rounds off is 2^-17 (bf16; fp16 2^-23, and 2^-40 of the row's largest where that is more) of a weight, not the 2^-9 that
                // would stand beside the result's own rounding; these products are not what bounds a pass over the cache
                pv_u4 hi, lo;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    hi[x] = round2<E>(p[2 * x], p[2 * x + 1]);
                    const pv_f2 w = wide2<E>(hi[x]);
                    lo[x] = round2<E>(p[2 * x] - w[0], p[2 * x + 1] - w[1]);
                }
                const unsigned short *base = vl + (4 * q4 + (c >> 2)) * VR + 4 * (c & 3);
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    typedef __attribute__((address_space(3))) s4 lds_s4;
                    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(base + 16 * d)), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(base + 16 * VR + 16 * d));
                    pv_u4 vt;
                    const pv_u2 xx = __builtin_bit_cast(pv_u2, x), yy = __builtin_bit_cast(pv_u2, y);
                    vt[0] = xx[0]; vt[1] = xx[1]; vt[2] = yy[0]; vt[3] = yy[1];
                    o[r][d] = mfma<E>(vt, hi, o[r][d]);
                    o[r][d] = mfma<E>(vt, lo, o[r][d]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < VI; i++) {
                    const int x = i % (DP / 64);
#pragma unroll
                    for (int e = 0; e < 4; e++) o[r][4 * x + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vk[i][e]), p[i / (DP / 64)], o[r][4 * x + e], 0, 0, 0);
                }
            }
        }
    }
    // the four waves together
    float *ol = (float *)lds;
    odd = __syncthreads_or(odd);
#pragma unroll
    for (int r = 0; r < RT; r++) {
        if (r) __syncthreads();
        l[r] += __shfl_xor(l[r], 16, 64);
        l[r] += __shfl_xor(l[r], 32, 64);
        if (q4 == 0) { lm[wave][c] = m[r]; ll[wave][c] = l[r]; }
        float *mine = ol + (wave * 16 + c) * OP;
        if constexpr (E::SIZE == 2) {
#pragma unroll
            for (int d = 0; d < ND; d++) *(pv_f4 *)(mine + 16 * d + 4 * q4) = o[r][d];
        } else {
#pragma unroll
            for (int x = 0; x < DP / 64; x++)
#pragma unroll
                for (int i = 0; i < 4; i++) *(pv_f4 *)(mine + 64 * x + 16 * q4 + 4 * i) = (pv_f4){o[r][4 * x][i], o[r][4 * x + 1][i], o[r][4 * x + 2][i], o[r][4 * x + 3][i]};
        }
        __syncthreads();
        const int tile = rb * RT + r, rr = tid >> 4, row = tile * 16 + rr;
        if (row >= L.cnt * a.R) continue;
        float top = fmaxf(fmaxf(lm[0][rr], lm[1][rr]), fmaxf(lm[2][rr], lm[3][rr])), f[4], sum = 0.f;
        const float ms = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < 4; w++) { f[w] = ex<E>(lm[w][rr] - ms); sum = fmaf(ll[w][rr], f[w], sum); }
        const int t = token_of(a, row), hd = g * a.R + row - t * a.R;
        float *part = a.part + ((((long long)s * a.G + g) * a.tiles + tile) * a.parts + split) * (16 * (a.dim + 2));
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        for (int e = (tid & 15) * 4; e < a.dim; e += 64) {
            pv_f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const pv_f4 x = *(const pv_f4 *)(ol + (w * 16 + rr) * OP + e);
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = fmaf(x[i], f[w], v[i]);
            }
            if (odd)
                for (int j = max(k0, L.n0); j < k1; j++) {
                    if (!sees(a, s, t, j - L.n0)) continue;
                    const char *src = row_at(vb_, vn, j) + e * E::SIZE;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float x = number<E>(src + i * E::SIZE);
                        if (odd32(x)) v[i] += x;
                    }
                }
            // An infinite value is NaN by now where it met a weight's second number, which may be 0 or below it, or a weight or a factor too small for its type: what the infinities and NaN that the row
            // sees add up to, where the row's weights are numbers and there are any
            if (sum == sum && (v[0] != v[0] || v[1] != v[1] || v[2] != v[2] || v[3] != v[3])) {
                pv_f4 x = {0.f, 0.f, 0.f, 0.f};
                auto add = [&](int j) {
                    const char *src = row_at(vb_, vn, j) + e * E::SIZE;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float y = number<E>(src + i * E::SIZE);
                        x[i] += odd32(y) ? y : 0.f;
                    }
                };
#pragma unroll 4
                for (int j = k0; j < min(k1, L.n0); j++) add(j);
                for (int j = max(k0, L.n0); j < k1; j++)
                    if (sees(a, s, t, j - L.n0)) add(j);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (v[i] != v[i] && x[i] != 0.f) v[i] = x[i];
            }
            if (a.parts > 1) *(pv_f4 *)(part + rr * a.dim + e) = v;
            else {
                char *dst = a.out + s * a.o_seq + t * a.o_row + ((long long)hd * a.dim + e) * E::SIZE;
                if constexpr (E::SIZE == 2) *(pv_u2 *)dst = (pv_u2){round2<E>(v[0] * inv, v[1] * inv), round2<E>(v[2] * inv, v[3] * inv)};
                else *(pv_f4 *)dst = (pv_f4){v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
            }
        }
        if ((tid & 15) == 0) {
            if (a.parts > 1) { part[16 * a.dim + rr] = top; part[16 * a.dim + 16 + rr] = sum; }
            else a.lse[((long long)s * a.G + g) * a.T * a.R + row] = sum == 0.f ? INFINITY : ms + lg<E>(sum);
        }
    }
}

// Row r of a tile from the maxima and sums of its n parts, by four lanes 16 apart: the sum, its logarithm for the weights, and what each part's result is multiplied with (f: LDS, or NULL)
template <class E> __device__ __forceinline__ float row_sum(const ca_args &a, const float *part, int n, int r, int lane4, float (*f)[16], float &lse) {
    const long long step = 16 * (a.dim + 2);
    const float *m = part + 16 * a.dim + r, *l = m + 16;
    float top = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int i = lane4; i < n; i += 4) top = fmaxf(top, m[i * step]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float ms = top == -INFINITY ? 0.f : top;
#pragma unroll 4
    for (int i = lane4; i < n; i += 4) {
        const float v = m[i * step], x = ex<E>(v - ms);
        sum = fmaf(l[i * step], x, sum);
        if (f) f[i][r] = v == -INFINITY ? 0.f : fmaxf(x, 1e-45f); // (an infinite result counts however small its part's weights are)
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    lse = sum == 0.f ? INFINITY : ms + lg<E>(sum);
    return sum;
}
// The first `joins` work-groups: a tile's parts together, 16 lanes a row; where it has fewer rows the others take parts of them.  Behind them, up to 32 rows: the weights from the scores that the
// attention has left, a thread a key, `scorers` work-groups a kv head, which work the rows' sums out for themselves instead of waiting for them (32 sequences of up to 8191, one launch behind the
// other: 16.5 us, 10.3 so; the number of work-groups, empty ones among them, is what it costs: 2 n_cu of them 17.5, 4 n_cu 12, one each 256 slots 17.5).
template <class E>
__global__ __launch_bounds__(256) void cache_join_kernel(const ca_args a, unsigned joins) {
    __shared__ float f[64][16], total[16], lse[32];
    __shared__ __attribute__((aligned(16))) float acc[16][132];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15;
    unsigned id = blockIdx.x;
    if (id >= joins) {
        id -= joins;
        const int s = (int)(id / a.scorers) / a.G, j0 = (int)(id % a.scorers) * 256;
        const long long head = id / a.scorers;
        const ca_lens L = lens_of(a, s);
        if (j0 >= L.len) return;
        const int rows = L.cnt * a.R, pitch = a.score_rows;
        if (tid < 128) {
            const int tile = tid >> 6, row = tile * 16 + c;
            float x = INFINITY;
            if (tile * 16 < rows) {
                if (a.parts > 1) {
                    const int chunk = chunk_of(a, s, L.len);
                    row_sum<E>(a, a.part + (head * a.tiles + tile) * a.parts * (16 * (a.dim + 2)), (L.len + chunk - 1) / chunk, c, lane >> 4, nullptr, x);
                } else if (row < rows) x = a.lse[head * a.T * a.R + row];
            }
            if (lane < 16) lse[row] = row < rows ? x : INFINITY;
        }
        __syncthreads();
#pragma unroll 2
        for (int j = j0 + tid; j < L.len; j += a.scorers * 256) {
            const long long at = head * a.n_ctx + j;
            float w = 0.f;
            for (int row = 0; row < rows; row += 4) {
                const pv_f4 z = *(const pv_f4 *)(a.score + at * pitch + row);
#pragma unroll
                for (int i = 0; i < 4; i++) w += lse[row + i] == INFINITY ? 0.f : ex<E>(z[i] - lse[row + i]);
            }
            a.weight_out[at] = j < L.n0 && a.weight ? a.weight[at] + w : w;
        }
        return;
    }
    const int tile = id % a.tiles; id /= a.tiles;
    const int g = id % a.G, s = id / a.G;
    const ca_lens L = lens_of(a, s);
    const int rows = min(16, L.cnt * a.R - tile * 16);
    if (rows <= 0) return;
    const int chunk = chunk_of(a, s, L.len), n = (L.len + chunk - 1) / chunk;
    const long long step = 16 * (a.dim + 2);
    const float *part = a.part + (((long long)s * a.G + g) * a.tiles + tile) * a.parts * step;
    if (tid < 64) {
        float x;
        const float sum = row_sum<E>(a, part, n, c, lane >> 4, f, x);
        if (lane < 16) {
            total[c] = sum;
            if (c < rows) a.lse[((long long)s * a.G + g) * a.T * a.R + tile * 16 + c] = x;
        }
    }
    __syncthreads();
    const int nr = rows > 8 ? 16 : rows > 4 ? 8 : rows > 2 ? 4 : rows, groups = 16 / nr, slot = tid >> 4, rr = slot % nr, first = slot / nr;
    const bool has = rr < rows && first < groups;
    for (int e = c * 4; e < a.dim; e += 64) {
        pv_f4 v = {0.f, 0.f, 0.f, 0.f};
        if (has)
#pragma unroll 4
            for (int i = first; i < n; i += groups) {
                const float w = f[i][rr];
                const pv_f4 x = *(const pv_f4 *)(part + i * step + rr * a.dim + e);
#pragma unroll
                for (int y = 0; y < 4; y++) v[y] = w == 0.f ? v[y] : fmaf(x[y], w, v[y]);
            }
        *(pv_f4 *)&acc[slot][e] = v;
    }
    __syncthreads();
    if (slot >= rows) return;
    const int row = tile * 16 + slot, t = token_of(a, row), hd = g * a.R + row - t * a.R;
    const float inv = total[slot] == 0.f ? 0.f : 1.f / total[slot];
    for (int e = c * 4; e < a.dim; e += 64) {
        pv_f4 v = *(const pv_f4 *)&acc[slot][e];
        for (int x = 1; x < groups; x++) v += *(const pv_f4 *)&acc[x * nr + slot][e];
        char *dst = a.out + s * a.o_seq + t * a.o_row + ((long long)hd * a.dim + e) * E::SIZE;
        if constexpr (E::SIZE == 2) *(pv_u2 *)dst = (pv_u2){round2<E>(v[0] * inv, v[1] * inv), round2<E>(v[2] * inv, v[3] * inv)};
        else *(pv_f4 *)dst = (pv_f4){v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
    }
}

// The work of the weights of a kv head: blocks of B slots, each with the tiles of 64 rows that can see a slot of it, one behind the other.  Work-group w of `groups` has the tiles n w / groups ..,
// so that all have as many whatever the lengths are; where it stands changes the group, the block or both, so that group + block is a place of its own for each pair that meets.
constexpr int QT = 64;
template <int B> struct received {
    long long n;  // tiles of all blocks
    int tiles, held, groups; // of a block that all see; blocks that begin before the new tokens; work-groups that have any
    const ca_args &a;
    const ca_lens &L;
    __device__ __forceinline__ int from(int b) const { return a.tree || b < held ? 0 : (b * B - L.n0) * a.R / QT; } // rows of tokens before a block's first slot see none of it
    __device__ __forceinline__ received(const ca_args &a_, const ca_lens &L_) : a(a_), L(L_) {
        tiles = (L.cnt * a.R + QT - 1) / QT;
        const int blocks = (L.len + B - 1) / B;
        held = a.tree ? blocks : min((L.n0 + B - 1) / B, blocks);
        n = (long long)held * tiles;
        for (int b = held; b < blocks; b++) n += tiles - from(b);
        groups = (int)min((long long)a.wgroups, n);
    }
    // the block that tile `at` is in, and the first tile of it
    __device__ __forceinline__ int block_of(long long at, long long &first) const {
        int b = (int)min(at / tiles, (long long)held);
        first = (long long)b * tiles;
        while (b >= held && first + tiles - from(b) <= at) { first += tiles - from(b); b++; }
        return b;
    }
    __device__ __forceinline__ long long start(int w) const { return n * w / groups; }
    __device__ __forceinline__ int group_of(long long tile) const { return (int)(((tile + 1) * groups + n - 1) / n) - 1; }
};
// fp32 caches, more rows: 64 keys of a kv head against the rows that see any, the waves 16 of 64 rows each (1024 tokens behind 1000, 14 heads of 2, dim 64: 53 us, 52 TFLOP/s; a work-group a block: 251)
template <class E, int DP>
__global__ __launch_bounds__(256, 2) void cache_weight_kernel(const ca_args a) {
    constexpr int NS = STEPS<E, DP>;
    __shared__ float red[4][64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c = lane & 15, q4 = lane >> 4;
    int id = blockIdx.x;
    const int heads = a.n_seqs * a.G, hs = id % heads, s = hs / a.G, g = hs - s * a.G; id /= heads;
    const ca_lens L = lens_of(a, s);
    const int rows = L.cnt * a.R;
    const received<64> work(a, L);
    int b = id;
    long long at = 0, end = 0, first = 0; // the tiles that are left, and the block's first
    if (a.wgroups) {
        if (id >= work.groups) return;
        at = work.start(id);
        end = work.start(id + 1);
        b = work.block_of(at, first);
    } else if (b * 64 >= L.len) return;
    const float *lse = a.lse + (long long)hs * a.T * a.R;
#pragma unroll 1
    do {
        int t0 = work.from(b), t1 = work.tiles;
        if (a.wgroups) {
            const int skip = t0;
            t0 = skip + (int)(at - first);
            t1 = (int)min((long long)t1, skip + (end - first));
            at = first = first + work.tiles - skip;
        }
        const int kb = b * 64;
        pv_u4 kf[4][NS];
        float w[4][4] = {};
#pragma unroll
        for (int u = 0; u < 4; u++) get_row<E, DP>(kf[u], a.k + s * a.seq + g * a.head + min(kb + 16 * u + c, L.len - 1) * a.slot, q4, a.dim);
        for (int r0 = t0 * QT + wave * 16; r0 < min(t1 * QT, rows); r0 += QT) {
            const int row = min(r0 + c, rows - 1), t = token_of(a, row);
            pv_u4 qf[NS];
            get_row<E, DP>(qf, a.q + s * a.q_seq + t * a.q_row + (long long)(g * a.R + row - t * a.R) * a.dim * E::SIZE, q4, a.dim);
            const float ls = r0 + c < rows ? lse[row] : INFINITY;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const pv_f4 z = dot<E, DP>(kf[u], qf);
                const unsigned seen = kb + 64 <= L.n0 ? 15u : sees4(a, L, s, t, kb + 16 * u + 4 * q4 - L.n0);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = ls == INFINITY ? 0.f : ex<E>(z[i] * a.sc2 - ls);
                    w[u][i] += seen >> i & 1 ? p : 0.f;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int x = 1; x < 16; x <<= 1) w[u][i] += __shfl_xor(w[u][i], x, 64);
                if (c == 0) red[wave][16 * u + 4 * q4 + i] = w[u][i];
            }
        __syncthreads();
        const int j = kb + lane;
        if (wave == 0) {
            const float sum = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
            if (a.wgroups) a.wpart[(hs * (a.wgroups + (a.n_ctx + 63ll) / 64) + id + b) * 64 + lane] = sum;
            else if (j < L.len) {
                const long long to = (long long)hs * a.n_ctx + j;
                a.weight_out[to] = j < L.n0 && a.weight ? a.weight[to] + sum : sum;
            }
        }
        __syncthreads();
        b++;
    } while (at < end);
}

typedef float f16v __attribute__((ext_vector_type(16)));
template <class E> __device__ __forceinline__ f16v mfma32(const pv_u4 &x, const pv_u4 &y, const f16v &c);
template <> __device__ __forceinline__ f16v mfma32<BF16>(const pv_u4 &x, const pv_u4 &y, const f16v &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f16v mfma32<F16>(const pv_u4 &x, const pv_u4 &y, const f16v &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0, 0);
}
// new rows into the caches, for the forms that read everything from there: 16 bytes a thread
__global__ __launch_bounds__(256) void cache_append_kernel(const ca_args a, int row_bytes) {
    const int s = blockIdx.y;
    const ca_lens L = lens_of(a, s);
    const int per = row_bytes / 16, x = blockIdx.x * 256 + threadIdx.x, t = x / (a.G * per), g = x / per % a.G, e = x % per * 16;
    if (t >= L.cnt) return;
    const long long to = s * a.seq + (L.n0 + t) * a.slot + g * a.head + e, from = s * a.new_seq + t * a.new_row + (long long)g * row_bytes + e;
    *(pv_u4 *)(a.k + to) = *(const pv_u4 *)(a.k_new + from);
    *(pv_u4 *)(a.v + to) = *(const pv_u4 *)(a.v_new + from);
    if (e == 0 && a.pos_new && a.pos) a.pos[((long long)s * a.G + g) * a.n_ctx + L.n0 + t] = a.pos_new[(long long)s * a.T + t];
}

// Many rows of a 16-bit cache: 128 of a kv head against a part of its keys, a wave 32 of them against all, 64 keys at a time through two LDS stages that the four waves fill.  The products are
// v_mfma_f32_32x32x16: S^T = K Q^T with the queries in registers (a lane: one row, 16 keys a tile), O^T = V^T P^T with the weights as they come, values transposed on their way out of LDS.
// The weights go into the second product as two 16-bit numbers each, as in cache_attn_kernel, so that a token's result is as exact among many new tokens as among few; one number each, 2^-9 of a weight off
// (bf16), would take a third fewer matrix instructions (2048 tokens behind 2047: 138 us instead of 175).  Their sum is taken before they are rounded.
// What bounds it: a wave and 64 keys take 48 matrix instructions of 32 clocks, 32 KB of operands from LDS and some 300 vector instructions, which two waves a SIMD hardly run at the same time: matrix units 51 % and
// vector units 55 % of the CUs' time (2048 tokens behind 2047: 175 us, 590 TFLOP/s, 880 with the weights' second numbers).  Work-groups of eight waves read a tile for twice the rows, and their sizes even out
// worse (with one number a weight 168 us there instead of 138; 8192 tokens 5 % faster).
constexpr int ROWS = 128, KEYS = 64;
// which of new tokens x + 8 (i / 4) + i % 4, a lane's 16 keys of a tile of 32, token tok sees, as sees4
__device__ __forceinline__ unsigned sees16(const ca_args &a, const ca_lens &L, int s, int tok, int x) {
    unsigned bits = 0;
#pragma unroll
    for (int q = 0; q < 4; q++) bits |= sees4(a, L, s, tok, x + 8 * q) << 4 * q;
    return bits;
}
template <class E, int DP>
__global__ __launch_bounds__(256, 2) void cache_rows_kernel(const ca_args a) {
    constexpr int KS = DP / 16, MD = DP / 32, KR = DP + 8, VR = DP + 32, PER = DP / 8, ST = KEYS * PER / 256; // rows in LDS: 16 banks further for the next value row, 4 for the next key
    __shared__ __attribute__((aligned(16))) unsigned short kl[2][KEYS * KR], vl[2][KEYS * VR];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c = lane & 31, h = lane >> 5;
    const int rows_all = a.T * a.R, blocks = (rows_all + ROWS - 1) / ROWS;
    int rb, g, s, split, chunk;
    if (a.share) {
        if (!shared_part(a, blockIdx.x, blocks, rb, g, s, split, chunk)) return;
    } else {
        // neighbours are kv heads, so that a head's keys stay in one XCD's L2; the rows with the most causal keys first, those with the fewest from the middle on: a CU's two work-groups add up alike
        const int heads = a.n_seqs * a.G, hs = blockIdx.x % heads, id = blockIdx.x / heads, p = id / a.parts, half = (blocks + 1) / 2;
        s = hs / a.G;
        g = hs - s * a.G;
        split = id % a.parts;
        rb = p < half ? blocks - 1 - p : p - half;
    }
    const ca_lens L = lens_of(a, s);
    if (!a.share) chunk = chunk_of(a, s, L.len);
    const int rows = L.cnt * a.R, k0 = split * chunk, k1 = min(L.len, k0 + chunk);
    if (rb * ROWS >= rows || k0 >= L.len) return;
    const int r0 = rb * ROWS + wave * 32, row = min(r0 + c, rows - 1), tok = token_of(a, row), first = token_of(a, min(r0, rows - 1));
    const int kend = a.tree ? k1 : min(k1, L.n0 + token_of(a, min(rb * ROWS + ROWS - 1, rows - 1)) + 1); // behind the last key that a row of the work-group sees
    const char *kb_ = a.k + s * a.seq + g * a.head, *vb_ = a.v + s * a.seq + g * a.head;
    pv_u4 qf[KS];
    {
        const char *q = a.q + s * a.q_seq + tok * a.q_row + (long long)(g * a.R + row - tok * a.R) * a.dim * 2;
#pragma unroll
        for (int st = 0; st < KS; st++) {
            const int e = 16 * st + 8 * h;
            qf[st] = *(const pv_u4 *)(q + (e < a.dim ? e * 2 : 0));
            if (e >= a.dim) qf[st] = (pv_u4){0, 0, 0, 0};
            if (a.sc2 < 0.f) qf[st] ^= 0x80008000u; // a negative scale turns the queries round
        }
    }
    const float sc = fabsf(a.sc2);
    f16v o[MD];
#pragma unroll
    for (int m = 0; m < MD; m++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[m][i] = 0.f;
    float mx = -INFINITY, l = 0.f;
    bool odd = false;
    pv_u4 ks[ST], vs[ST];
    long long off[ST]; // of a thread's pieces of a tile
#pragma unroll
    for (int i = 0; i < ST; i++) { const int x = tid + 256 * i, e = x % PER * 8; off[i] = x / PER * a.slot + (e < a.dim ? e * 2 : 0); }
    auto fetch = [&](int kb) {
        if (kb + KEYS <= L.len && a.dim == DP) {
            const char *kt = kb_ + kb * a.slot, *vt = vb_ + kb * a.slot;
#pragma unroll
            for (int i = 0; i < ST; i++) { ks[i] = *(const pv_u4 *)(kt + off[i]); vs[i] = *(const pv_u4 *)(vt + off[i]); }
            return;
        }
#pragma unroll
        for (int i = 0; i < ST; i++) {
            const int x = tid + 256 * i, j = kb + x / PER, e = x % PER * 8;
            const long long at = min(j, L.len - 1) * a.slot + (e < a.dim ? e * 2 : 0);
            ks[i] = *(const pv_u4 *)(kb_ + at);
            vs[i] = *(const pv_u4 *)(vb_ + at);
            if (e >= a.dim) ks[i] = (pv_u4){0, 0, 0, 0};
            if (j >= L.len || e >= a.dim) vs[i] = (pv_u4){0, 0, 0, 0};
        }
    };
    auto put = [&](int kb, int buf) {
#pragma unroll
        for (int i = 0; i < ST; i++) {
            const int x = tid + 256 * i, r = x / PER, e = x % PER * 8;
            if (kb + KEYS > L.n0) { // a new token's infinities and NaN stay out of the products
                unsigned any = 0;
#pragma unroll
                for (int y = 0; y < 4; y++) any |= odd_bits<E>(vs[i][y]);
                if (any && kb + r >= L.n0) {
                    odd = true;
#pragma unroll
                    for (int y = 0; y < 4; y++) vs[i][y] = without_odd<E>(vs[i][y]);
                }
            }
            *(pv_u4 *)(kl[buf] + r * KR + e) = ks[i];
            *(pv_u4 *)(vl[buf] + r * VR + e) = vs[i];
        }
    };
    if (k0 < kend) { fetch(k0); put(k0, 0); }
    __syncthreads();
    int cur = 0;
#pragma unroll 1
    for (int kb = k0; kb < kend; kb += KEYS, cur ^= 1) {
        const bool more = kb + KEYS < kend;
        if (more) fetch(kb + KEYS);
        f16v z[2];
#pragma unroll
        for (int i = 0; i < 16; i++) z[0][i] = z[1][i] = 0.f;
#pragma unroll
        for (int st = 0; st < KS; st++)
#pragma unroll
            for (int u = 0; u < 2; u++) z[u] = mfma32<E>(*(const pv_u4 *)(kl[cur] + (32 * u + c) * KR + 16 * st + 8 * h), qf[st], z[u]);
        // keys are loaded six products ahead, not two as the compiler has them (4 sequences of 1801 to 4001, trees of 24 tokens: 25.0 us, 26.2 without; a portion the same)
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (int i = 0; i < 2 * KS - 6; i++) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 6, 0);
        if (kb + KEYS > (a.tree ? L.n0 : L.n0 + first + 1)) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const unsigned bits = sees16(a, L, s, tok, kb + 32 * u + 4 * h - L.n0);
#pragma unroll
                for (int i = 0; i < 16; i++) z[u][i] = bits >> i & 1 ? z[u][i] : -INFINITY;
            }
        }
        float top = fmaxf(z[0][0], z[1][0]); // (of scores before the scale, which is above 0 here)
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(fmaxf(z[0][i], z[1][i]), top);
        top = against<E>(fmaxf(top, __shfl_xor(top, 32, 64)) * sc);
        if (__any(top > mx)) { // most blocks behind the first few raise no maximum
            const float mn = fmaxf(mx, top), ms = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(mx - ms);
            l *= al;
#pragma unroll
            for (int m = 0; m < MD; m++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[m][i] *= al;
            mx = mn;
        }
        const float ms = mx == -INFINITY ? 0.f : mx;
        pv_u4 pk[4], pl[4]; // the weights as two 16-bit numbers each
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(z[u][i], sc, -ms)), p1 = __builtin_amdgcn_exp2f(fmaf(z[u][i + 1], sc, -ms));
                sum += p0 + p1;
                const unsigned hi = round2<E>(p0, p1);
                const pv_f2 w = wide2<E>(hi);
                pk[2 * u + (i >> 3)][(i >> 1) & 3] = hi;
                pl[2 * u + (i >> 3)][(i >> 1) & 3] = round2<E>(p0 - w[0], p1 - w[1]);
            }
        l += sum;
        const unsigned short *base = vl[cur] + (4 * h + ((lane & 15) >> 2)) * VR + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        typedef __attribute__((address_space(3))) s4 lds_s4;
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int m = 0; m < MD; m++) {
                const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(base + 16 * k * VR + 32 * m)), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(base + (16 * k + 8) * VR + 32 * m));
                const pv_u2 xx = __builtin_bit_cast(pv_u2, x), yy = __builtin_bit_cast(pv_u2, y);
                const pv_u4 v = {xx[0], xx[1], yy[0], yy[1]};
                o[m] = mfma32<E>(v, pk[k], o[m]);
                o[m] = mfma32<E>(v, pl[k], o[m]);
            }
        if (more) put(kb + KEYS, cur ^ 1);
        __syncthreads();
    }
    odd = __syncthreads_or(odd);
    l += __shfl_xor(l, 32, 64);
    if (r0 + c >= rows) return;
    // the infinities and NaN of new tokens; and results that are NaN where an infinite value met a weight's second number, or a weight or a factor of 0, as in cache_attn_kernel
    unsigned long long nan = 0;
#pragma unroll
    for (int m = 0; m < MD; m++)
#pragma unroll
        for (int i = 0; i < 16; i++) nan |= (o[m][i] != o[m][i] ? 1ull : 0ull) << (16 * m + i);
    if (l != l) nan = 0;
    if (odd || nan) {
#pragma unroll
        for (int m = 0; m < MD; m++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[m][i] = nan >> (16 * m + i) & 1 ? 0.f : o[m][i];
#pragma unroll 1
        for (int x = 0; x < 16 * MD; x++) { // (one at a time: all together would not fit the registers)
            const int e = 32 * (x >> 4) + 8 * (x >> 2 & 3) + 4 * h + (x & 3);
            const bool all = nan >> x & 1;
            float more = 0.f;
            if (e < a.dim && (odd || all)) {
                auto value = [&](int j) { const float y = number<E>(vb_ + j * a.slot + e * 2); return odd32(y) ? y : 0.f; };
                if (all)
#pragma unroll 8
                    for (int j = k0; j < min(kend, L.n0); j++) more += value(j);
                for (int j = max(k0, L.n0); j < kend; j++)
                    if (sees(a, s, tok, j - L.n0)) more += value(j);
            }
#pragma unroll
            for (int m = 0; m < MD; m++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[m][i] += x == 16 * m + i ? more : 0.f;
        }
#pragma unroll
        for (int m = 0; m < MD; m++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[m][i] = (nan >> (16 * m + i) & 1) && o[m][i] == 0.f ? NAN : o[m][i];
    }
    const float ms = mx == -INFINITY ? 0.f : mx;
    if (a.parts > 1) {
        float *part = a.part + ((((long long)s * a.G + g) * a.tiles + row / 16) * a.parts + split) * (16 * (a.dim + 2));
        const int rr = row % 16;
#pragma unroll
        for (int m = 0; m < MD; m++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int e = 32 * m + 2 * i + 4 * h;
                if (e < a.dim) *(pv_f4 *)(part + rr * a.dim + e) = (pv_f4){o[m][i], o[m][i + 1], o[m][i + 2], o[m][i + 3]};
            }
        if (h == 0) { part[16 * a.dim + rr] = mx; part[16 * a.dim + 16 + rr] = l; }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    char *dst = a.out + s * a.o_seq + tok * a.o_row + (long long)(g * a.R + row - tok * a.R) * a.dim * 2;
#pragma unroll
    for (int m = 0; m < MD; m++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int e = 32 * m + 2 * i + 4 * h;
            if (e < a.dim) *(pv_u2 *)(dst + e * 2) = (pv_u2){round2<E>(o[m][i] * inv, o[m][i + 1] * inv), round2<E>(o[m][i + 2] * inv, o[m][i + 3] * inv)};
        }
    if (h == 0) a.lse[((long long)s * a.G + g) * a.T * a.R + row] = l == 0.f ? INFINITY : ms + log2f(l);
}

// which of 16 rows, row + 8 (i / 4) + i % 4, see new token x of a tree (below 0: a held slot, which all see), a bit each; rows behind the last repeat it
__device__ __forceinline__ unsigned seen_by16(const ca_args &a, const ca_lens &L, int s, int row, int rows, int x) {
    const uint8_t *see = a.tree + (long long)s * a.T * a.T + min(max(x, 0), L.cnt - 1);
    uint8_t v[16];
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = see[(long long)token_of(a, min(row + 8 * (i >> 2) + (i & 3), rows - 1)) * a.T];
    unsigned bits = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) bits |= (x < 0 || (x < L.cnt && v[i]) ? 1u : 0u) << i;
    return bits;
}
// The weights that slots receive from many rows of a 16-bit cache: 256 keys of a kv head (a wave 64 of them, in registers) against the rows that see any, 64 at a time through LDS.  S = Q K^T here: a
// lane has a key, so that the sum over rows is its registers' and its other half's (S^T: 32 sums a lane and 160 moves between lanes, 8 us of 24 of a small step); the sums of the work-groups that share a block are
// left side by side.  What bounds it: 96 vector instructions, 32 of them 2^x, beside 16 matrix instructions.
template <class E, int DP>
__global__ __launch_bounds__(256, 2) void cache_receive_kernel(const ca_args a) {
    constexpr int KS = DP / 16, QR = DP + 8, PER = DP / 8, ST = QT * PER / 256;
    __shared__ __attribute__((aligned(16))) unsigned short ql[2][QT * QR];
    __shared__ __attribute__((aligned(16))) float lsl[2][QT];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c = lane & 31, h = lane >> 5;
    int id = blockIdx.x;
    const int heads = a.n_seqs * a.G, hs = id % heads, s = hs / a.G, g = hs - s * a.G; id /= heads; // (neighbours: kv heads, as above)
    const ca_lens L = lens_of(a, s);
    const int rows = L.cnt * a.R;
    const received<256> work(a, L);
    int b, t0, t1;
    long long at = 0, end = 0, first = 0; // the tiles that are left, and the block's first
    if (a.wgroups) {
        if (id >= work.groups) return;
        at = work.start(id);
        end = work.start(id + 1);
        b = work.block_of(at, first);
    } else {
        b = id;
        if (b * 256 >= L.len) return;
    }
    const float *lse = a.lse + ((long long)s * a.G + g) * a.T * a.R;
    const char *qh = a.q + s * a.q_seq + (long long)g * a.R * a.dim * 2;
    pv_u4 qs[ST];
    float ls = 0.f;
    auto fetch = [&](int tile) {
#pragma unroll
        for (int i = 0; i < ST; i++) {
            const int x = tid + 256 * i, row = min(tile * QT + x / PER, rows - 1), tok = token_of(a, row), e = x % PER * 8;
            if (a.near) qs[i] = *(const pv_u4 *)(qh + (unsigned)(tok * (int)a.q_row + (row - tok * a.R) * a.dim * 2 + (e < a.dim ? e * 2 : 0)));
            else qs[i] = *(const pv_u4 *)(qh + tok * a.q_row + ((long long)(row - tok * a.R) * a.dim * 2 + (e < a.dim ? e * 2 : 0)));
            if (e >= a.dim) qs[i] = (pv_u4){0, 0, 0, 0};
        }
        if (tid < QT) ls = tile * QT + tid < rows ? lse[tile * QT + tid] : INFINITY;
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int i = 0; i < ST; i++) { const int x = tid + 256 * i; *(pv_u4 *)(ql[buf] + x / PER * QR + x % PER * 8) = qs[i]; }
        if (tid < QT) lsl[buf][tid] = ls;
    };
#pragma unroll 1
    do {
    t0 = work.from(b);
    t1 = work.tiles;
    if (a.wgroups) {
        const int skip = t0;
        t0 = skip + (int)(at - first);
        t1 = (int)min((long long)t1, skip + (end - first));
        at = first = first + work.tiles - skip;
    }
    const int kb = b * 256 + wave * 64;
    pv_u4 kf[2][KS];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const char *k = a.k + s * a.seq + g * a.head + min(kb + 32 * u + c, L.len - 1) * a.slot;
#pragma unroll
        for (int st = 0; st < KS; st++) {
            const int e = 16 * st + 8 * h;
            kf[u][st] = *(const pv_u4 *)(k + (e < a.dim ? e * 2 : 0));
            if (e >= a.dim) kf[u][st] = (pv_u4){0, 0, 0, 0};
        }
    }
    float w[2][2] = {};
    if (t0 < t1) { fetch(t0); put(0); }
    __syncthreads();
    int cur = 0;
#pragma unroll 1
    for (int tile = t0; tile < t1; tile++, cur ^= 1) {
        if (tile + 1 < t1) fetch(tile + 1);
#pragma unroll 1
        for (int sub = 0; sub < QT / 32; sub++) {
            const int r0 = tile * QT + 32 * sub;
            if (kb - L.n0 > (a.tree ? L.cnt : token_of(a, min(r0 + 31, rows - 1)))) continue; // these tokens all come before the wave's keys
            f16v z[2];
#pragma unroll
            for (int i = 0; i < 16; i++) z[0][i] = z[1][i] = 0.f;
#pragma unroll
            for (int st = 0; st < KS; st++) {
                const pv_u4 q = *(const pv_u4 *)(ql[cur] + (32 * sub + c) * QR + 16 * st + 8 * h);
                z[0] = mfma32<E>(q, kf[0][st], z[0]);
                z[1] = mfma32<E>(q, kf[1][st], z[1]);
            }
            pv_f4 lr[4]; // of rows r0 + 8 (i / 4) + 4 h + i % 4
#pragma unroll
            for (int x = 0; x < 4; x++) lr[x] = *(const pv_f4 *)(lsl[cur] + 32 * sub + 8 * x + 4 * h);
            if (kb + 64 <= (a.tree ? L.n0 : L.n0 + token_of(a, r0) + 1)) { // all see all
#pragma unroll
                for (int i = 0; i < 16; i++)
#pragma unroll
                    for (int u = 0; u < 2; u++) w[u][i & 1] += __builtin_amdgcn_exp2f(fmaf(z[u][i], a.sc2, -lr[i >> 2][i & 3]));
            } else if (!a.tree) { // row r sees new token x where r >= x R
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int behind = min(max(kb + 32 * u + c - L.n0, 0), L.cnt) * a.R - r0 - 4 * h;
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(z[u][i], a.sc2, -lr[i >> 2][i & 3]));
                        w[u][i & 1] += 8 * (i >> 2) + (i & 3) >= behind ? p : 0.f;
                    }
                }
            } else if (kb < L.len) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int x = kb + 32 * u + c - L.n0; // the lane's key among the new ones
                    const unsigned bits = seen_by16(a, L, s, r0 + 4 * h, rows, x);
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float ls = lr[i >> 2][i & 3], p = __builtin_amdgcn_exp2f(fmaf(z[u][i], a.sc2, -ls));
                        w[u][i & 1] += ls != INFINITY && (bits >> i & 1) ? p : 0.f;
                    }
                }
            }
        }
        if (tile + 1 < t1) put(cur ^ 1);
        __syncthreads();
    }
    float v[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        v[u] = w[u][0] + w[u][1];
        v[u] += __shfl_xor(v[u], 32, 64);
    }
    const int j = kb + lane;
    const float sum = h ? v[1] : v[0];
    if (a.wgroups) a.wpart[(hs * (a.wgroups + (a.n_ctx + 255ll) / 256) + id + b) * 256 + wave * 64 + lane] = sum;
    else if (j < L.len) {
        const long long to = (long long)hs * a.n_ctx + j;
        a.weight_out[to] = j < L.n0 && a.weight ? a.weight[to] + sum : sum;
    }
    b++;
    } while (at < end);
}
template <int B>
__global__ __launch_bounds__(256) void cache_gather_kernel(const ca_args a) { // the sums of a block's work-groups, in order
    const int j = blockIdx.x * 256 + threadIdx.x, b = j / B, g = blockIdx.y, s = blockIdx.z;
    const ca_lens L = lens_of(a, s);
    if (j >= L.len) return;
    const long long head = (long long)s * a.G + g, at = head * a.n_ctx + j;
    const received<B> work(a, L);
    float v = 0.f;
    if (work.n) {
        long long first = (long long)min(b, work.held) * work.tiles;
        for (int x = work.held; x < b; x++) first += work.tiles - work.from(x);
        const int w0 = work.group_of(first), w1 = work.group_of(first + work.tiles - work.from(b) - 1);
#pragma unroll 8
        for (int w = w0; w <= w1; w++) v += a.wpart[(head * (a.wgroups + (a.n_ctx + B - 1ll) / B) + w + b) * B + j % B];
    }
    a.weight_out[at] = j < L.n0 && a.weight ? a.weight[at] + v : v;
}

// an accepted path: a work-group per kv head and sequence, token after token (a row moves down, or stays)
__global__ __launch_bounds__(256) void cache_take_kernel(char *k, char *v, long long seq, long long slot, long long head, int n_ctx, int row_bytes, const int32_t *n_kv, const int32_t *count, const int32_t *take,
                                                         int n_take, int32_t *pos, float *weight) {
    const int g = blockIdx.x, s = blockIdx.y, n0 = min(max(n_kv[s], 0), n_ctx), cnt = min(max(count[s], 0), min(n_take, n_ctx - n0));
    char *kr = k + s * seq + g * head, *vr = v + s * seq + g * head;
    const long long at = ((long long)s * gridDim.x + g) * n_ctx;
    int last = -1;
    for (int i = 0; i < cnt; i++) {
        const int t = take[(long long)s * n_take + i];
        if (t <= last || t >= n_ctx - n0) return;
        last = t;
        if (t == i) continue;
        const int from = n0 + t, to = n0 + i; // to < from: no later row reads `to`
        for (int x = threadIdx.x * 16; x < 2 * row_bytes; x += 4096) {
            char *r = x < row_bytes ? kr + x : vr + (x - row_bytes);
            *(pv_u4 *)(r + to * slot) = *(const pv_u4 *)(r + from * slot);
        }
        if (threadIdx.x == 0) {
            if (pos) pos[at + to] = pos[at + from];
            if (weight) weight[at + to] = weight[at + from];
        }
    }
}
__global__ __launch_bounds__(256) void cache_count_kernel(int32_t *n_kv, const int32_t *count, const int32_t *take, int n_take, int n_seqs, int n_ctx) {
    const int s = blockIdx.x * 256 + threadIdx.x;
    if (s >= n_seqs) return;
    const int n0 = min(max(n_kv[s], 0), n_ctx);
    int cnt = min(max(count[s], 0), n_ctx - n0);
    if (take) {
        cnt = min(cnt, n_take);
        int last = -1, i = 0;
        for (; i < cnt; i++) {
            const int t = take[(long long)s * n_take + i];
            if (t <= last || t >= n_ctx - n0) break;
            last = t;
        }
        cnt = i;
    }
    n_kv[s] = n0 + cnt;
}

template <class E, int DP>
void launch_attn(ca_args a, bool many, hipStream_t st) {
    const long long heads = (long long)a.n_seqs * a.G;
    if (a.tiles > 2 && a.k_new) { // more than 32 rows: the new rows go into the cache first, and everything is read from there
        const int row_bytes = a.dim * E::SIZE, pieces = a.T * a.G * (row_bytes / 16);
        hipLaunchKernelGGL(cache_append_kernel, dim3((unsigned)((pieces + 255) / 256), (unsigned)a.n_seqs), dim3(256), 0, st, a, row_bytes);
        a.k_new = a.v_new = nullptr;
    }
    if constexpr (E::SIZE == 2) {
        if (many) {
            const long long blocks = (a.T * a.R + ROWS - 1) / ROWS;
            hipLaunchKernelGGL((cache_rows_kernel<E, DP>), dim3((unsigned)(a.share ? a.share + heads * blocks : heads * a.parts * blocks)), dim3(256), 0, st, a);
            if (a.parts > 1) hipLaunchKernelGGL((cache_join_kernel<E>), dim3((unsigned)(heads * a.tiles)), dim3(256), 0, st, a, (unsigned)(heads * a.tiles));
            if (!a.weight_out) return;
            hipLaunchKernelGGL((cache_receive_kernel<E, DP>), dim3((unsigned)(heads * (a.wgroups ? a.wgroups : (a.n_ctx + 255) / 256))), dim3(256), 0, st, a);
            if (a.wgroups) hipLaunchKernelGGL((cache_gather_kernel<256>), dim3((unsigned)((a.n_ctx + 255) / 256), (unsigned)a.G, (unsigned)a.n_seqs), dim3(256), 0, st, a);
            return;
        }
    }
    // two tiles of rows a wave where there are two: its keys are read once for both
    const unsigned grid = (unsigned)(a.share ? a.share + heads * ((a.tiles + 1) / 2) : heads * a.parts * ((a.tiles + 1) / 2)); // (shared out: a sequence's last part may be a short one)
    if (a.tiles > 1) hipLaunchKernelGGL((cache_attn_kernel<E, DP, 2>), dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((cache_attn_kernel<E, DP, 1>), dim3(grid), dim3(256), 0, st, a);
    const unsigned joins = a.parts > 1 ? (unsigned)(heads * a.tiles) : 0, scores = a.weight_out && a.tiles <= 2 ? (unsigned)(heads * a.scorers) : 0;
    if (joins + scores) hipLaunchKernelGGL((cache_join_kernel<E>), dim3(joins + scores), dim3(256), 0, st, a, joins);
    if (!a.weight_out || a.tiles <= 2) return;
    if constexpr (E::SIZE == 4) {
        hipLaunchKernelGGL((cache_weight_kernel<E, DP>), dim3((unsigned)(heads * (a.wgroups ? a.wgroups : (a.n_ctx + 63) / 64))), dim3(256), 0, st, a);
        if (a.wgroups) hipLaunchKernelGGL((cache_gather_kernel<64>), dim3((unsigned)((a.n_ctx + 255) / 256), (unsigned)a.G, (unsigned)a.n_seqs), dim3(256), 0, st, a);
    }
}
// work-groups of 256 threads that parts may make of a launch, whose grid has fewer than 2^32 threads
constexpr long long MOST_PARTS = 64000 * 256;
} // namespace

// The most that any call of up to n_seqs sequences and n_new tokens takes, piece by piece: fewer rows have more parts, and up to 32 rows scores.
size_t psv_attn_most(int n_cu, const ps_kv_cache &c, const ps_cache_attn_params &p) {
    const long long R = p.heads / c.kv_heads, size = c.dtype == PS_F32 ? 4 : 2, T = p.n_new, few = size == 4 ? T : std::min(T, 32 / R), cap = std::min(64, (c.n_ctx + 127) / 128);
    // work-groups times parts, of up to g work-groups that `fill` of them fill the chip, each in `x` parts at least; one part needs no place
    auto in_parts = [&](long long g, long long fill, long long x) {
        if (x == 1) g = std::min(g, fill - 1);
        return cap == 1 ? 0 : std::min({std::max(fill + g - 1, x * g), cap * g, MOST_PARTS});
    };
    auto bytes = [&](long long n_seqs, bool chunks) {
        const long long heads = n_seqs * c.kv_heads;
        long long part = 0;
        if (few) {
            const long long tiles = (few * R + 15) / 16;
            part = (tiles > 1 ? 2 : 1) * in_parts(heads * ((tiles + 1) / 2), 3 * n_cu, (c.n_ctx + 511) / 512);
        }
        if (T > few) {
            part = std::max(part, std::min<long long>(ROWS / 16, (T * R + 15) / 16) * in_parts(heads, n_cu, n_seqs > 1 ? (c.n_ctx + 1023) / 1024 : 1));
            part = std::max(part, ROWS / 16 * in_parts(heads * ((T * R + ROWS - 1) / ROWS), n_cu, 1));
        }
        ps_carve ws{nullptr};
        ws.take<float>((size_t)(heads * T * R));
        ws.take<float>((size_t)(part * 16 * (c.dim + 2)));
        if (chunks) ws.take<int>((size_t)n_seqs);
        if (!p.weight_out) return ws.at;
        ws.take<float>((size_t)(heads * c.n_ctx * ((std::min(T, 32 / R) * R + 3) / 4 * 4)));
        if (T * R > 32) {
            const long long block = size == 2 ? 256 : 64, blocks = (c.n_ctx + block - 1) / block, shared = T * R > 4 * QT ? heads : std::min(heads, (2 * n_cu - 1) / blocks);
            if (shared) ws.take<float>((size_t)((2 * n_cu + shared - 1 + shared * blocks) * block));
        }
        return ws.at;
    };
    return std::max(bytes(c.n_seqs, false), c.n_seqs > 1 && cap > 1 ? bytes(std::min(c.n_seqs, 256), true) : 0);
}
size_t psv_attn_space(int n_cu, const ps_kv_cache &c, const ps_cache_attn_params &p, void *base, bool launch, hipStream_t st) {
    const int R = p.heads / c.kv_heads, size = c.dtype == PS_F32 ? 4 : 2;
    const long long heads = (long long)c.n_seqs * c.kv_heads, rows = (long long)p.n_new * R;
    ca_args a{};
    a.tiles = (int)((rows + 15) / 16);
    // more than 32 rows of a 16-bit cache: 128 rows a work-group (one side and the other, bf16, 32 heads of 8, dim 128, with weights: 4 sequences of 1801 to 4001, 20 rows 42 and 40 us, 32 rows 36 and 40; 32 sequences
    // of up to 8100, 20 rows 76 and 95, 32 rows 91 and 96; without: 40 and 30, 32 and 31; 63 and 58, 65 and 59)
    const bool many = size == 2 && rows > 32;
    const long long groups = heads * (many ? (rows + ROWS - 1) / ROWS : (a.tiles + 1) / 2);
    // parts of the keys: until the chip is full (few rows: three times, or 512 keys each); 1024 keys each where several sequences have one work-group's rows, so that the longest does not keep the others
    // waiting (32 sequences of up to 8100, 48 rows: 230 us in one part each, 110 so)
    a.parts = (int)std::min<long long>({std::max<long long>(((many ? 1 : 3) * n_cu + groups - 1) / groups, !many ? (c.n_ctx + 511) / 512 : rows <= ROWS && c.n_seqs > 1 ? (c.n_ctx + 1023) / 1024 : 1), (c.n_ctx + 127) / 128, 64, std::max(1ll, MOST_PARTS / groups)});
    a.near = p.q_row_stride >= 0 && p.q_row_stride < (1 << 28) && (p.n_new + 1ll) * (p.q_row_stride + (long long)R * c.dim) < (1 << 29);
    a.plain = c.slot_stride >= 0 && c.slot_stride < (1 << 24);
    ps_carve ws{(char *)base};
    a.lse = ws.take<float>((size_t)(heads * rows));
    if (a.parts > 1) a.part = ws.take<float>((size_t)(heads * a.tiles * a.parts * 16 * (c.dim + 2)));
    a.score_rows = (int)((rows + 3) / 4 * 4);
    if (a.parts > 1 && c.n_seqs > 1 && c.n_seqs <= 256) {
        a.share = (many ? 2 : 4) * n_cu;
        a.chunks = ws.take<int>(c.n_seqs);
    }
    a.scorers = (int)std::max<long long>(1, std::min<long long>((c.n_ctx + 255) / 256, 8 * n_cu / heads));
    if (p.weight_out && a.tiles <= 2) a.score = ws.take<float>((size_t)(heads * c.n_ctx * a.score_rows));
    if (a.tiles > 2 && p.weight_out) { // up to 256 rows of slots enough to fill the chip: a block's rows are few; else the blocks' rows, which a sequence's length and the causal mask make unequal, are shared out
        const long long block = many ? 256 : 64, blocks = (c.n_ctx + block - 1) / block;
        if (rows > 4 * QT || heads * blocks < 2 * n_cu) {
            a.wgroups = (int)((2 * n_cu + heads - 1) / heads); // (two a CU: half as many, 2048 tokens behind 2047: 87 -> 129 us; twice as many in fp32, 1024 behind 1000: 53 -> 65)
            a.wpart = ws.take<float>((size_t)(heads * (a.wgroups + blocks) * block));
        }
    }
    if (!launch) return ws.at;
    a.k = (char *)c.k; a.v = (char *)c.v; a.out = (char *)p.out; a.q = (const char *)p.q; a.k_new = (const char *)p.k_new; a.v_new = (const char *)p.v_new;
    a.seq = c.seq_stride * size; a.slot = c.slot_stride * size; a.head = c.head_stride * size;
    a.q_seq = p.q_seq_stride * size; a.q_row = p.q_row_stride * size; a.o_seq = p.out_seq_stride * size; a.o_row = p.out_row_stride * size;
    a.new_seq = p.new_seq_stride * size; a.new_row = p.new_row_stride * size;
    a.n_seqs = c.n_seqs; a.n_ctx = c.n_ctx; a.G = c.kv_heads; a.dim = c.dim; a.R = R; a.T = p.n_new;
    a.by_R = R == 1 ? 0 : (unsigned)((((unsigned long long)1 << 32) + R - 1) / R);
    a.sc2 = p.scale == 0.f ? 1e-37f : size == 4 ? p.scale : p.scale * 1.44269504088896340736f; // (never 0: a masked score is minus infinity times it)
    a.n_kv = c.n_kv; a.count = p.count; a.pos_new = p.pos_new; a.pos = c.pos; a.tree = p.tree; a.weight = c.weight; a.weight_out = p.weight_out;
    if (c.dtype == PS_F32) c.dim > 64 ? launch_attn<F32, 128>(a, many, st) : launch_attn<F32, 64>(a, many, st);
    else if (c.dtype == PS_F16) c.dim > 64 ? launch_attn<F16, 128>(a, many, st) : launch_attn<F16, 64>(a, many, st);
    else c.dim > 64 ? launch_attn<BF16, 128>(a, many, st) : launch_attn<BF16, 64>(a, many, st);
    return ws.at;
}

void psv_advance(hipStream_t st, const ps_kv_cache &c, const int32_t *count, const int32_t *take, int n_take) {
    const int size = c.dtype == PS_F32 ? 4 : 2;
    if (take)
        hipLaunchKernelGGL(cache_take_kernel, dim3((unsigned)c.kv_heads, (unsigned)c.n_seqs), dim3(256), 0, st, (char *)c.k, (char *)c.v, c.seq_stride * size, c.slot_stride * size, c.head_stride * size, c.n_ctx,
                           c.dim * size, c.n_kv, count, take, n_take, c.pos, c.weight);
    hipLaunchKernelGGL(cache_count_kernel, dim3((unsigned)((c.n_seqs + 255) / 256)), dim3(256), 0, st, c.n_kv, count, take, n_take, c.n_seqs, c.n_ctx);
}
