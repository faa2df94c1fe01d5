// Low-rank adapters of many requests beside a shared projection (ps_hip_adapters_apply): out[t] = base[t] + scale_a up_a (down_a x[t]), a = ids[t].
//   The tokens of one adapter are taken 16 at a time (a tile), wherever they stand in the batch, so that its matrices are read once for all of them and the products run on
//   v_mfma_f32_16x16x32_bf16.
//   adapt_plan_kernel  the tokens sorted by adapter and the tiles, for large batches; in small ones every work-group finds its tile from the ids itself
//   adapt_down_kernel  h = down x: a tile against a part of K, four waves a quarter each; the parts' sums are left side by side
//   adapt_up_kernel    the parts' sums together, then 64 columns a wave of base + scale up h
// A factor that is not bfloat16 -- x in fp32, h -- goes in as three bfloat16 numbers that add up to it, 24 bits together: every product is exact and every sum fp32.  Both matrices
// together are read once per tile and step; what bounds a decode step is that read, a prompt the pass over base and out.
// Measured: 253 tokens of 64 adapters of rank 64, 4096 to 14336, bf16: plan 6, down 10 us (34 MB), up 28 us for 146 MB, 5.2 TB/s (a large copy: 5.0); 2048 tokens of four, rank 16, 4096 to 4096: plan 5, down 9 us,
// up 18 us for 67 MB, 3.7 TB/s; 4 tokens: 5 + 5 us, latency.
#include "ps_serve.h"

#include <algorithm>

namespace {
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
constexpr int TILE = 16;
// Without a plan a launch is saved, and there are work-groups for every token, most of which find that their tile begins elsewhere: up to 256 tokens (a thread each) and 2^19 results.  K 2048, rank 16, a quarter as
// many adapters as tokens, without and with: 16 x 14336 11.1 and 13.6 us, 64 x 4096 11.4 and 14.1, 32 x 14336 14.6 and 14.2, 128 x 4096 14.4 and 15.4, 253 x 2048 15.1 and 16.3, 64 x 14336 23.0 and 16.6.
inline bool plans_itself(int64_t T, int64_t N) { return T <= 256 && T * N <= 1 << 19; }
struct ad_args {
    const uint16_t *down, *up;
    const int32_t *rank, *ids;
    const float *scale;
    const char *x;
    const float *base;
    float *out;
    long long N, K, KP, RP, ldx, ldo;
    int n_slots, T, parts, vec, columns; // columns of a work-group of the second product
    int32_t *order, *tiles; // the plan: tokens by adapter; [0] tiles, then (adapter, first, tokens) each
    float *h;               // [part][tile][RP][16]
};
__device__ __forceinline__ pv_f4 mfma(const pv_u4 &x, const pv_u4 &y, const pv_f4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
}
__device__ __forceinline__ unsigned round2(float a, float b) { return __builtin_bit_cast(unsigned, __builtin_convertvector((pv_f2){a, b}, b2)); }
// a number as three: rounded, the rounded rest, the rest of that; one that rounds to infinity is cut off instead, infinity and NaN have no rest
__device__ __forceinline__ void split2(float a, float b, unsigned &u1, unsigned &u2, unsigned &u3) {
    u1 = round2(a, b);
    float a1 = __uint_as_float(u1 << 16), b1 = __uint_as_float(u1 & 0xffff0000u);
    if (__builtin_isinf(a1)) { u1 = (u1 & 0xffff0000u) | (__float_as_uint(a) >> 16); a1 = __uint_as_float(u1 << 16); }
    if (__builtin_isinf(b1)) { u1 = (u1 & 0xffffu) | (__float_as_uint(b) & 0xffff0000u); b1 = __uint_as_float(u1 & 0xffff0000u); }
    float ra = a - a1, rb = b - b1;
    if (__builtin_isinf(a1)) ra = 0.f;
    if (__builtin_isinf(b1)) rb = 0.f;
    u2 = round2(ra, rb);
    u3 = round2(ra - __uint_as_float(u2 << 16), rb - __uint_as_float(u2 & 0xffff0000u));
}
__device__ __forceinline__ int adapter_of(const ad_args &a, int t) { // -1: none
    const int i = a.ids[t];
    return i >= 0 && i < a.n_slots && a.rank[i] > 0 ? i : -1;
}
// The work-group's tile: its adapter (-2: no such tile), its tokens in tok[16].  Without a plan tile b belongs to token b where that is the first, 17th, 33rd .. of its adapter (a thread a
// token).
__device__ __forceinline__ int tile_of(const ad_args &a, int b, int *tok, int *n, int *sh) {
    const int tid = threadIdx.x;
    if (a.order) {
        if (b >= a.tiles[0]) return -2;
        const int32_t *t = a.tiles + 1 + 3 * b;
        *n = t[2];
        if (tid < TILE) tok[tid] = a.order[t[1] + min(tid, t[2] - 1)];
        __syncthreads();
        return t[0];
    }
    if (b >= a.T) return -2;
    const int me = adapter_of(a, b), lane = tid & 63, wave = tid >> 6;
    const bool same = tid < a.T && adapter_of(a, tid) == me;
    const unsigned long long m = __ballot(same);
    if (lane == 0) sh[wave] = __popcll(m);
    __syncthreads();
    int at = __popcll(m & ((1ull << lane) - 1)), all = 0;
    for (int w = 0; w < 4; w++) { if (w < wave) at += sh[w]; all += sh[w]; }
    if (tid == b) sh[4] = at; // of those before token b
    __syncthreads();
    const int first = sh[4];
    if (first % TILE) return -2;
    *n = min(TILE, all - first);
    if (same && at >= first && at < first + TILE) tok[at - first] = tid;
    __syncthreads();
    if (tid < TILE && tid >= *n) tok[tid] = b;
    __syncthreads();
    return me;
}

// the tokens by adapter: slot n_slots stands for none.  count [n_slots + 1]: LDS where it has room, else global scratch.  Lanes of a wave that have the same adapter count as one: in a prompt they
// all have (2048 tokens of 4 adapters: 69 us with an atomic a token).
constexpr int PLAN_LDS = 8192;
// The lanes of a wave that count for adapter i: those of the first two adapters found there together, the others each for itself.  f(adapter, lanes, whether this lane adds for them)
template <class F> __device__ __forceinline__ void by_adapter(int i, bool there, F f) {
    const int lane = threadIdx.x & 63;
    unsigned long long todo = __ballot(there);
#pragma unroll 1
    for (int k = 0; k < 2 && todo; k++) {
        const int one = __builtin_amdgcn_readlane(i, __ffsll(todo) - 1);
        const unsigned long long same = __ballot(there && i == one) & todo;
        if (same >> lane & 1) f(one, same);
        todo &= ~same;
    }
    if (todo >> lane & 1) f(i, 1ull << lane);
}
__global__ __launch_bounds__(1024) void adapt_plan_kernel(const ad_args a, int32_t *spare) {
    extern __shared__ int32_t in_lds[];
    __shared__ int sc[16], st[16], run[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = a.n_slots + 1;
    const bool lds = bins <= PLAN_LDS;
    auto add = [&](int i, int n) { return lds ? atomicAdd(&in_lds[i], n) : atomicAdd(&spare[i], n); };
    auto get = [&](int i) { return lds ? in_lds[i] : __hip_atomic_load(&spare[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto set = [&](int i, int v) { if (lds) in_lds[i] = v; else __hip_atomic_store(&spare[i], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    for (int i = tid; i < bins; i += 1024) set(i, 0);
    if (tid < 2) run[tid] = 0;
    __syncthreads();
    auto slot = [&](int t) { const int i = t < a.T ? adapter_of(a, t) : 0; return i < 0 ? a.n_slots : i; };
    for (int t = tid; t - lane < a.T; t += 1024) by_adapter(slot(t), t < a.T, [&](int i, unsigned long long same) { if (lane == __ffsll(same) - 1) add(i, (int)__popcll(same)); });
    __syncthreads();
    for (int base = 0; base < bins; base += 1024) {
        const int i = base + tid, c = i < bins ? get(i) : 0, nt = (c + TILE - 1) / TILE;
        int x = c, y = nt;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(x, o, 64), v = __shfl_up(y, o, 64);
            if (lane >= o) { x += u; y += v; }
        }
        if (lane == 63) { sc[wave] = x; st[wave] = y; }
        __syncthreads();
        int before_c = run[0], before_t = run[1], all_c = 0, all_t = 0;
        for (int w = 0; w < 16; w++) {
            if (w < wave) { before_c += sc[w]; before_t += st[w]; }
            all_c += sc[w];
            all_t += st[w];
        }
        const int first = before_c + x - c, tile = before_t + y - nt;
        if (i < bins) {
            set(i, first);
            for (int k = 0; k < nt; k++) {
                int32_t *t = a.tiles + 1 + 3 * (tile + k);
                t[0] = i == a.n_slots ? -1 : i;
                t[1] = first + k * TILE;
                t[2] = min(TILE, c - k * TILE);
            }
        }
        __syncthreads();
        if (tid == 0) { run[0] += all_c; run[1] += all_t; }
        __syncthreads();
    }
    if (tid == 0) a.tiles[0] = run[1];
    for (int t = tid; t - lane < a.T; t += 1024) // (the order of an adapter's tokens is nobody's business: a token's result does not depend on its tile)
        by_adapter(slot(t), t < a.T, [&](int i, unsigned long long same) {
            const int leader = __ffsll(same) - 1;
            int at = lane == leader ? add(i, (int)__popcll(same)) : 0;
            at = __shfl(at, leader, 64);
            a.order[at + (int)__popcll(same & ((1ull << lane) - 1))] = t;
        });
}

template <bool F32X>
__global__ __launch_bounds__(256) void adapt_down_kernel(const ad_args a) {
    __shared__ int tok[TILE], sh[8];
    __shared__ float red[4][64][17];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c = lane & 15, q4 = lane >> 4, b = blockIdx.x;
    int n;
    const int ad = tile_of(a, b, tok, &n, sh);
    if (ad < 0) return;
    const int rank = a.rank[ad], rt = (rank + 15) / 16;
    const long long steps = a.KP / 32, per = (steps + a.parts - 1) / a.parts, s0 = blockIdx.y * per, s1 = min(steps, s0 + per);
    const uint16_t *down = a.down + (long long)ad * a.RP * a.KP;
    const char *x = a.x + tok[c] * a.ldx * (F32X ? 4 : 2);
    for (int r0 = 0; r0 < rt; r0 += 4) { // up to 64 ranks at a time
        const int m = min(4, rt - r0);
        pv_f4 h[4];
#pragma unroll
        for (int r = 0; r < 4; r++) h[r] = (pv_f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
        for (long long s = s0 + wave; s < s1; s += 4) {
            const long long k = 32 * s + 8 * q4;
            pv_u4 p1, p2, p3;
            if constexpr (F32X) {
                float v[8];
                if ((a.vec & 1) && k + 8 <= a.K) {
                    const pv_f4 u = *(const pv_f4 *)(x + k * 4), w = *(const pv_f4 *)(x + k * 4 + 16);
#pragma unroll
                    for (int e = 0; e < 4; e++) { v[e] = u[e]; v[4 + e] = w[e]; }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = k + e < a.K ? ((const float *)x)[k + e] : 0.f;
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    unsigned u1, u2, u3;
                    split2(v[2 * e], v[2 * e + 1], u1, u2, u3);
                    p1[e] = u1; p2[e] = u2; p3[e] = u3;
                }
            } else {
                if ((a.vec & 1) && k + 8 <= a.K) p1 = *(const pv_u4 *)(x + k * 2);
                else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        p1[e] = (k + 2 * e < a.K ? ((const uint16_t *)x)[k + 2 * e] : 0u) | (k + 2 * e + 1 < a.K ? (unsigned)((const uint16_t *)x)[k + 2 * e + 1] << 16 : 0u);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (r >= m) continue;
                const pv_u4 d = *(const pv_u4 *)(down + ((r0 + r) * 16 + c) * a.KP + k);
                if constexpr (F32X) {
                    h[r] = mfma(d, p3, h[r]);
                    h[r] = mfma(d, p2, h[r]);
                }
                h[r] = mfma(d, p1, h[r]);
            }
        }
        if (r0) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int i = 0; i < 4; i++) red[wave][16 * r + 4 * q4 + i][c] = h[r][i];
        __syncthreads();
        float *o = a.h + (((long long)blockIdx.y * gridDim.x + b) * a.RP + r0 * 16) * TILE;
        for (int i = tid; i < m * 256; i += 256) o[i] = (red[0][i >> 4][i & 15] + red[1][i >> 4][i & 15]) + (red[2][i >> 4][i & 15] + red[3][i >> 4][i & 15]);
    }
}

__global__ __launch_bounds__(256) void adapt_up_kernel(const ad_args a) {
    __shared__ int tok[TILE], sh[8];
    extern __shared__ __attribute__((aligned(16))) uint16_t hl[]; // [16 tokens][3 rank16 + 8]: h as three numbers
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c = lane & 15, q4 = lane >> 4, b = blockIdx.x;
    int n;
    const int ad = tile_of(a, b, tok, &n, sh);
    if (ad == -2) return;
    float scale = 0.f;
    int r16 = 0, ld = 0;
    if (ad >= 0) {
        const int rank = a.rank[ad];
        r16 = (rank + 15) / 16 * 16;
        ld = 3 * r16 + 8;
        scale = a.scale[ad];
        for (int i = tid; i < r16 * 8; i += 256) { // two ranks of a token
            const int t = i & 15, r = (i >> 4) * 2;
            float v[2] = {0.f, 0.f};
#pragma unroll 4
            for (int p = 0; p < a.parts; p++) {
                const float *h = a.h + (((long long)p * gridDim.x + b) * a.RP + r) * TILE + t;
                v[0] += h[0];
                v[1] += h[TILE];
            }
            if (r >= rank) v[0] = 0.f; // (0 times an infinite x behind the last rank)
            if (r + 1 >= rank) v[1] = 0.f;
            unsigned u1, u2, u3;
            split2(v[0], v[1], u1, u2, u3);
            *(unsigned *)(hl + t * ld + r) = u1;
            *(unsigned *)(hl + t * ld + r16 + r) = u2;
            *(unsigned *)(hl + t * ld + 2 * r16 + r) = u3;
        }
        __syncthreads();
    }
    const uint16_t *up = a.up + (long long)max(ad, 0) * a.N * a.RP;
    const long long end = min(a.N, (long long)(blockIdx.y + 1) * a.columns);
    for (long long n0 = (long long)blockIdx.y * a.columns + wave * 64; n0 < end; n0 += 256) {
        const long long col = n0 + 4 * c;
        pv_f4 o[4], v[4];
        // base is on its way while the products are made
#pragma unroll
        for (int i = 0; i < 4; i++) {
            o[i] = v[i] = (pv_f4){0.f, 0.f, 0.f, 0.f};
            const int t = 4 * q4 + i;
            if ((a.vec & 2) && a.base && t < n && col < a.N) v[i] = *(const pv_f4 *)(a.base + tok[t] * a.ldo + col);
        }
        for (int r0 = 0; r0 < r16; r0 += 32) {
            const int r = r0 + 8 * q4;
            const bool there = r < r16;
            pv_u4 u[4], hv[3];
#pragma unroll
            for (int e = 0; e < 4; e++) u[e] = there ? *(const pv_u4 *)(up + min(col + e, a.N - 1) * r16 + r) : (pv_u4){0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < 3; x++) hv[x] = there ? *(const pv_u4 *)(hl + c * ld + x * r16 + r) : (pv_u4){0, 0, 0, 0};
#pragma unroll
            for (int x = 2; x >= 0; x--)
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = mfma(hv[x], u[e], o[e]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = 4 * q4 + i;
            if (t >= n || col >= a.N) continue;
            const long long at = tok[t] * a.ldo + col;
            if (a.vec & 2) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[i][e] = ad >= 0 ? fmaf(o[e][i], scale, v[i][e]) : v[i][e];
                *(pv_f4 *)(a.out + at) = v[i];
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (col + e >= a.N) continue;
                    const float x = a.base ? a.base[at + e] : 0.f;
                    a.out[at + e] = ad >= 0 ? fmaf(o[e][i], scale, x) : x;
                }
            }
        }
    }
}
} // namespace

// parts of K, for `most` tiles: so that the tiles of a batch of one adapter each fill the chip four times, 64 numbers of K a wave at least (64 adapters of rank 64, K 4096: 13 parts, 10.3 us; 7 parts, 13.8)
static int parts_of(const ps_adapters &s, int64_t most) { return (int)std::max<int64_t>(1, std::min<int64_t>({(4 * s.n_cu + most - 1) / most, s.KP / 256, 16})); }
static int64_t tiles_of(const ps_adapters &s, int64_t T, bool plan) { return !plan ? T : std::min<int64_t>(T, (int64_t)s.n_slots + 1 + T / TILE); } // there can be
static void adapt_carve(const ps_adapters &s, ad_args &a, ps_carve &ws, int64_t T, int64_t tiles, int64_t in_parts, bool plan, int32_t **count) {
    a.h = ws.take<float>((size_t)(in_parts * s.RP * TILE));
    if (!plan) return;
    a.order = ws.take<int32_t>((size_t)T);
    a.tiles = ws.take<int32_t>(1 + 3 * (size_t)tiles);
    *count = ws.take<int32_t>((size_t)s.n_slots + 1);
}
// The most that any call of up to T tokens takes.
size_t psv_adapt_most(const ps_adapters &s, int T) {
    const bool plan = !plans_itself(T, s.N);
    const int64_t alone = std::min<int64_t>({(int64_t)T, 256, (1 << 19) / s.N}), tiles = std::max(alone, plan ? tiles_of(s, T, true) : 0);
    int64_t in_parts = tiles; // of one part each, or of p > 1 parts: as many tiles as still have them
    for (int p = 2; p <= std::min<int64_t>(s.KP / 256, 16); p++) in_parts = std::max(in_parts, p * std::min<int64_t>(tiles, (4 * s.n_cu - 1) / (p - 1)));
    ad_args a{};
    ps_carve ws{nullptr};
    int32_t *count = nullptr;
    adapt_carve(s, a, ws, T, tiles, in_parts, plan, &count);
    return ws.at;
}
size_t psv_adapt_space(const ps_adapters &s, int x_dtype, const void *x, int64_t ldx, int T, const int32_t *ids, const float *base_out, float *out, int64_t ldo, void *base, bool launch, hipStream_t st) {
    ad_args a{};
    const bool plan = !plans_itself(T, s.N);
    const int most = (int)tiles_of(s, T, plan);
    a.parts = parts_of(s, most);
    ps_carve ws{(char *)base};
    int32_t *count = nullptr;
    adapt_carve(s, a, ws, T, most, (int64_t)a.parts * most, plan, &count);
    if (!launch) return ws.at;
    a.down = s.down; a.up = s.up; a.rank = s.rank; a.ids = ids; a.scale = s.scale; a.x = (const char *)x; a.base = base_out; a.out = out;
    a.N = s.N; a.K = s.K; a.KP = s.KP; a.RP = s.RP; a.ldx = ldx; a.ldo = ldo; a.n_slots = s.n_slots; a.T = T;
    const int size = x_dtype == PS_F32 ? 4 : 2;
    a.vec = ((uintptr_t)x % 16 == 0 && ldx * size % 16 == 0 ? 1 : 0) | ((uintptr_t)out % 16 == 0 && (uintptr_t)base_out % 16 == 0 && ldo % 4 == 0 && s.N % 4 == 0 ? 2 : 0);
    if (plan) hipLaunchKernelGGL(adapt_plan_kernel, dim3(1), dim3(1024), s.n_slots + 1 <= PLAN_LDS ? (size_t)(s.n_slots + 1) * 4 : 0, st, a, count);
    if (x_dtype == PS_F32) hipLaunchKernelGGL(adapt_down_kernel<true>, dim3(most, a.parts), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(adapt_down_kernel<false>, dim3(most, a.parts), dim3(256), 0, st, a);
    // 256 columns a work-group until the chip is full four times, then more
    const int64_t stretches = (s.N + 255) / 256, groups = std::min<int64_t>(stretches, std::max<int64_t>(1, (16 * s.n_cu + most - 1) / most));
    a.columns = (int)((stretches + groups - 1) / groups * 256);
    hipLaunchKernelGGL(adapt_up_kernel, dim3(most, (unsigned)((s.N + a.columns - 1) / a.columns)), dim3(256), (size_t)TILE * (3 * s.RP + 8) * 2, st, a);
    return ws.at;
}
