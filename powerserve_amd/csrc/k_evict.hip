// Eviction from the caches of many sequences by accumulated attention weight (ps_hip_cache_evict).
//   evict_choose_kernel  a work-group per sequence and kv head: an order of 32-bit keys (protected slots above every weight, weights as whole numbers of the same order), the keep-th largest of them
//                        by three digits of 11, 11 and 10 bits (a histogram in LDS each), then one walk over the slots that lists the holes below the bound and the kept slots behind it
//   evict_move_kernel    the i-th hole takes the i-th kept slot: sources lie behind the bound and destinations below it, so that nothing waits for anything
// Moving a row for a hole, instead of closing the gaps, moves what has to move: at most the evicted number of rows, and never more than keep.
// Measured: 16 sequences of 2100 to 16384 slots down to 2048, 8 heads of 128 bf16: the choice 21 us (128 work-groups, each a chain of twelve barriers behind two loads of its slots: latency), the moves
// 34 us for 168 MB, 4.9 TB/s, what a large copy reaches.  A slot more than 2048 of 8 sequences: 10 and 3 us, latency both.
#include "ps_serve.h"

#include <algorithm>

namespace {
typedef int i4 __attribute__((ext_vector_type(4)));
constexpr int EV_THREADS = 1024, EV_LDS_KEYS = 32768;
struct ev_args {
    char *k, *v;
    long long seq, slot, head; // strides in bytes
    int G, n_ctx, row_bytes, keep, recent, first, cap, in_lds;
    const int32_t *n_kv;
    const int32_t *pos;
    const float *weight;
    int32_t *n_kv_out, *pos_out;
    float *weight_out;
    int32_t *hole, *moved; // [seq][kv head][cap]
    int32_t *meta;         // [seq][kv head][2]: moves, slots that stay
};
// weights as whole numbers of the same order, NaN lowest
__device__ __forceinline__ unsigned order_of(float w) {
    const unsigned u = __float_as_uint(w == 0.f ? 0.f : w); // (the two zeros are equal)
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
    return min((u & 0x80000000u) ? ~u : u | 0x80000000u, 0xfffffffeu);
}
// sums over a wave's lanes up to and with each
template <int CTRL, int ROWS> __device__ __forceinline__ int moved(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 15, false); }
__device__ __forceinline__ int wave_sums(int v) {
    v += moved<0x111, 15>(v); // row_shr: 1, 2, 4, 8
    v += moved<0x112, 15>(v);
    v += moved<0x114, 15>(v);
    v += moved<0x118, 15>(v);
    v += moved<0x142, 10>(v); // row_bcast: 15 into rows 1 and 3, 31 into rows 2 and 3
    v += moved<0x143, 12>(v);
    return v;
}
// sum over the threads before this one; *total: over all (sh: 16 numbers; barriers inside)
__device__ __forceinline__ int scan_before(int v, int *sh, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = wave_sums(v);
    if (lane == 63) sh[wave] = x;
    __syncthreads();
    const int y = lane < EV_THREADS / 64 ? sh[lane] : 0, z = wave_sums(y);
    *total = __builtin_amdgcn_readlane(z, 63);
    const int before = __builtin_amdgcn_readlane(z - y, wave) + x - v;
    __syncthreads();
    return before;
}

__global__ __launch_bounds__(EV_THREADS) void evict_choose_kernel(const ev_args a) {
    extern __shared__ unsigned keys[]; // in_lds: a key per held slot
    __shared__ unsigned hist[2048];
    __shared__ unsigned stay[EV_THREADS];
    __shared__ int sh[16], cut[2], newest_;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = blockIdx.x, s = blockIdx.y;
    const long long head = (long long)s * a.G + g, at = head * a.n_ctx;
    const int n = min(max(a.n_kv[s], 0), a.n_ctx), keep = a.keep;
    const float *w = a.weight + at;
    const int32_t *p = a.pos + at;
    float *wo = a.weight_out == a.weight ? nullptr : a.weight_out + at;
    int32_t *po = a.pos_out == a.pos ? nullptr : a.pos_out + at;
    if (n <= keep) {
        for (int j = tid; j < n; j += EV_THREADS) {
            if (wo) wo[j] = w[j];
            if (po) po[j] = p[j];
        }
        if (tid == 0) { a.meta[2 * head] = 0; a.meta[2 * head + 1] = n; }
        return;
    }
    // four slots at a time where a head's numbers are 16-byte aligned, four such pieces of a thread in flight
    const bool wide = a.n_ctx % 4 == 0 && ((uintptr_t)a.weight | (uintptr_t)a.pos) % 16 == 0;
    auto load_pos = [&](int j) {
        if (wide) return *(const i4 *)(p + j);
        return (i4){p[j], p[min(j + 1, n - 1)], p[min(j + 2, n - 1)], p[min(j + 3, n - 1)]};
    };
    auto load_weight = [&](int j) {
        if (wide) return *(const pv_f4 *)(w + j);
        return (pv_f4){w[j], w[min(j + 1, n - 1)], w[min(j + 2, n - 1)], w[min(j + 3, n - 1)]};
    };
    constexpr int STEP = EV_THREADS * 4, AT_ONCE = 4 * STEP;
    i4 v[4];
    pv_f4 u[4];
    const bool once = n <= AT_ONCE; // positions and weights of so many slots are loaded together, and once
    // the largest position
    int top = INT32_MIN;
    for (int base = 4 * tid; base < n; base += AT_ONCE) {
#pragma unroll
        for (int x = 0; x < 4; x++) v[x] = load_pos(base + x * STEP < n ? base + x * STEP : base);
        if (once)
#pragma unroll
            for (int x = 0; x < 4; x++) u[x] = load_weight(base + x * STEP < n ? base + x * STEP : base);
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (base + x * STEP + e < n) top = max(top, v[x][e]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
    if (tid == 0) newest_ = INT32_MIN;
    for (int b = tid; b < 2048; b += EV_THREADS) hist[b] = 0;
    __syncthreads();
    if (lane == 0) atomicMax(&newest_, top);
    __syncthreads();
    const long long since = (long long)newest_ - a.recent; // positions above it are recent
    auto key_from = [&](int pos, float weight) { return pos < a.first || pos > since ? 0xffffffffu : order_of(weight); };
    auto key = [&](int j) { return a.in_lds ? keys[j] : key_from(p[j], w[j]); };
    // the first digit's histogram, and the keys into LDS.  A wave whose keys all have the same digit counts them at once: one behind the other in one place of the LDS, 16384 equal weights would be 52 us
    // instead of 30.
    auto count = [&](unsigned k, int shift, int bits) {
        const unsigned d = k >> shift & ((1u << bits) - 1), one = (unsigned)__builtin_amdgcn_readfirstlane((int)d);
        const unsigned long long there = __ballot(true);
        if (__ballot(d == one) == there) {
            if (lane == __ffsll(there) - 1) atomicAdd(&hist[d], (unsigned)__popcll(there));
        } else atomicAdd(&hist[d], 1u);
    };
    for (int base = 4 * tid; base < n; base += AT_ONCE) {
        if (!once)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int j = base + x * STEP < n ? base + x * STEP : base;
                v[x] = load_pos(j);
                u[x] = load_weight(j);
            }
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = base + x * STEP + e;
                if (j >= n) continue;
                const unsigned k = key_from(v[x][e], u[x][e]);
                if (a.in_lds) keys[j] = k;
                count(k, 21, 11);
            }
    }
    // the keep-th largest key, digit by digit
    unsigned found = 0, mask = 0;
    int need = keep;
#pragma unroll 1
    for (int d = 0; d < 3; d++) {
        const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, bits = d == 2 ? 10 : 11;
        if (d)
            for (int j = tid; j < n; j += EV_THREADS) {
                const unsigned x = key(j);
                if ((x & mask) == found) count(x, shift, bits);
            }
        __syncthreads();
        // from the largest digit down: thread t has digits 2047 - 2 t and 2046 - 2 t
        const int hi = (int)hist[2047 - 2 * tid], lo = (int)hist[2046 - 2 * tid];
        int all;
        const int before = scan_before(hi + lo, sh, &all);
        if (before < need && need <= before + hi) { cut[0] = 2047 - 2 * tid; cut[1] = need - before; }
        else if (before + hi < need && need <= before + hi + lo) { cut[0] = 2046 - 2 * tid; cut[1] = need - before - hi; }
        hist[2047 - 2 * tid] = hist[2046 - 2 * tid] = 0;
        __syncthreads();
        found |= (unsigned)cut[0] << shift;
        mask |= ((1u << bits) - 1) << shift;
        need = cut[1]; // of those that share the digits so far
        __syncthreads();
    }
    // the walk: of the slots whose key is the one found, the first `need` stay.  A thread has up to 32 slots in a row, a bit each.
    int ties = 0, holes = 0, moves = 0;
    int32_t *hole = a.hole + head * a.cap, *moved = a.moved + head * a.cap;
    for (int base = 0; base < n; base += EV_LDS_KEYS) {
        const int end = min(n, base + EV_LDS_KEYS), per = (end - base + EV_THREADS - 1) / EV_THREADS, j0 = base + tid * per;
        unsigned gt = 0, eq = 0;
        int i = tid % per; // (each begins elsewhere: 32 lanes would read one LDS bank)
        for (int x = 0; x < per; x++, i = i + 1 == per ? 0 : i + 1) {
            if (j0 + i >= end) continue;
            const unsigned k = key(j0 + i);
            gt |= (k > found ? 1u : 0u) << i;
            eq |= (k == found ? 1u : 0u) << i;
        }
        int all;
        int room = need - (ties + scan_before((int)__popc(eq), sh, &all));
        ties += all;
        unsigned kept = gt;
        if (room >= (int)__popc(eq)) kept |= eq;
        else
            for (; room > 0; room--) { // its lowest ones
                kept |= eq & -eq;
                eq &= eq - 1;
            }
        auto ones = [](int k) { return k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1; };
        const unsigned there = ones(min(per, end - j0)), below = ones(keep - j0);
        unsigned h = there & below & ~kept, m = there & kept & ~below;
        const int before = scan_before((int)(__popc(h) << 16 | __popc(m)), sh, &all); // (at most 32768 each)
        int hi = holes + (int)((unsigned)before >> 16), mi = moves + (before & 0xffff);
        holes += (int)((unsigned)all >> 16);
        moves += all & 0xffff;
        for (; h; h &= h - 1) hole[hi++] = j0 + __ffs(h) - 1;
        for (; m; m &= m - 1) moved[mi++] = j0 + __ffs(m) - 1;
        if (wo || po) { // what stays where it is, into the caller's new arrays
            stay[tid] = kept;
            __syncthreads();
            for (int j = base + tid; j < min(end, keep); j += EV_THREADS)
                if (stay[(j - base) / per] >> ((j - base) % per) & 1) {
                    if (wo) wo[j] = w[j];
                    if (po) po[j] = p[j];
                }
            __syncthreads();
        }
    }
    if (tid == 0) { a.meta[2 * head] = moves; a.meta[2 * head + 1] = keep; }
}

constexpr int EV_ROWS = 32; // rows a work-group moves
__global__ __launch_bounds__(256) void evict_move_kernel(const ev_args a) {
    const int g = blockIdx.y, s = blockIdx.z, i0 = blockIdx.x * EV_ROWS;
    const long long head = (long long)s * a.G + g, at = head * a.n_ctx;
    const int moves = a.meta[2 * head];
    if (blockIdx.x == 0 && g == 0 && threadIdx.x == 0) a.n_kv_out[s] = a.meta[2 * head + 1];
    if (i0 >= moves) return;
    const int32_t *hole = a.hole + head * a.cap, *moved = a.moved + head * a.cap;
    const int rows = min(EV_ROWS, moves - i0), per = a.row_bytes / 16;
    char *kr = a.k + s * a.seq + g * a.head, *vr = a.v + s * a.seq + g * a.head;
    for (int x = threadIdx.x; x < rows * per; x += 256) {
        const int i = i0 + x / per;
        const long long to = hole[i] * a.slot + x % per * 16, from = moved[i] * a.slot + x % per * 16;
        const pv_u4 kv = *(const pv_u4 *)(kr + from), vv = *(const pv_u4 *)(vr + from);
        *(pv_u4 *)(kr + to) = kv;
        *(pv_u4 *)(vr + to) = vv;
    }
    if ((int)threadIdx.x < rows) {
        const int i = i0 + threadIdx.x;
        a.weight_out[at + hole[i]] = a.weight[at + moved[i]];
        a.pos_out[at + hole[i]] = a.pos[at + moved[i]];
    }
}
} // namespace

size_t psv_evict_space(const ps_kv_cache &c, const ps_cache_evict_params &p, void *base, bool launch, hipStream_t st) {
    const int size = c.dtype == PS_F32 ? 4 : 2;
    const size_t heads = (size_t)c.n_seqs * c.kv_heads;
    ev_args a{};
    a.cap = std::max(0, std::min(p.keep, c.n_ctx - p.keep));
    ps_carve ws{(char *)base};
    a.meta = ws.take<int32_t>(heads * 2);
    a.hole = ws.take<int32_t>(heads * a.cap);
    a.moved = ws.take<int32_t>(heads * a.cap);
    if (!launch) return ws.at;
    a.k = (char *)c.k; a.v = (char *)c.v;
    a.seq = c.seq_stride * size; a.slot = c.slot_stride * size; a.head = c.head_stride * size;
    a.G = c.kv_heads; a.n_ctx = c.n_ctx; a.row_bytes = c.dim * size; a.keep = p.keep; a.recent = p.recent; a.first = p.first;
    a.n_kv = c.n_kv; a.pos = c.pos; a.weight = c.weight;
    a.n_kv_out = p.n_kv_out ? p.n_kv_out : c.n_kv; a.pos_out = p.pos_out ? p.pos_out : c.pos; a.weight_out = p.weight_out ? p.weight_out : c.weight;
    // the keys of up to 32768 slots fit the LDS (128 KB): the passes behind the first read them there, else weights and positions again
    a.in_lds = c.n_ctx <= EV_LDS_KEYS;
    const size_t lds = a.in_lds ? (size_t)c.n_ctx * 4 : 0;
    static std::atomic<unsigned long long> done{0};
    if (lds) ps_allow_lds((const void *)evict_choose_kernel, EV_LDS_KEYS * 4, done);
    hipLaunchKernelGGL(evict_choose_kernel, dim3((unsigned)c.kv_heads, (unsigned)c.n_seqs), dim3(EV_THREADS), lds, st, a);
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)std::max(1, (a.cap + EV_ROWS - 1) / EV_ROWS), (unsigned)c.kv_heads, (unsigned)c.n_seqs), dim3(256), 0, st, a);
    return ws.at;
}
