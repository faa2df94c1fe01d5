// Eviction from the caches of many sequences by accumulated attention weight (ps_hip_cache_evict).
//   evict_choose_kernel  a work-group per sequence and kv head: an order of 32-bit keys (protected slots above every weight, weights as whole numbers of the same order), the keep-th largest of them
//                        by three digits of 11, 11 and 10 bits (a histogram in LDS each), then one walk over the slots that lists the holes below the bound and the kept slots behind it
//   evict_move_kernel    the i-th hole takes the i-th kept slot: sources lie behind the bound and destinations below it, so that nothing waits for anything
// Moving a row for a hole, instead of closing the gaps, moves what has to move: at most the evicted number of rows, and never more than keep.
#include "ps_serve.h"

#include <algorithm>

namespace {
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
    const unsigned u = __float_as_uint(w);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
    return min((u & 0x80000000u) ? ~u : u | 0x80000000u, 0xfffffffeu);
}
// sum over the threads before this one; *total: over all (sh: 17 numbers; barriers inside)
__device__ __forceinline__ int scan_before(int v, int *sh, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) sh[wave] = x;
    __syncthreads();
    if (threadIdx.x < 64) {
        int y = threadIdx.x < EV_THREADS / 64 ? sh[threadIdx.x] : 0;
        const int own = y;
#pragma unroll
        for (int o = 1; o < EV_THREADS / 64; o <<= 1) {
            const int z = __shfl_up(y, o, 64);
            if (lane >= o) y += z;
        }
        if (threadIdx.x < EV_THREADS / 64) sh[threadIdx.x] = y - own;
        if (threadIdx.x == EV_THREADS / 64 - 1) sh[16] = y;
    }
    __syncthreads();
    const int before = sh[wave] + x - v;
    *total = sh[16];
    __syncthreads();
    return before;
}

__global__ __launch_bounds__(EV_THREADS) void evict_choose_kernel(const ev_args a) {
    extern __shared__ unsigned keys[]; // in_lds: a key per held slot
    __shared__ unsigned hist[2048];
    __shared__ int sh[17], counts[1024], pre[1024], cut[2], newest_;
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
    // the largest position
    int top = INT32_MIN;
    for (int j = tid; j < n; j += EV_THREADS) top = max(top, p[j]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
    if (tid == 0) newest_ = INT32_MIN;
    for (int b = tid; b < 2048; b += EV_THREADS) hist[b] = 0;
    __syncthreads();
    if (lane == 0) atomicMax(&newest_, top);
    __syncthreads();
    const long long since = (long long)newest_ - a.recent; // positions above it are recent
    auto key_of = [&](int j) { return p[j] < a.first || p[j] > since ? 0xffffffffu : order_of(w[j]); };
    auto key = [&](int j) { return a.in_lds ? keys[j] : key_of(j); };
    // the keep-th largest key, digit by digit
    unsigned found = 0, mask = 0;
    int need = keep;
#pragma unroll
    for (int d = 0; d < 3; d++) {
        const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, bits = d == 2 ? 10 : 11;
        for (int j = tid; j < n; j += EV_THREADS) {
            const unsigned x = d == 0 ? key_of(j) : key(j);
            if (d == 0 && a.in_lds) keys[j] = x;
            if ((x & mask) == found) atomicAdd(&hist[x >> shift & ((1u << bits) - 1)], 1u);
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
    // the walk: of the slots whose key is the one found, the first `need` stay
    int ties = 0, holes = 0, moves = 0;
    int32_t *hole = a.hole + head * a.cap, *moved = a.moved + head * a.cap;
    const unsigned long long below = (1ull << lane) - 1;
    for (int base = 0; base < n; base += 65536) {
        const int nb = min(1024, (n - base + 63) / 64);
        for (int b = wave; b < nb; b += EV_THREADS / 64) {
            const int j = base + 64 * b + lane;
            const unsigned long long eq = __ballot(j < n && key(min(j, n - 1)) == found);
            if (lane == 0) counts[b] = __popcll(eq);
        }
        __syncthreads();
        int all;
        const int t0 = ties + scan_before(tid < nb ? counts[tid] : 0, sh, &all);
        pre[tid] = t0;
        ties += all;
        __syncthreads();
        auto stays = [&](int b, int j) {
            const unsigned x = key(min(j, n - 1));
            const unsigned long long eq = __ballot(j < n && x == found);
            return j < n && (x > found || (x == found && pre[b] + (int)__popcll(eq & below) < need));
        };
        for (int b = wave; b < nb; b += EV_THREADS / 64) {
            const int j = base + 64 * b + lane;
            const bool kept = stays(b, j);
            const int h = __popcll(__ballot(j < n && j < keep && !kept)), m = __popcll(__ballot(kept && j >= keep));
            if (lane == 0) counts[b] = h << 8 | m;
        }
        __syncthreads();
        const int c = tid < nb ? counts[tid] : 0;
        int all_h, all_m;
        const int h0 = holes + scan_before(c >> 8, sh, &all_h), m0 = moves + scan_before(c & 255, sh, &all_m);
        counts[tid] = h0;
        hist[tid] = (unsigned)m0;
        holes += all_h;
        moves += all_m;
        __syncthreads();
        for (int b = wave; b < nb; b += EV_THREADS / 64) {
            const int j = base + 64 * b + lane;
            const bool kept = stays(b, j);
            const bool h = j < n && j < keep && !kept, m = kept && j >= keep;
            const unsigned long long hb = __ballot(h), mb = __ballot(m);
            if (h) hole[counts[b] + (int)__popcll(hb & below)] = j;
            if (m) moved[(int)hist[b] + (int)__popcll(mb & below)] = j;
            if (kept && j < keep) {
                if (wo) wo[j] = w[j];
                if (po) po[j] = p[j];
            }
        }
        __syncthreads();
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
    static unsigned long long seen = 0;
    if (lds && ps_first_on_device(&seen)) (void)hipFuncSetAttribute((const void *)evict_choose_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, EV_LDS_KEYS * 4);
    hipLaunchKernelGGL(evict_choose_kernel, dim3((unsigned)c.kv_heads, (unsigned)c.n_seqs), dim3(EV_THREADS), lds, st, a);
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)std::max(1, (a.cap + EV_ROWS - 1) / EV_ROWS), (unsigned)c.kv_heads, (unsigned)c.n_seqs), dim3(256), 0, st, a);
    return ws.at;
}
