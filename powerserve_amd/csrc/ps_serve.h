// Launchers of the operators of a serving step of many sequences (include/ps_hip.h): attention over caches (k_cacheattn.hip), eviction (k_evict.hip), sampling (k_sample.hip), low-rank adapters
// (k_adapt.hip).  The entries (serve.hip) have checked what they are given; everything enqueues on `st`, nothing waits.
#pragma once
#include "ps_internal.h"

#include <atomic>

// Scratch memory in pieces of 256 bytes' alignment: the same steps give the size (base NULL) and the pieces.
struct ps_carve {
    char *base;
    size_t at = 0;
    template <class T> T *take(size_t n) {
        T *p = base ? (T *)(base + at) : nullptr;
        at += (n * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

// More than 64 KB of LDS for a kernel's launches, once on each device.  Two contexts may come here at the same time: a device counts as done when it is, and both may do it.
inline void ps_allow_lds(const void *kernel, size_t bytes, std::atomic<unsigned long long> &done) {
    int dev = 0;
    (void)hipGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == hipSuccess) done.fetch_or(bit, std::memory_order_release);
}

// psv_*_space: the bytes that a call takes; psv_*_most: the most that any call takes of no more sequences, new tokens, logits, rows or tokens, which is what a server that keeps one workspace asks for
size_t psv_attn_most(int n_cu, const ps_kv_cache &c, const ps_cache_attn_params &p);
size_t psv_sample_most(int n_cu, int64_t n, int64_t rows);
size_t psv_attn_space(int n_cu, const ps_kv_cache &c, const ps_cache_attn_params &p, void *base, bool launch, hipStream_t st); // the bytes it takes; launch: enqueues
void psv_advance(hipStream_t st, const ps_kv_cache &c, const int32_t *count, const int32_t *take, int n_take);
size_t psv_evict_space(const ps_kv_cache &c, const ps_cache_evict_params &p, void *base, bool launch, hipStream_t st);
size_t psv_sample_space(int n_cu, int dtype, const void *logits, int64_t n, int64_t rows, int64_t stride, const ps_sample_params *p, int32_t *ids, float *prob, void *base, bool launch, hipStream_t st);

struct ps_adapters {
    int64_t N = 0, K = 0, KP = 0; // KP: K up to a multiple of 32 (zeros behind K)
    int n_slots = 0, max_rank = 0, RP = 0; // RP: max_rank up to a multiple of 16
    uint16_t *down = nullptr; // [n_slots][RP][KP]
    uint16_t *up = nullptr;   // [n_slots][N][RP]
    int32_t *rank = nullptr;  // [n_slots], 0: empty
    float *scale = nullptr;   // [n_slots]
    int device = 0, n_cu = 256;
};
size_t psv_adapt_most(const ps_adapters &a, int T);
size_t psv_adapt_space(const ps_adapters &a, int x_dtype, const void *x, int64_t ldx, int T, const int32_t *ids, const float *base_out, float *out, int64_t ldo, void *base, bool launch, hipStream_t st);

// a 16-byte piece of 16-bit numbers, and the wave's fp32 accumulators
typedef unsigned pv_u4 __attribute__((ext_vector_type(4)));
typedef unsigned pv_u2 __attribute__((ext_vector_type(2)));
typedef float pv_f4 __attribute__((ext_vector_type(4)));
typedef float pv_f2 __attribute__((ext_vector_type(2)));
