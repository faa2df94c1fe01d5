// C-ABI (include/ps_hip.h): the operators of a serving step of many sequences -- what a call may ask for, and on to the kernels.
#include "ps_serve.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>

// Launches go to the device that is current; a caller's other device is current again afterwards.
namespace {
struct on_device {
    int was = -1;
    bool ok;
    explicit on_device(const ps_hip_ctx *c) {
        ok = hipGetDevice(&was) == hipSuccess && (was == c->device || hipSetDevice(c->device) == hipSuccess);
        now = c->device;
    }
    ~on_device() {
        if (ok && was != now) (void)hipSetDevice(was);
    }
    int now;
};
bool aligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
constexpr int64_t MOST_GROUPS = (1 << 24) - 1; // work-groups of 256 threads of a launch: a grid has fewer than 2^32 threads a direction
int number_size(int dtype) { return dtype == PS_F32 ? 4 : dtype == PS_F16 || dtype == PS_BF16 ? 2 : 0; }

// what is wrong with a cache, or NULL
const char *wrong_cache(const ps_kv_cache *k) {
    if (!k) return "no cache";
    const int size = number_size(k->dtype);
    if (!size) return "the cache's type must be F32, F16 or BF16";
    if (k->n_seqs < 0 || k->n_ctx < 1 || k->kv_heads < 1) return "the cache has no slots or heads";
    if (k->dim < 8 || k->dim > 128 || k->dim % 8) return "a head's size must be a multiple of 8, 8 to 128";
    if (k->n_seqs > 65535 || k->kv_heads > 65535 || k->n_ctx > (1 << 28)) return "too many sequences, heads or slots";
    if (k->n_seqs && (!k->k || !k->v || !k->n_kv || k->k == k->v)) return "keys, values and lengths are missing or the same";
    if (!aligned(k->k, 16) || !aligned(k->v, 16) || k->seq_stride * size % 16 || k->slot_stride * size % 16 || k->head_stride * size % 16) return "rows must be 16-byte aligned";
    return nullptr;
}
const char *wrong_attn(const ps_kv_cache *k, const ps_cache_attn_params *p) {
    if (const char *w = wrong_cache(k)) return w;
    if (!p) return "no parameters";
    const int size = number_size(k->dtype);
    if (p->heads < 1 || p->heads % k->kv_heads) return "the query heads must be a multiple of the cache's heads";
    if (p->n_new < 0 || p->n_new > k->n_ctx) return "more new tokens than slots";
    if (!(std::fabs(p->scale) <= 1e30f)) return "the scale is not a number, or above 1e30";
    const int64_t heads = (int64_t)k->n_seqs * k->kv_heads, rows = (int64_t)p->n_new * (p->heads / k->kv_heads);
    if (rows > (1 << 24) || rows * (p->heads / k->kv_heads) > UINT32_MAX || (int64_t)p->n_new * k->kv_heads * 32 > INT32_MAX || heads * ((rows + 15) / 16) > MOST_GROUPS / 2 - 65536 || heads * ((k->n_ctx + 63) / 64) > MOST_GROUPS) return "too many rows or slots";
    if (!k->n_seqs || !p->n_new) return nullptr;
    if (!p->q || !p->out || p->q == p->out) return "q and out are missing or the same";
    if (!p->k_new != !p->v_new) return "new keys and values come together";
    if (!aligned(p->q, 16) || !aligned(p->out, 16) || !aligned(p->k_new, 16) || !aligned(p->v_new, 16) || p->q_seq_stride * size % 16 || p->q_row_stride * size % 16 || p->out_seq_stride * size % 16 ||
        p->out_row_stride * size % 16 || p->new_seq_stride * size % 16 || p->new_row_stride * size % 16)
        return "rows must be 16-byte aligned";
    if (p->pos_new && !k->pos) return "positions have no place in the cache";
    if (p->pos_new && !p->k_new) return "positions come with new keys and values";
    return nullptr;
}
// rows one behind the other where a stride is 0
ps_cache_attn_params with_strides(const ps_kv_cache &k, ps_cache_attn_params p) {
    if (!p.q_row_stride) p.q_row_stride = (int64_t)p.heads * k.dim;
    if (!p.out_row_stride) p.out_row_stride = (int64_t)p.heads * k.dim;
    if (!p.new_row_stride) p.new_row_stride = (int64_t)k.kv_heads * k.dim;
    if (!p.q_seq_stride) p.q_seq_stride = p.n_new * p.q_row_stride;
    if (!p.out_seq_stride) p.out_seq_stride = p.n_new * p.out_row_stride;
    if (!p.new_seq_stride) p.new_seq_stride = p.n_new * p.new_row_stride;
    return p;
}
#define SV_FAIL(ctx, call, what) PS_FAIL(ctx, std::string(call ": ") + (what))
#define SV_DEVICE(ctx, call)                                                                   \
    const on_device dev_(ctx);                                                                 \
    if (!dev_.ok) { (void)hipGetLastError(); (ctx)->err = call ": the device"; return 1; }
} // namespace

extern "C" {

size_t ps_hip_cache_attn_workspace(ps_hip_ctx *c, const ps_kv_cache *k, const ps_cache_attn_params *p) {
    if (!c || wrong_attn(k, p) || !k->n_seqs || !p->n_new) return 0;
    return psv_attn_most(c->n_cu, *k, *p);
}
int ps_hip_cache_attn(ps_hip_ctx *c, const ps_kv_cache *k, const ps_cache_attn_params *p, void *ws, size_t bytes) {
    if (!c) return 2;
    if (const char *w = wrong_attn(k, p)) SV_FAIL(c, "cache_attn", w);
    if (!k->n_seqs || !p->n_new) return 0;
    if (!ws || !aligned(ws, 16) || bytes < psv_attn_space(c->n_cu, *k, *p, nullptr, false, c->stream)) SV_FAIL(c, "cache_attn", "the workspace is too small or not aligned");
    SV_DEVICE(c, "cache_attn")
    psv_attn_space(c->n_cu, *k, with_strides(*k, *p), ws, true, c->stream);
    PS_CHECK(c, hipGetLastError());
    return 0;
}
int ps_hip_cache_advance(ps_hip_ctx *c, const ps_kv_cache *k, const int32_t *count, const int32_t *take, int n_take) {
    if (!c) return 2;
    if (const char *w = wrong_cache(k)) SV_FAIL(c, "cache_advance", w);
    if (!k->n_seqs) return 0;
    if (!count) SV_FAIL(c, "cache_advance", "no counts");
    if (n_take < 0) SV_FAIL(c, "cache_advance", "a negative number of indices");
    SV_DEVICE(c, "cache_advance")
    psv_advance(c->stream, *k, count, take, n_take);
    PS_CHECK(c, hipGetLastError());
    return 0;
}


// ------------------------------------------------------------------ eviction
static const char *wrong_evict(const ps_kv_cache *k, const ps_cache_evict_params *p) {
    if (const char *w = wrong_cache(k)) return w;
    if (!p) return "no parameters";
    if (p->keep < 1 || p->recent < 0 || p->first < 0 || (int64_t)p->recent + p->first > p->keep) return "keep must be at least 1, and at least recent + first";
    if (k->n_seqs && (!k->pos || !k->weight)) return "the cache has no positions or weights";
    return nullptr;
}
size_t ps_hip_cache_evict_workspace(ps_hip_ctx *c, const ps_kv_cache *k, const ps_cache_evict_params *p) {
    if (!c || wrong_evict(k, p) || !k->n_seqs) return 0;
    return psv_evict_space(*k, *p, nullptr, false, c->stream);
}
int ps_hip_cache_evict(ps_hip_ctx *c, const ps_kv_cache *k, const ps_cache_evict_params *p, void *ws, size_t bytes) {
    if (!c) return 2;
    if (const char *w = wrong_evict(k, p)) SV_FAIL(c, "cache_evict", w);
    if (!k->n_seqs) return 0;
    if (!ws || !aligned(ws, 16) || bytes < psv_evict_space(*k, *p, nullptr, false, c->stream)) SV_FAIL(c, "cache_evict", "the workspace is too small or not aligned");
    SV_DEVICE(c, "cache_evict")
    psv_evict_space(*k, *p, ws, true, c->stream);
    PS_CHECK(c, hipGetLastError());
    return 0;
}

// ------------------------------------------------------------------ sampling
static const char *wrong_sample(int64_t n, int64_t rows) {
    if (n < 1 || n > (1 << 24)) return "a row has 1 to 2^24 logits";
    if (rows < 0 || rows > MOST_GROUPS / 4) return "0 to 2^22 - 1 rows"; // (1024 threads each)
    return nullptr;
}
size_t ps_hip_sample_workspace(ps_hip_ctx *c, int64_t n, int64_t rows) {
    if (!c || wrong_sample(n, rows) || !rows) return 0;
    return psv_sample_most(c->n_cu, n, rows);
}
int ps_hip_sample(ps_hip_ctx *c, int dtype, const void *logits, int64_t n, int64_t rows, int64_t stride, const ps_sample_params *p, int32_t *ids, float *prob, void *ws, size_t bytes) {
    if (!c) return 2;
    if (const char *w = wrong_sample(n, rows)) SV_FAIL(c, "sample", w);
    const int size = number_size(dtype);
    if (!size) SV_FAIL(c, "sample", "logits must be F32, F16 or BF16");
    if (stride < n && rows > 1) SV_FAIL(c, "sample", "rows overlap");
    if (!rows) return 0;
    if (!p || !p->u) SV_FAIL(c, "sample", "no random numbers");
    if (!logits || !ids || !aligned(logits, size)) SV_FAIL(c, "sample", "logits or ids are missing or not aligned");
    const size_t need = psv_sample_space(c->n_cu, dtype, nullptr, n, rows, stride, nullptr, nullptr, nullptr, nullptr, false, c->stream);
    if (need && (!ws || !aligned(ws, 16) || bytes < need)) SV_FAIL(c, "sample", "the workspace is too small or not aligned");
    SV_DEVICE(c, "sample")
    psv_sample_space(c->n_cu, dtype, logits, n, rows, stride, p, ids, prob, ws, true, c->stream);
    PS_CHECK(c, hipGetLastError());
    return 0;
}

// ------------------------------------------------------------------ low-rank adapters
// (The other factor goes in as three numbers that add up to it, of which the last ones are 0 where the first is exact: an infinite number in a matrix times those would be NaN instead of infinity.)
static bool any_infinite(const uint16_t *m, int64_t n) {
    bool any = false;
    for (int64_t i = 0; i < n; i++) any |= (m[i] & 0x7fff) == 0x7f80;
    return any;
}
int ps_hip_adapters_create(ps_hip_ctx *c, int64_t N, int64_t K, int n_slots, int max_rank, ps_adapters **out) {
    if (!c) return 2;
    if (!out) SV_FAIL(c, "adapters_create", "no place for the handle");
    *out = nullptr;
    if (N < 1 || K < 1 || N > (1 << 24) || K > (1 << 24)) SV_FAIL(c, "adapters_create", "a matrix of 1 to 2^24 rows and columns");
    if (n_slots < 1 || n_slots > 65536 || max_rank < 1 || max_rank > 256) SV_FAIL(c, "adapters_create", "1 to 65536 slots of rank 1 to 256");
    SV_DEVICE(c, "adapters_create")
    auto a = new (std::nothrow) ps_adapters();
    if (!a) SV_FAIL(c, "adapters_create", "out of memory");
    a->N = N; a->K = K; a->KP = (K + 31) / 32 * 32; a->n_slots = n_slots; a->max_rank = max_rank; a->RP = (max_rank + 15) / 16 * 16;
    a->device = c->device; a->n_cu = c->n_cu;
    const bool ok = hipMalloc((void **)&a->down, (size_t)n_slots * a->RP * a->KP * 2) == hipSuccess && hipMalloc((void **)&a->up, (size_t)n_slots * a->RP * N * 2) == hipSuccess &&
                    hipMalloc((void **)&a->rank, (size_t)n_slots * 4) == hipSuccess && hipMalloc((void **)&a->scale, (size_t)n_slots * 4) == hipSuccess &&
                    hipMemsetAsync(a->rank, 0, (size_t)n_slots * 4, c->stream) == hipSuccess && hipMemsetAsync(a->scale, 0, (size_t)n_slots * 4, c->stream) == hipSuccess &&
                    hipStreamSynchronize(c->stream) == hipSuccess;
    if (!ok) {
        (void)hipGetLastError();
        ps_hip_adapters_free(c, a);
        c->err = "adapters_create: device memory";
        return 1;
    }
    *out = a;
    return 0;
}
void ps_hip_adapters_free(ps_hip_ctx *c, ps_adapters *a) {
    if (!a) return;
    if (c) (void)hipStreamSynchronize(c->stream);
    for (void *p : {(void *)a->down, (void *)a->up, (void *)a->rank, (void *)a->scale})
        if (p) (void)hipFree(p);
    delete a;
}
int ps_hip_adapters_load(ps_hip_ctx *c, ps_adapters *a, int slot, const uint16_t *down, const uint16_t *up, int rank, float scale) {
    if (!c) return 2;
    if (!a || a->device != c->device) SV_FAIL(c, "adapters_load", "no adapters, or another device's");
    if (slot < 0 || slot >= a->n_slots) SV_FAIL(c, "adapters_load", "no such slot");
    if (rank < 0 || rank > a->max_rank) SV_FAIL(c, "adapters_load", "the rank is above the set's");
    if (rank && (!down || !up)) SV_FAIL(c, "adapters_load", "no matrices");
    if (rank && (any_infinite(down, rank * a->K) || any_infinite(up, rank * a->N))) SV_FAIL(c, "adapters_load", "a matrix holds an infinite number");
    SV_DEVICE(c, "adapters_load")
    PS_CHECK(c, hipStreamSynchronize(c->stream));
    const int32_t none = 0;
    if (rank) {
        // rows up to a multiple of 16 ranks, zeros behind the last rank and behind K
        const int64_t r16 = (rank + 15) / 16 * 16;
        uint16_t *host = new (std::nothrow) uint16_t[(size_t)(r16 * std::max(a->KP, a->N))];
        if (!host) SV_FAIL(c, "adapters_load", "out of memory");
        memset(host, 0, (size_t)(r16 * a->KP) * 2);
        for (int r = 0; r < rank; r++) memcpy(host + r * a->KP, down + r * a->K, (size_t)a->K * 2);
        hipError_t e = hipMemcpy(a->rank + slot, &none, 4, hipMemcpyHostToDevice); // (a failed load leaves an empty slot)
        if (e == hipSuccess) e = hipMemcpy(a->down + (size_t)slot * a->RP * a->KP, host, (size_t)(r16 * a->KP) * 2, hipMemcpyHostToDevice);
        if (e == hipSuccess) {
            memset(host, 0, (size_t)(r16 * a->N) * 2);
            for (int64_t i = 0; i < a->N; i++) memcpy(host + i * r16, up + i * rank, (size_t)rank * 2);
            e = hipMemcpy(a->up + (size_t)slot * a->RP * a->N, host, (size_t)(r16 * a->N) * 2, hipMemcpyHostToDevice);
        }
        delete[] host;
        PS_CHECK(c, e);
        PS_CHECK(c, hipMemcpy(a->scale + slot, &scale, 4, hipMemcpyHostToDevice));
    }
    const int32_t now = rank;
    PS_CHECK(c, hipMemcpy(a->rank + slot, &now, 4, hipMemcpyHostToDevice));
    return 0;
}
size_t ps_hip_adapters_workspace(const ps_adapters *a, int T) {
    if (!a || T < 1) return 0;
    return psv_adapt_most(*a, T);
}
int ps_hip_adapters_apply(ps_hip_ctx *c, const ps_adapters *a, int x_dtype, const void *x, int64_t ldx, int T, const int32_t *ids, const float *base, float *out, int64_t ldo, void *ws, size_t bytes) {
    if (!c) return 2;
    if (!a || a->device != c->device) SV_FAIL(c, "adapters_apply", "no adapters, or another device's");
    if (x_dtype != PS_F32 && x_dtype != PS_BF16) SV_FAIL(c, "adapters_apply", "x must be F32 or BF16");
    if (T < 0 || T > (1 << 22)) SV_FAIL(c, "adapters_apply", "0 to 2^22 tokens");
    if (!T) return 0;
    if (!x || !ids || !out || !aligned(x, number_size(x_dtype)) || (const void *)out == x) SV_FAIL(c, "adapters_apply", "x, ids or out are missing, not aligned or the same");
    if (T > 1 && (ldx < a->K || ldo < a->N)) SV_FAIL(c, "adapters_apply", "rows overlap");
    if (!ws || !aligned(ws, 16) || bytes < psv_adapt_space(*a, x_dtype, nullptr, 0, T, nullptr, nullptr, nullptr, 0, nullptr, false, nullptr)) SV_FAIL(c, "adapters_apply", "the workspace is too small or not aligned");
    SV_DEVICE(c, "adapters_apply")
    psv_adapt_space(*a, x_dtype, x, ldx, T, ids, base, out, ldo, ws, true, c->stream);
    PS_CHECK(c, hipGetLastError());
    return 0;
}

} // extern "C"
