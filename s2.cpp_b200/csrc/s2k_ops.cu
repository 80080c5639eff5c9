// s2k_ops.cu -- the C ABI of the operators on device memory (include/s2k.h):
// the 8-bit KV cache and the token log probabilities.  Checks of arguments,
// then one launch on the caller's stream.
#include "../../include/s2k.h"
#include "s2k_common.cuh"
#include "s2k_kv8.h"
#include "s2k_model.h"

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

namespace s2k {

static_assert(OT_F32 == S2K_TYPE_F32 && OT_F16 == S2K_TYPE_F16 && OT_BF16 == S2K_TYPE_BF16, "operator types");

namespace {

// Makes `device` current for the call and puts the caller's device back.
struct OnDevice {
    int before = -1;
    s2k_status enter(int device) {
        static std::atomic<int> count{0};
        int n = count.load(std::memory_order_relaxed);
        if (n == 0) {
            if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
                cudaGetLastError();
                return fail(S2K_ERR_NO_DEVICE, "no CUDA device");
            }
            count.store(n, std::memory_order_relaxed);
        }
        if (device < 0 || device >= n) return fail(S2K_ERR_ARG, "device %d out of range (%d devices)", device, n);
        int cur = -1;
        CU(cudaGetDevice(&cur));
        if (cur != device) {
            CU(cudaSetDevice(device));
            before = cur;
        }
        return S2K_OK;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

constexpr double kMaxExtent = (double)((int64_t)1 << 40);  // elements from a tensor's first to its last

int elem_size(int type) { return type == S2K_TYPE_F32 ? 4 : type == S2K_TYPE_F16 || type == S2K_TYPE_BF16 ? 2 : 0; }

s2k_status check_cache(const s2k_kv8 *c, int layer, Kv8 *out) {
    if (!c) return fail(S2K_ERR_ARG, "NULL cache");
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(S2K_ERR_UNSUPPORTED, "head_dim %d (64 or 128)", c->head_dim);
    if (c->n_pages <= 0 || c->n_layers <= 0 || c->n_kv_heads <= 0 || c->n_kv_heads > 4096)
        return fail(S2K_ERR_ARG, "cache of %d pages, %d layers, %d kv heads", c->n_pages, c->n_layers, c->n_kv_heads);
    if (layer < 0 || layer >= c->n_layers) return fail(S2K_ERR_ARG, "layer %d of %d", layer, c->n_layers);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(S2K_ERR_ARG, "NULL cache memory");
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16 || (uintptr_t)c->k_scale % 4 || (uintptr_t)c->v_scale % 4)
        return fail(S2K_ERR_ARG, "cache pages must be 16-byte aligned");
    out->k = c->k;
    out->v = c->v;
    out->k_scale = c->k_scale;
    out->v_scale = c->v_scale;
    out->n_pages = c->n_pages;
    out->n_layers = c->n_layers;
    out->n_kv_heads = c->n_kv_heads;
    out->head_dim = c->head_dim;
    out->layer = layer;
    return S2K_OK;
}

s2k_status check_rows(const s2k_kv8_rows *r, Kv8Rows *out) {
    if (!r) return fail(S2K_ERR_ARG, "NULL rows");
    if (r->n_seqs < 0 || r->n_rows < 0 || r->max_rows < 0 || r->max_rows > r->n_rows)
        return fail(S2K_ERR_ARG, "%d sequences, %d rows, at most %d each", r->n_seqs, r->n_rows, r->max_rows);
    if (!r->row_start && (int64_t)r->n_seqs * r->max_rows > r->n_rows)
        return fail(S2K_ERR_ARG, "%d sequences of %d rows, %d rows given", r->n_seqs, r->max_rows, r->n_rows);
    // positions are int32; a grid's x dimension holds every (sequence, 16 rows)
    if (r->table_ld <= 0 || r->table_ld > INT_MAX / kPage)
        return fail(S2K_ERR_ARG, "block table of %d entries per sequence", r->table_ld);
    if ((int64_t)r->n_seqs * ((int64_t)r->max_rows + 2) > INT_MAX || r->max_rows >= INT_MAX - kPage)
        return fail(S2K_ERR_ARG, "%d sequences of up to %d rows in one call", r->n_seqs, r->max_rows);
    if (r->n_seqs > 0 && (!r->past || !r->block_table)) return fail(S2K_ERR_ARG, "NULL past or block table");
    out->n_seqs = r->n_seqs;
    out->n_rows = r->n_rows;
    out->max_rows = r->max_rows;
    out->table_ld = r->table_ld;
    out->past = r->past;
    out->row_start = r->row_start;
    out->table = r->block_table;
    out->err = r->err;
    return S2K_OK;
}

// n_rows > 0 rows of n_heads heads; written: no two elements may coincide.
s2k_status check_heads(const char *what, const s2k_heads *t, const Kv8Rows &r, int n_heads, int hd, bool written,
                       Rows *out) {
    if (!t) return fail(S2K_ERR_ARG, "NULL %s", what);
    const int es = elem_size(t->type);
    if (!es) return fail(S2K_ERR_UNSUPPORTED, "%s of type %d (F32, F16 or BF16)", what, t->type);
    if (!t->data && r.n_rows > 0) return fail(S2K_ERR_ARG, "NULL %s", what);
    if ((uintptr_t)t->data % es) return fail(S2K_ERR_ARG, "%s is not aligned to its elements", what);
    if (t->row_stride < 0 || t->head_stride < 0) return fail(S2K_ERR_ARG, "%s has a negative stride", what);
    // no memory is that large, and every offset stays within 64 bits
    if ((double)t->row_stride * std::max(r.n_rows - 1, 0) + (double)t->head_stride * (n_heads - 1) > kMaxExtent)
        return fail(S2K_ERR_ARG, "%s reaches too far", what);
    if (written) {
        // [rows][heads][dim] or [heads][rows][dim], each with gaps or without
        const int64_t rs = t->row_stride, hs = t->head_stride;
        const bool by_row = (n_heads == 1 || hs >= hd) && (r.n_rows <= 1 || rs >= (n_heads - 1) * hs + hd);
        const bool by_head = (r.n_rows <= 1 || rs >= hd) && (n_heads == 1 || hs >= (r.n_rows - 1) * rs + hd);
        if (!by_row && !by_head) return fail(S2K_ERR_ARG, "rows of %s overlap", what);
    }
    out->p = t->data;
    out->type = t->type;
    out->row_stride = t->row_stride;
    out->head_stride = t->head_stride;
    return S2K_OK;
}

s2k_status launched(cudaError_t e, const char *what) {
    return e == cudaSuccess ? S2K_OK : fail(S2K_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace

}  // namespace s2k

using namespace s2k;

static s2k_status kv8_move(bool append, const s2k_kv8 *c, int32_t layer, const s2k_kv8_rows *r, const s2k_heads *k,
                           const s2k_heads *v, void *stream) {
    Kv8 cache;
    Kv8Rows rows;
    Rows kr, vr;
    s2k_status rc;
    if ((rc = check_cache(c, layer, &cache)) || (rc = check_rows(r, &rows)) ||
        (rc = check_heads("k", k, rows, c->n_kv_heads, c->head_dim, !append, &kr)) ||
        (rc = check_heads("v", v, rows, c->n_kv_heads, c->head_dim, !append, &vr)))
        return rc;
    if (k->type != v->type) return fail(S2K_ERR_ARG, "k and v have different types");
    OnDevice on;
    if ((rc = on.enter(c->device))) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    return launched(append ? launch_kv8_append(cache, rows, kr, vr, st) : launch_kv8_read(cache, rows, kr, vr, st),
                    append ? "s2k_kv8_append" : "s2k_kv8_read");
}

S2K_API s2k_status s2k_kv8_append(const s2k_kv8 *c, int32_t layer, const s2k_kv8_rows *r, const s2k_heads *k,
                                  const s2k_heads *v, void *stream) {
    return kv8_move(true, c, layer, r, k, v, stream);
}

S2K_API s2k_status s2k_kv8_read(const s2k_kv8 *c, int32_t layer, const s2k_kv8_rows *r, const s2k_heads *k,
                                const s2k_heads *v, void *stream) {
    return kv8_move(false, c, layer, r, k, v, stream);
}

S2K_API s2k_status s2k_kv8_attend(const s2k_kv8 *c, int32_t layer, const s2k_kv8_rows *r, const s2k_heads *q,
                                  const s2k_heads *out, int32_t n_heads, float scale, int32_t window, int32_t sinks,
                                  void *stream) {
    Kv8 cache;
    Kv8Rows rows;
    Kv8Attn a;
    s2k_status rc;
    if ((rc = check_cache(c, layer, &cache)) || (rc = check_rows(r, &rows))) return rc;
    if (n_heads <= 0 || n_heads > 65536 || n_heads % c->n_kv_heads)
        return fail(S2K_ERR_ARG, "%d query heads over %d kv heads", n_heads, c->n_kv_heads);
    if (!std::isfinite(scale)) return fail(S2K_ERR_ARG, "scale is not finite");
    if (window < 0 || sinks < 0) return fail(S2K_ERR_ARG, "window %d, sinks %d", window, sinks);
    if ((rc = check_heads("q", q, rows, n_heads, c->head_dim, false, &a.q)) ||
        (rc = check_heads("out", out, rows, n_heads, c->head_dim, true, &a.out)))
        return rc;
    if (q->type != out->type) return fail(S2K_ERR_ARG, "q and out have different types");
    a.n_heads = n_heads;
    a.scale = scale;
    a.window = window;
    a.sinks = sinks;
    OnDevice on;
    if ((rc = on.enter(c->device))) return rc;
    return launched(launch_kv8_attend(cache, rows, a, (cudaStream_t)stream), "s2k_kv8_attend");
}

S2K_API int32_t s2k_debug_kv8_attend_kernel(void) { return g_kv8_attend_kernel; }

S2K_API s2k_status s2k_logprobs(int32_t device, const void *logits, int32_t type, int32_t rows, int32_t n,
                                int64_t row_stride, const int32_t *targets, int32_t n_top, float *logprob,
                                float *entropy, int32_t *top_ids, float *top_logprobs, void *stream) {
    const int es = elem_size(type);
    if (!es) return fail(S2K_ERR_UNSUPPORTED, "logits of type %d (F32, F16 or BF16)", type);
    if (rows < 0 || n <= 0 || n > 1 << 30) return fail(S2K_ERR_ARG, "%d rows of %d logits", rows, n);
    if (row_stride < 0) return fail(S2K_ERR_ARG, "negative row stride");
    if ((double)row_stride * std::max(rows - 1, 0) + n > kMaxExtent) return fail(S2K_ERR_ARG, "logits reach too far");
    if (n_top < 0 || n_top > S2K_LOGPROBS_MAX_TOP || n_top > n)
        return fail(S2K_ERR_ARG, "%d alternatives of %d logits (at most %d)", n_top, n, S2K_LOGPROBS_MAX_TOP);
    if (rows > 0 && (!logits || (logprob && !targets) || (n_top > 0 && (!top_ids || !top_logprobs))))
        return fail(S2K_ERR_ARG, "NULL logits, targets or top outputs");
    if ((uintptr_t)logits % es) return fail(S2K_ERR_ARG, "logits are not aligned to their elements");
    LogprobArgs a;
    a.x = logits;
    a.type = type;
    a.rows = rows;
    a.n = n;
    a.ld = row_stride;
    a.targets = targets;
    a.n_top = n_top;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprob = top_logprobs;
    OnDevice on;
    s2k_status rc;
    if ((rc = on.enter(device))) return rc;
    return launched(launch_logprobs(a, (cudaStream_t)stream), "s2k_logprobs");
}
