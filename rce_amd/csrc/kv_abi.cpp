// kv_abi.cpp -- the rce_qmm_kv_*, rce_qmm_rope_table and rce_qmm_sample_dev
// entry points (include/rce_qmm.h): argument checks in front of kv_cache.hip,
// kv_attention.hip and sample.hip.
#include "abi_internal.h"
#include "kv_cache.h"

#include <climits>
#include <cmath>

using namespace rce_qmm;
using namespace rce_qmm_abi;

namespace {

// The context's device for the call, the caller's again after it.
class OnDevice {
  public:
    explicit OnDevice(int device) {
        if (hipGetDevice(&before_) != hipSuccess) before_ = device;
        err_ = before_ == device ? hipSuccess : hipSetDevice(device);
        other_ = before_ != device;
    }
    ~OnDevice() {
        if (other_) (void)hipSetDevice(before_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
    hipError_t error() const { return err_; }

  private:
    int before_ = 0;
    bool other_ = false;
    hipError_t err_ = hipSuccess;
};

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

size_t value_bytes(uint32_t dtype) { return dtype == T_F32 ? 4 : dtype == T_F16 || dtype == T_BF16 ? 2 : 0; }

// kernels launch fewer than 2^32 threads
constexpr size_t MAX_WAVES = (size_t)1 << 26;

rce_qmm_status check_pool(const rce_qmm_kv_cache *c, KvPool &p) {
    if (!c) return fail(RCE_QMM_NULL_ARGUMENT, "null cache");
    const size_t pt = c->page_tokens, d = c->d_head;
    if (pt < 16 || pt > 4096 || (pt & (pt - 1)))
        return fail(RCE_QMM_BAD_SHAPE, "page_tokens must be a power of two from 16 to 4096");
    if (d != 64 && d != 128 && d != 192 && d != 256)
        return fail(RCE_QMM_BAD_SHAPE, "d_head must be 64, 128, 192 or 256");
    if (c->n_kv_heads == 0 || c->n_kv_heads > 65536) return fail(RCE_QMM_BAD_SHAPE, "n_kv_heads must be 1 to 65536");
    if (c->n_pages == 0 || c->n_pages > (size_t)INT_MAX) return fail(RCE_QMM_BAD_SHAPE, "n_pages must be 1 to 2^31 - 1");
    // blocks are numbered in 32 bits (at 64 dimensions 2^32 of them are 8 TiB)
    if (c->n_pages * c->n_kv_heads > (((size_t)1 << 32) - 1) / (pt / 16))
        return fail(RCE_QMM_BAD_SHAPE, "n_pages * n_kv_heads * page_tokens / 16 must be below 2^32");
    p.n_pages = (int)c->n_pages;
    p.heads = (int)c->n_kv_heads;
    p.lg_b = 0;
    while ((size_t)16 << p.lg_b < pt) p.lg_b++;
    p.k = c->k;
    p.v = c->v;
    p.k_scale = c->k_scale;
    p.v_scale = c->v_scale;
    return RCE_QMM_OK;
}

rce_qmm_status check_call(rce_qmm_context *ctx, const rce_qmm_kv_cache *c, const rce_qmm_kv_batch *b, KvPool &p,
                          KvRows &r) {
    if (!ctx) return fail(RCE_QMM_NULL_ARGUMENT, "null context");
    if (!b) return fail(RCE_QMM_NULL_ARGUMENT, "null batch");
    rce_qmm_status st = check_pool(c, p);
    if (st) return st;
    if (!p.k || !p.v || !p.k_scale || !p.v_scale) return fail(RCE_QMM_NULL_ARGUMENT, "null cache buffer");
    if (!aligned(p.k, 16) || !aligned(p.v, 16) || !aligned(p.k_scale, 4) || !aligned(p.v_scale, 4))
        return fail(RCE_QMM_BAD_SHAPE, "cache codes must be 16-byte aligned, scales 4");
    if (b->n_seqs > (size_t)1 << 20) return fail(RCE_QMM_BAD_SHAPE, "n_seqs must be at most 2^20");
    if (b->n_rows > (size_t)1 << 27) return fail(RCE_QMM_BAD_SHAPE, "n_rows must be at most 2^27");
    if (b->max_pages > ((size_t)INT_MAX - 4096) / c->page_tokens)
        return fail(RCE_QMM_BAD_SHAPE, "max_pages * page_tokens must stay below 2^31 - 4096");
    if (b->n_seqs && b->n_rows && b->max_pages) {
        if (!b->row_offsets || !b->seq_lens || !b->pages) return fail(RCE_QMM_NULL_ARGUMENT, "null batch array");
        if (!aligned(b->row_offsets, 4) || !aligned(b->seq_lens, 4) || !aligned(b->pages, 4))
            return fail(RCE_QMM_BAD_SHAPE, "batch arrays must be 4-byte aligned");
    }
    r = {b->row_offsets, b->seq_lens, b->pages, (int)b->n_seqs, (int)b->n_rows, (int)b->max_pages,
         (int)(b->max_pages * c->page_tokens)};
    return RCE_QMM_OK;
}

rce_qmm_status check_rope(const rce_qmm_rope *rope, size_t d_head, const KvRows &r, KvRope &out) {
    out = {nullptr, 0};
    if (!rope || rope->dim == 0) return RCE_QMM_OK;
    if (!rope->cs) return fail(RCE_QMM_NULL_ARGUMENT, "null rotation table");
    if (!aligned(rope->cs, 4)) return fail(RCE_QMM_BAD_SHAPE, "the rotation table must be 4-byte aligned");
    if (rope->dim % 2 || rope->dim > d_head) return fail(RCE_QMM_BAD_SHAPE, "rope dim must be even and at most d_head");
    if (rope->n_pos < (size_t)r.cap)
        return fail(RCE_QMM_BAD_SHAPE, "the rotation table has " + std::to_string(rope->n_pos) + " positions, the batch's tables span " +
                                           std::to_string(r.cap));
    out = {rope->cs, (int)(rope->dim / 2)};
    return RCE_QMM_OK;
}

rce_qmm_status check_rows(const char *what, const void *p, uint32_t dtype, size_t stride, size_t width) {
    const size_t b = value_bytes(dtype);
    if (!b) return fail(RCE_QMM_UNSUPPORTED_DTYPE, std::string(what) + " must be F32, F16 or BF16");
    if (!p) return fail(RCE_QMM_NULL_ARGUMENT, std::string("null ") + what);
    if (!aligned(p, b)) return fail(RCE_QMM_BAD_SHAPE, std::string(what) + " must be aligned to its values");
    if (stride < width) return fail(RCE_QMM_BAD_SHAPE, std::string(what) + ": rows overlap (stride " + std::to_string(stride) +
                                                           " below " + std::to_string(width) + ")");
    if (stride > ((size_t)1 << 40)) return fail(RCE_QMM_BAD_SHAPE, std::string(what) + ": stride above 2^40");
    return RCE_QMM_OK;
}

bool empty(const KvRows &r) { return !r.n_seqs || !r.n_rows; }

// Waves of the append's and the read's launch.
bool launchable(const KvPool &p, const KvRows &r) {
    return ((size_t)r.n_rows / 16 + 2 * (size_t)r.n_seqs) * p.heads * 2 <= MAX_WAVES ||
           (size_t)r.n_rows * p.heads * 2 <= MAX_WAVES;
}

// No C++ exception leaves a C entry point.
template <class F>
rce_qmm_status entry(F f) {
    try {
        return f();
    } catch (...) {
        return RCE_QMM_INTERNAL;
    }
}

}  // namespace

void rce_qmm_abi::fill_rope_table(float freq_base, size_t dim, size_t n_pos, float *cs) {
    const size_t half = dim / 2;
    const float log_base = logf(freq_base);
    for (size_t i = 0; i < half; i++) {
        float ex = log_base * (2.0f * (float)i);
        ex = ex / (float)dim;
        const float inv_freq = 1.0f / expf(ex);
        for (size_t p = 0; p < n_pos; p++) {
            const float theta = (float)p * inv_freq;
            cs[(p * half + i) * 2] = cosf(theta);
            cs[(p * half + i) * 2 + 1] = sinf(theta);
        }
    }
}

extern "C" {

rce_qmm_status rce_qmm_rope_table(float freq_base, size_t dim, size_t n_pos, float *cs) {
    return entry([&] {
        if (!cs && dim && n_pos) return fail(RCE_QMM_NULL_ARGUMENT, "null table");
        if (dim % 2 || dim > 65536 || n_pos > (size_t)INT_MAX)
            return fail(RCE_QMM_BAD_SHAPE, "dim must be even and at most 65536, n_pos below 2^31");
        if (!(freq_base > 0.0f) || !std::isfinite(freq_base)) return fail(RCE_QMM_BAD_SHAPE, "freq_base must be positive and finite");
        fill_rope_table(freq_base, dim, n_pos, cs);
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_kv_sizes(const rce_qmm_kv_cache *cache, size_t *code_bytes, size_t *n_scales) {
    return entry([&] {
        if (!code_bytes || !n_scales) return fail(RCE_QMM_NULL_ARGUMENT, "null argument");
        KvPool p;
        rce_qmm_status st = check_pool(cache, p);
        if (st) return st;
        *code_bytes = cache->n_pages * cache->n_kv_heads * cache->page_tokens * cache->d_head;
        *n_scales = cache->n_pages * cache->n_kv_heads * (cache->page_tokens / 16);
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_kv_append_dev(rce_qmm_context *ctx, const rce_qmm_kv_cache *cache,
                                     const rce_qmm_kv_batch *batch, const void *k_dev, size_t k_stride,
                                     const void *v_dev, size_t v_stride, uint32_t dtype, const rce_qmm_rope *rope,
                                     void *stream) {
    return entry([&] {
        KvPool p;
        KvRows r;
        KvRope ro;
        rce_qmm_status st;
        if ((st = check_call(ctx, cache, batch, p, r)) || (st = check_rope(rope, cache->d_head, r, ro))) return st;
        const size_t width = cache->n_kv_heads * cache->d_head;
        if (!value_bytes(dtype)) return fail(RCE_QMM_UNSUPPORTED_DTYPE, "keys and values must be F32, F16 or BF16");
        if (empty(r)) return RCE_QMM_OK;
        if ((st = check_rows("keys", k_dev, dtype, k_stride, width)) ||
            (st = check_rows("values", v_dev, dtype, v_stride, width)))
            return st;
        if (!r.cap) return RCE_QMM_OK;  // no table: every row is left out
        if (!launchable(p, r)) return fail(RCE_QMM_BAD_SHAPE, "too many rows and heads for one launch");
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
        HIP_TRY(launch_kv_append(p, r, (int)cache->d_head, k_dev, k_stride, v_dev, v_stride, dtype, ro, s));
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_kv_read_dev(rce_qmm_context *ctx, const rce_qmm_kv_cache *cache, const rce_qmm_kv_batch *batch,
                                   void *k_out, void *v_out, uint32_t dtype, void *stream) {
    return entry([&] {
        KvPool p;
        KvRows r;
        rce_qmm_status st = check_call(ctx, cache, batch, p, r);
        if (st) return st;
        const size_t width = cache->n_kv_heads * cache->d_head;
        if (!value_bytes(dtype)) return fail(RCE_QMM_UNSUPPORTED_DTYPE, "the values' dtype must be F32, F16 or BF16");
        if (empty(r) || !r.cap || (!k_out && !v_out)) return RCE_QMM_OK;
        if ((k_out && (st = check_rows("k_out", k_out, dtype, width, width))) ||
            (v_out && (st = check_rows("v_out", v_out, dtype, width, width))))
            return st;
        if (!launchable(p, r)) return fail(RCE_QMM_BAD_SHAPE, "too many rows and heads for one launch");
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
        HIP_TRY(launch_kv_read(p, r, (int)cache->d_head, k_out, v_out, dtype, s));
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_kv_attention_dev(rce_qmm_context *ctx, const rce_qmm_kv_cache *cache,
                                        const rce_qmm_kv_batch *batch, const void *q_dev, uint32_t q_dtype,
                                        size_t q_stride, size_t n_q_heads, const rce_qmm_rope *rope, float scale,
                                        size_t window, void *out_dev, uint32_t out_dtype, size_t out_stride,
                                        void *stream) {
    return entry([&] {
        KvPool p;
        KvRows r;
        KvAttention a{};
        rce_qmm_status st;
        if ((st = check_call(ctx, cache, batch, p, r)) || (st = check_rope(rope, cache->d_head, r, a.rope))) return st;
        if (n_q_heads == 0 || n_q_heads % cache->n_kv_heads || n_q_heads > (size_t)1 << 20)
            return fail(RCE_QMM_BAD_SHAPE, "n_q_heads must be a multiple of n_kv_heads");
        if (!(scale >= 0.0f) || !std::isfinite(scale)) return fail(RCE_QMM_BAD_SHAPE, "scale must be finite and not negative");
        if (!value_bytes(q_dtype) || !value_bytes(out_dtype))
            return fail(RCE_QMM_UNSUPPORTED_DTYPE, "queries and outputs must be F32, F16 or BF16");
        if (empty(r)) return RCE_QMM_OK;
        const size_t width = n_q_heads * cache->d_head;
        if ((st = check_rows("queries", q_dev, q_dtype, q_stride, width)) ||
            (st = check_rows("outputs", out_dev, out_dtype, out_stride, width)))
            return st;
        if (!r.cap) return fail(RCE_QMM_BAD_SHAPE, "max_pages must be at least 1");
        const size_t rows = (size_t)r.n_rows * n_q_heads;
        if (rows > (size_t)INT_MAX / 2 || (rows / 12 + ((size_t)r.n_seqs + 2) * p.heads + 4096) * 4 > MAX_WAVES)
            return fail(RCE_QMM_BAD_SHAPE, "too many rows and heads for one launch");
        a.q = q_dev;
        a.q_dtype = q_dtype;
        a.q_stride = q_stride;
        a.out = out_dev;
        a.out_dtype = out_dtype;
        a.out_stride = out_stride;
        a.n_q = (int)n_q_heads;
        a.window = window == 0 || window > (size_t)INT_MAX ? INT_MAX : (int)window;
        a.scale = scale;
        a.parts = static_cast<float *>(ctx->kv_parts.p);
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
        HIP_TRY(launch_kv_attention(p, r, (int)cache->d_head, a, s));
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_sample_dev(rce_qmm_context *ctx, const void *logits_dev, uint32_t dtype, size_t n_rows,
                                  size_t vocab, size_t row_stride, const rce_qmm_sampling *sampling, int32_t *ids_dev,
                                  float *probs_dev, void *stream) {
    return entry([&] {
        if (!ctx || !sampling) return fail(RCE_QMM_NULL_ARGUMENT, "null context or sampling");
        if (!value_bytes(dtype)) return fail(RCE_QMM_UNSUPPORTED_DTYPE, "logits must be F32, F16 or BF16");
        if (vocab == 0 || vocab > (size_t)1 << 24) return fail(RCE_QMM_BAD_SHAPE, "vocab must be 1 to 2^24");
        if (n_rows > (size_t)1 << 20) return fail(RCE_QMM_BAD_SHAPE, "n_rows must be at most 2^20");
        if (!n_rows) return RCE_QMM_OK;
        rce_qmm_status st = check_rows("logits", logits_dev, dtype, row_stride, vocab);
        if (st) return st;
        const rce_qmm_sampling &p = *sampling;
        if (!p.u || !ids_dev) return fail(RCE_QMM_NULL_ARGUMENT, "null u or ids");
        for (const void *x : {(const void *)p.u, (const void *)p.temperature, (const void *)p.top_k, (const void *)p.top_p,
                              (const void *)p.min_p, (const void *)ids_dev, (const void *)probs_dev})
            if (!aligned(x, 4)) return fail(RCE_QMM_BAD_SHAPE, "arrays of one value per row must be 4-byte aligned");
        const SampleRows r{logits_dev, dtype, n_rows, vocab, row_stride, p.u, p.temperature, p.top_p, p.min_p, p.top_k,
                           ids_dev, probs_dev, ctx->kv_parts.p};
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        HIP_TRY(launch_sample(r, stream ? static_cast<hipStream_t>(stream) : ctx->stream));
        return RCE_QMM_OK;
    });
}

}  // extern "C"
