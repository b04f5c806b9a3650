// kv_abi.cpp -- the serving step's entry points (include/rce_qmm.h: rce_qmm_kv_*,
// rce_qmm_rope_table*, rce_qmm_qk_norm_rope_dev, rce_qmm_moe_route_dev,
// rce_qmm_sample_dev): argument checks in front of kv_cache.hip,
// kv_attention.hip, kv_pages.hip, qk_rope.hip, moe_route.hip and sample.hip.
#include "abi_internal.h"
#include "kv_cache.h"
#include "kv_pages.h"
#include "moe_route.h"
#include "qk_rope.h"

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

rce_qmm_status check_pool_buffers(const KvPool &p) {
    if (!p.k || !p.v || !p.k_scale || !p.v_scale) return fail(RCE_QMM_NULL_ARGUMENT, "null cache buffer");
    if (!aligned(p.k, 16) || !aligned(p.v, 16) || !aligned(p.k_scale, 4) || !aligned(p.v_scale, 4))
        return fail(RCE_QMM_BAD_SHAPE, "cache codes must be 16-byte aligned, scales 4");
    return RCE_QMM_OK;
}

rce_qmm_status check_call(rce_qmm_context *ctx, const rce_qmm_kv_cache *c, const rce_qmm_kv_batch *b, KvPool &p,
                          KvRows &r) {
    if (!ctx) return fail(RCE_QMM_NULL_ARGUMENT, "null context");
    if (!b) return fail(RCE_QMM_NULL_ARGUMENT, "null batch");
    rce_qmm_status st = check_pool(c, p);
    if (st) return st;
    if ((st = check_pool_buffers(p))) return st;
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

// The arrays of a call on page tables; a null table is refused, an empty one comes back with no sequences.
rce_qmm_status check_table(const rce_qmm_kv_table *t, KvTable &out) {
    if (!t) return fail(RCE_QMM_NULL_ARGUMENT, "null table");
    if (t->n_seqs > (size_t)1 << 20) return fail(RCE_QMM_BAD_SHAPE, "n_seqs must be at most 2^20");
    if (t->max_pages > (size_t)INT_MAX || t->n_seqs * t->max_pages > (size_t)INT_MAX)
        return fail(RCE_QMM_BAD_SHAPE, "n_seqs * max_pages must be below 2^31");
    out = {t->pages, (int)t->n_seqs, (int)t->max_pages};
    if (!out.entries()) return RCE_QMM_OK;
    if (!t->pages) return fail(RCE_QMM_NULL_ARGUMENT, "null pages");
    if (!aligned(t->pages, 4)) return fail(RCE_QMM_BAD_SHAPE, "pages must be 4-byte aligned");
    return RCE_QMM_OK;
}

rce_qmm_status check_refs(const int32_t *refs) {
    if (!refs) return fail(RCE_QMM_NULL_ARGUMENT, "null refs");
    if (!aligned(refs, 4)) return fail(RCE_QMM_BAD_SHAPE, "refs must be 4-byte aligned");
    return RCE_QMM_OK;
}

rce_qmm_status check_each(const char *what, const int32_t *p, bool needed) {
    if (needed && !p) return fail(RCE_QMM_NULL_ARGUMENT, std::string("null ") + what);
    if (!aligned(p, 4)) return fail(RCE_QMM_BAD_SHAPE, std::string(what) + " must be 4-byte aligned");
    return RCE_QMM_OK;
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

rce_qmm_status attention(rce_qmm_context *ctx, const rce_qmm_kv_cache *cache, const rce_qmm_kv_batch *batch,
                         const void *q_dev, uint32_t q_dtype, size_t q_stride, size_t n_q_heads,
                         const rce_qmm_rope *rope, float scale, size_t window, size_t sinks, void *out_dev,
                         uint32_t out_dtype, size_t out_stride, void *stream) {
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
        // sinks that no window leaves behind are seen anyway
        a.sinks = a.window == INT_MAX ? 0 : sinks > (size_t)r.cap ? r.cap : (int)sinks;
        a.scale = scale;
        a.parts = static_cast<float *>(ctx->kv_parts.p);
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
        HIP_TRY(launch_kv_attention(p, r, (int)cache->d_head, a, s));
        return RCE_QMM_OK;
    });
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

rce_qmm_status rce_qmm_rope_table_scaled(float freq_base, size_t dim, size_t n_pos, const rce_qmm_rope_scaling *how, float *cs) {
    return entry([&] {
        if (!how || (!cs && dim && n_pos)) return fail(RCE_QMM_NULL_ARGUMENT, "null scaling or table");
        if (dim % 2 || dim > 65536 || n_pos > (size_t)INT_MAX)
            return fail(RCE_QMM_BAD_SHAPE, "dim must be even and at most 65536, n_pos below 2^31");
        auto positive = [](float x) { return x > 0.0f && std::isfinite(x); };
        if (!positive(freq_base)) return fail(RCE_QMM_BAD_SHAPE, "freq_base must be positive and finite");
        if (!positive(how->factor) || !positive(how->magnitude)) return fail(RCE_QMM_BAD_SHAPE, "factor and magnitude must be positive and finite");
        const bool ramp = how->orig_context != 0;
        if (ramp && (!positive(how->beta_fast) || !positive(how->beta_slow) || !(freq_base > 1.0f)))
            return fail(RCE_QMM_BAD_SHAPE, "beta_fast and beta_slow must be positive and finite, freq_base above 1");
        const size_t half = dim / 2;
        if (how->divisors)
            for (size_t i = 0; i < half; i++)
                if (!positive(how->divisors[i])) return fail(RCE_QMM_BAD_SHAPE, "divisors must be positive and finite");
        // the pair that turns `turns` times over the original context
        auto pair_of = [&](double turns) {
            return (double)dim * std::log((double)how->orig_context / (turns * 2 * M_PI)) / (2 * std::log((double)freq_base));
        };
        const double low = ramp ? std::max(0.0, std::floor(pair_of(how->beta_fast))) : 0.0;
        const double high = ramp ? std::min((double)dim - 1, std::ceil(pair_of(how->beta_slow))) : 0.0;
        for (size_t i = 0; i < half; i++) {
            double freq = std::pow((double)freq_base, -2.0 * (double)i / (double)dim);
            if (how->divisors) freq /= how->divisors[i];
            double keep = 0.0;  // share of the frequency that is not divided
            if (ramp) keep = 1.0 - std::min(1.0, std::max(0.0, ((double)i - low) / std::max(0.001, high - low)));
            freq = freq * keep + freq / how->factor * (1.0 - keep);
            for (size_t p = 0; p < n_pos; p++) {
                const double theta = (double)p * freq;
                cs[(p * half + i) * 2] = (float)(std::cos(theta) * how->magnitude);
                cs[(p * half + i) * 2 + 1] = (float)(std::sin(theta) * how->magnitude);
            }
        }
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
    return attention(ctx, cache, batch, q_dev, q_dtype, q_stride, n_q_heads, rope, scale, window, 0, out_dev, out_dtype, out_stride, stream);
}

rce_qmm_status rce_qmm_kv_attention_sinks_dev(rce_qmm_context *ctx, const rce_qmm_kv_cache *cache,
                                              const rce_qmm_kv_batch *batch, const void *q_dev, uint32_t q_dtype,
                                              size_t q_stride, size_t n_q_heads, const rce_qmm_rope *rope,
                                              float scale, size_t window, size_t sinks, void *out_dev,
                                              uint32_t out_dtype, size_t out_stride, void *stream) {
    return attention(ctx, cache, batch, q_dev, q_dtype, q_stride, n_q_heads, rope, scale, window, sinks, out_dev, out_dtype, out_stride, stream);
}

rce_qmm_status rce_qmm_kv_copy_dev(rce_qmm_context *ctx, const rce_qmm_kv_cache *from, const rce_qmm_kv_cache *to,
                                   const int32_t *src_dev, const int32_t *dst_dev, size_t n, void *stream) {
    return entry([&] {
        if (!ctx) return fail(RCE_QMM_NULL_ARGUMENT, "null context");
        KvPool a, b;
        rce_qmm_status st;
        if ((st = check_pool(from, a)) || (st = check_pool(to, b))) return st;
        if (from->page_tokens != to->page_tokens || a.heads != b.heads || from->d_head != to->d_head)
            return fail(RCE_QMM_BAD_SHAPE, "pages of the two pools differ in their shape");
        if ((st = check_pool_buffers(a)) || (st = check_pool_buffers(b))) return st;
        if (n > (size_t)INT_MAX) return fail(RCE_QMM_BAD_SHAPE, "n must be below 2^31");
        if (!n) return RCE_QMM_OK;
        if ((st = check_each("src", src_dev, true)) || (st = check_each("dst", dst_dev, true))) return st;
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
        HIP_TRY(launch_kv_copy(a, b, (int)from->d_head, src_dev, dst_dev, (int)n, s));
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_kv_fork_dev(rce_qmm_context *ctx, const rce_qmm_kv_cache *cache, const rce_qmm_kv_table *from,
                                   const rce_qmm_kv_table *to, const int32_t *parents_dev, int32_t *refs_dev, void *stream) {
    return entry([&] {
        if (!ctx) return fail(RCE_QMM_NULL_ARGUMENT, "null context");
        KvPool p;
        KvTable a, b;
        rce_qmm_status st;
        if ((st = check_pool(cache, p)) || (st = check_table(from, a)) || (st = check_table(to, b))) return st;
        if (!b.entries()) return RCE_QMM_OK;
        if ((st = check_each("parents", parents_dev, true)) || (st = check_refs(refs_dev))) return st;
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
        HIP_TRY(launch_kv_fork(a, b, parents_dev, {refs_dev, p.n_pages}, s));
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_kv_release_dev(rce_qmm_context *ctx, const rce_qmm_kv_cache *cache, const rce_qmm_kv_table *table,
                                      const int32_t *from_dev, const int32_t *to_dev, int32_t *refs_dev, void *stream) {
    return entry([&] {
        if (!ctx) return fail(RCE_QMM_NULL_ARGUMENT, "null context");
        KvPool p;
        KvTable t;
        rce_qmm_status st;
        if ((st = check_pool(cache, p)) || (st = check_table(table, t))) return st;
        if (!t.entries()) return RCE_QMM_OK;
        if ((st = check_each("from", from_dev, false)) || (st = check_each("to", to_dev, false)) || (st = check_refs(refs_dev))) return st;
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
        HIP_TRY(launch_kv_release(t, (int)cache->page_tokens, from_dev, to_dev, {refs_dev, p.n_pages}, s));
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_kv_reserve_dev(rce_qmm_context *ctx, const rce_qmm_kv_cache *cache, const rce_qmm_kv_batch *batch,
                                      int32_t *refs_dev, int32_t *missing_dev, void *stream) {
    return entry([&] {
        KvPool p;
        KvRows r;
        rce_qmm_status st;
        if ((st = check_call(ctx, cache, batch, p, r))) return st;
        if (!r.n_seqs) return RCE_QMM_OK;
        if ((st = check_each("missing", missing_dev, false)) || (st = check_refs(refs_dev))) return st;
        if (!r.n_rows || !r.cap) {  // no row touches a page; the arrays of the batch may be null
            r.n_rows = 0;
            if (!missing_dev) return RCE_QMM_OK;
        }
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
        HIP_TRY(launch_kv_reserve(p, r, (int)cache->d_head, const_cast<int32_t *>(r.pages), refs_dev, missing_dev, ctx->kv_parts.p, s));
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_kv_compact_dev(rce_qmm_context *ctx, const rce_qmm_kv_cache *cache, const rce_qmm_kv_table *table,
                                      int32_t *refs_dev, int32_t *new_ids_dev, int32_t *n_used_dev, void *stream) {
    return entry([&] {
        if (!ctx) return fail(RCE_QMM_NULL_ARGUMENT, "null context");
        KvPool p;
        KvTable t;
        rce_qmm_status st;
        if ((st = check_pool(cache, p)) || (st = check_table(table, t)) || (st = check_pool_buffers(p))) return st;
        if (cache->n_pages > KV_COMPACT_PAGES) return fail(RCE_QMM_BAD_SHAPE, "n_pages must be at most 2^23");
        if ((st = check_refs(refs_dev)) || (st = check_each("new_ids", new_ids_dev, true)) || (st = check_each("n_used", n_used_dev, false)))
            return st;
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        hipStream_t s = stream ? static_cast<hipStream_t>(stream) : ctx->stream;
        HIP_TRY(launch_kv_compact(p, (int)cache->d_head, t, refs_dev, new_ids_dev, n_used_dev, ctx->kv_parts.p, s));
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_qk_norm_rope_dev(rce_qmm_context *ctx, const rce_qmm_kv_batch *batch, const rce_qmm_heads *q,
                                        const rce_qmm_heads *k, size_t d_head, uint32_t in_dtype, uint32_t out_dtype,
                                        float eps, const rce_qmm_rope *rope, int interleaved, void *stream) {
    return entry([&] {
        if (!ctx || !batch) return fail(RCE_QMM_NULL_ARGUMENT, "null context or batch");
        if (d_head == 0 || d_head % 2 || d_head > QK_HEAD) return fail(RCE_QMM_BAD_SHAPE, "d_head must be even, 2 to 1024");
        if (eps != eps || eps == INFINITY) return fail(RCE_QMM_BAD_SHAPE, "eps must not be NaN or infinite");
        if (batch->n_seqs > (size_t)1 << 20) return fail(RCE_QMM_BAD_SHAPE, "n_seqs must be at most 2^20");
        if (batch->n_rows > (size_t)1 << 27) return fail(RCE_QMM_BAD_SHAPE, "n_rows must be at most 2^27");
        const size_t in_size = value_bytes(in_dtype), out_size = value_bytes(out_dtype);
        if (!in_size || !out_size) return fail(RCE_QMM_UNSUPPORTED_DTYPE, "heads must be F32, F16 or BF16");
        QkNormRope c{};
        c.rows = {batch->row_offsets, batch->seq_lens, nullptr, (int)batch->n_seqs, (int)batch->n_rows, 0, 0};
        rce_qmm_status st;
        if ((st = check_rope(rope, d_head, c.rows, c.rope))) return st;
        c.n_pos = c.rope.cs ? (int)std::min(rope->n_pos, (size_t)INT_MAX) : 0;
        if (empty(c.rows)) return RCE_QMM_OK;
        if (!batch->row_offsets || !batch->seq_lens) return fail(RCE_QMM_NULL_ARGUMENT, "null batch array");
        if (!aligned(batch->row_offsets, 4) || !aligned(batch->seq_lens, 4)) return fail(RCE_QMM_BAD_SHAPE, "batch arrays must be 4-byte aligned");
        for (int i = 0; i < 2; i++) {
            const rce_qmm_heads *h = i ? k : q;
            if (!h || !h->n_heads) continue;
            if (h->n_heads > (size_t)1 << 20) return fail(RCE_QMM_BAD_SHAPE, "n_heads must be at most 2^20");
            const size_t width = h->n_heads * d_head;
            if ((st = check_rows(i ? "key heads" : "query heads", h->in, in_dtype, h->in_stride, width)) ||
                (st = check_rows(i ? "key results" : "query results", h->out, out_dtype, h->out_stride, width)))
                return st;
            if (!aligned(h->weight, 4)) return fail(RCE_QMM_BAD_SHAPE, "weights must be 4-byte aligned");
            if (h->in == h->out && (in_size != out_size || h->in_stride != h->out_stride))
                return fail(RCE_QMM_BAD_SHAPE, "heads written in place need one type size and one stride");
            (i ? c.k : c.q) = {h->in, h->out, h->in_stride, h->out_stride, h->weight, (int)h->n_heads};
        }
        const size_t heads = (size_t)c.q.n + c.k.n;
        if (!heads) return RCE_QMM_OK;
        if (heads * batch->n_rows > MAX_WAVES) return fail(RCE_QMM_BAD_SHAPE, "too many rows and heads for one launch");
        c.d = (int)d_head;
        c.in_dtype = in_dtype;
        c.out_dtype = out_dtype;
        c.eps = eps < 0.0f ? -1.0f : eps;
        c.interleaved = interleaved != 0;
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        HIP_TRY(launch_qk_norm_rope(c, stream ? static_cast<hipStream_t>(stream) : ctx->stream));
        return RCE_QMM_OK;
    });
}

rce_qmm_status rce_qmm_moe_route_dev(rce_qmm_context *ctx, const void *logits_dev, uint32_t dtype, size_t n_tokens,
                                     size_t n_expert, size_t row_stride, const rce_qmm_moe_routing *how,
                                     int32_t *ids_dev, float *weights_dev, void *stream) {
    return entry([&] {
        if (!ctx || !how) return fail(RCE_QMM_NULL_ARGUMENT, "null context or routing");
        if (!value_bytes(dtype)) return fail(RCE_QMM_UNSUPPORTED_DTYPE, "logits must be F32, F16 or BF16");
        if (n_expert == 0 || n_expert > (size_t)ROUTE_EXPERTS) return fail(RCE_QMM_BAD_SHAPE, "n_expert must be 1 to 1024");
        if (n_tokens > (size_t)1 << 24) return fail(RCE_QMM_BAD_SHAPE, "n_tokens must be at most 2^24");
        if (how->top_k == 0 || how->top_k > n_expert || how->top_k > (size_t)ROUTE_TOP_K)
            return fail(RCE_QMM_BAD_SHAPE, "need 0 < top_k <= n_expert, top_k at most 64");
        if (how->scoring != RCE_QMM_SCORES_SOFTMAX && how->scoring != RCE_QMM_SCORES_SIGMOID)
            return fail(RCE_QMM_BAD_SHAPE, "scoring must be RCE_QMM_SCORES_SOFTMAX or RCE_QMM_SCORES_SIGMOID");
        const size_t groups = how->n_group ? how->n_group : 1;
        if (groups > (size_t)ROUTE_GROUPS || n_expert % groups) return fail(RCE_QMM_BAD_SHAPE, "n_group must divide n_expert and be at most 64");
        const size_t kept = groups == 1 ? 1 : how->topk_group;
        if (kept == 0 || kept > groups || how->top_k > kept * (n_expert / groups))
            return fail(RCE_QMM_BAD_SHAPE, "topk_group must be 1 to n_group, its experts top_k at least");
        if (kept < groups && how->group_top != 1 && how->group_top != 2) return fail(RCE_QMM_BAD_SHAPE, "group_top must be 1 or 2");
        if (!std::isfinite(how->scale)) return fail(RCE_QMM_BAD_SHAPE, "scale must be finite");
        if (!aligned(how->bias, 4)) return fail(RCE_QMM_BAD_SHAPE, "the bias must be 4-byte aligned");
        if (!n_tokens) return RCE_QMM_OK;
        rce_qmm_status st = check_rows("logits", logits_dev, dtype, row_stride, n_expert);
        if (st) return st;
        if ((st = check_each("ids", ids_dev, true))) return st;
        if (!weights_dev) return fail(RCE_QMM_NULL_ARGUMENT, "null weights");
        if (!aligned(weights_dev, 4)) return fail(RCE_QMM_BAD_SHAPE, "weights must be 4-byte aligned");
        const Routing r{logits_dev, dtype, row_stride, (int)n_tokens, (int)n_expert, (int)how->top_k, (int)groups, (int)kept,
                        (int)how->group_top, how->scoring == RCE_QMM_SCORES_SIGMOID, how->normalize != 0, how->scale, how->bias,
                        ids_dev, weights_dev};
        OnDevice dev(ctx->device);
        HIP_TRY(dev.error());
        HIP_TRY(launch_moe_route(r, stream ? static_cast<hipStream_t>(stream) : ctx->stream));
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
