// The C ABI of the decoder-side operators (include/we_b200.h): few-row products with 4-bit weights, the paged 4-bit
// K/V cache and its attention, and cross attention. Argument checks and dispatch; the kernels are in k_matvec.cu,
// k_kv4.cu and k_cross.cu.
#include <algorithm>
#include <cmath>
#include <string>

#include "common.cuh"
#include "kernels.h"

// defined in we_api.cu
int we_ctx_fail(we_ctx* ctx, int code, const std::string& msg);
cudaStream_t we_ctx_stream(we_ctx* ctx);
uint32_t* we_ctx_dev_err(we_ctx* ctx);
void we_ctx_count_launch(we_ctx* ctx);
int we_ctx_scratch_take(we_ctx* ctx, size_t bytes, void** out);  // from the buffer pool, to be given back once queued
void we_ctx_scratch_put(we_ctx* ctx, void* p);
uint32_t* we_ctx_counters(we_ctx* ctx, int64_t count);  // zeroed device words that every user leaves zero, or NULL

namespace {

#define DLK(call, what)                                                                                        \
  do {                                                                                                         \
    cudaError_t e_ = (call);                                                                                   \
    if (e_ != cudaSuccess) return we_ctx_fail(ctx, WE_ECUDA, std::string(what) + ": " + cudaGetErrorString(e_)); \
    we_ctx_count_launch(ctx);                                                                                  \
  } while (0)

// Most keys of a sequence: the kernels count places in 31 bits, up to some thousands past the last key.
constexpr int64_t MAX_KEYS = 0x7fffffff - (1 << 24);
bool act_dtype_ok(int dt) { return dt == WE_F32 || dt == WE_BF16; }
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
size_t dsize(int dt) { return dt == WE_F32 ? 4 : 2; }

int cache_check(we_ctx* ctx, const we_kv4_cache* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->page_table || !c->lengths)
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: missing cache buffer");
  if (c->dim != 64 && c->dim != 128 && c->dim != 256)
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: dim must be 64, 128 or 256, got " + std::to_string(c->dim));
  if (c->page <= 0 || c->page % 16)
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: page must be a multiple of 16 tokens, got " + std::to_string(c->page));
  if (c->batch < 0 || c->kv_heads <= 0 || c->pages < 0 || c->max_pages < 0)
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: batch, pages and max_pages must not be negative, kv_heads positive");
  if (c->batch > 65535 || c->kv_heads > 65535)
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: at most 65535 sequences and kv heads");
  if (c->pages > 0x7fffffff || c->max_pages > MAX_KEYS / c->page)
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: pages must fit 31 bits, tokens per sequence be at most " + std::to_string(MAX_KEYS));
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) ||
      !aligned(c->page_table, 4) || !aligned(c->lengths, 4))
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: k and v must be 16-byte, scales, page table and lengths 4-byte aligned");
  return WE_OK;
}

}  // namespace

extern "C" {

int we_matvec(we_ctx* ctx, const we_matmul_desc* d, const void* x, const void* w, void* y) {
  if (!ctx) return WE_EINVAL;
  int rc = we_matmul_check(ctx, d);
  if (rc != WE_OK) return rc;
  if (d->w_dtype != WE_INT4G64) return we_ctx_fail(ctx, WE_EINVAL, "matvec takes int4 group-64 weights");
  if (d->m < 1 || d->m > WE_MATVEC_MAX_ROWS)
    return we_ctx_fail(ctx, WE_EINVAL, "matvec takes 1 to " + std::to_string(WE_MATVEC_MAX_ROWS) + " rows, got " +
                                           std::to_string(d->m) + " (use we_matmul)");
  if (d->k_split > 1 || d->chan_scale) return we_ctx_fail(ctx, WE_EINVAL, "matvec takes neither kSplit nor channel scales");
  if (d->flags & ~(uint32_t)WE_MM_ACCUMULATE) return we_ctx_fail(ctx, WE_EINVAL, "matvec: unknown flag");
  if (d->x_stride < 0 || d->y_stride < 0 || d->x_offset < 0 || d->y_offset < 0)
    return we_ctx_fail(ctx, WE_EINVAL, "matvec: strides and offsets must not be negative");
  if ((d->x_stride && d->x_stride < d->k) || (d->y_stride && d->y_stride < d->n))
    return we_ctx_fail(ctx, WE_EINVAL, "matvec: a row stride is shorter than its row");
  if (d->n == 0) return WE_OK;
  if (!y || (d->k > 0 && (!x || !w))) return we_ctx_fail(ctx, WE_EINVAL, "matvec: missing operand");
  if (!aligned(w, 16)) return we_ctx_fail(ctx, WE_EINVAL, "matvec needs 16-byte aligned packed weights");
  if (!aligned(x, dsize(d->x_dtype)) || !aligned(y, dsize(d->y_dtype)) || !aligned(d->bias, 4) ||
      !aligned(d->epi.gate, 4) || (d->epi.aux_op && !aligned(d->epi.aux, dsize(d->epi.aux_dtype))))
    return we_ctx_fail(ctx, WE_EINVAL, "matvec: an operand is not aligned to its element size");
  if (d->n > 0x7fffffff || d->k > 0x7fffffff) return we_ctx_fail(ctx, WE_EINVAL, "matvec: n and k must fit 31 bits");
  we::MatmulArgs a{};
  a.m = d->m;
  a.n = d->n;
  a.k = d->k;
  a.x_stride = d->x_stride ? d->x_stride : d->k;
  a.y_stride = d->y_stride ? d->y_stride : d->n;
  a.x_offset = d->x_offset;
  a.y_offset = d->y_offset;
  a.group_scale = d->group_scale;
  a.bias = d->bias;
  a.x_dtype = d->x_dtype;
  a.y_dtype = d->y_dtype;
  a.accumulate = (d->flags & WE_MM_ACCUMULATE) ? 1 : 0;
  a.epi.act = d->epi.act;
  a.epi.aux_op = d->epi.aux_op;
  a.epi.aux_dtype = d->epi.aux_dtype;
  a.epi.aux = d->epi.aux_op ? static_cast<const char*>(d->epi.aux) + a.y_offset * dsize(d->epi.aux_dtype) : nullptr;
  a.epi.gate = d->epi.gate;
  const char* xp = static_cast<const char*>(x) + a.x_offset * dsize(a.x_dtype);
  char* yp = static_cast<char*>(y) + a.y_offset * dsize(a.y_dtype);
  DLK(we::launch_matvec(xp, w, yp, a, we_num_sms(ctx), we_ctx_stream(ctx)), "matvec");
  return WE_OK;
}

int we_kv4_append(we_ctx* ctx, const we_kv4_cache* c, const void* k, const void* v, int32_t dtype, int64_t tokens,
                  int64_t stride) {
  if (!ctx) return WE_EINVAL;
  int rc = cache_check(ctx, c);
  if (rc != WE_OK) return rc;
  if (!act_dtype_ok(dtype)) return we_ctx_fail(ctx, WE_EINVAL, "kv4: k and v must be f32 or bf16");
  if (tokens < 0 || tokens > 0x7fffffff) return we_ctx_fail(ctx, WE_EINVAL, "kv4: tokens must be in 0..2^31-1");
  if (stride && stride < c->kv_heads * c->dim)
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: the token stride is shorter than a token's heads");
  if (tokens == 0 || c->batch == 0) return WE_OK;
  if (!k || !v) return we_ctx_fail(ctx, WE_EINVAL, "kv4: missing k or v");
  if (!aligned(k, dsize(dtype)) || !aligned(v, dsize(dtype)))
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: k and v must be aligned to their element size");
  DLK(we::launch_kv4_append(*c, k, v, dtype, tokens, stride ? stride : c->kv_heads * c->dim, we_ctx_dev_err(ctx),
                            we_num_sms(ctx), we_ctx_stream(ctx)),
      "kv4 append");
  return WE_OK;
}

int we_kv4_unpack(we_ctx* ctx, const we_kv4_cache* c, void* k, void* v, int32_t dtype, int64_t tokens,
                  const int32_t* start) {
  if (!ctx) return WE_EINVAL;
  int rc = cache_check(ctx, c);
  if (rc != WE_OK) return rc;
  if (!act_dtype_ok(dtype)) return we_ctx_fail(ctx, WE_EINVAL, "kv4: k and v must be f32 or bf16");
  if (tokens < 0 || tokens > 0x7fffffff) return we_ctx_fail(ctx, WE_EINVAL, "kv4: tokens must be in 0..2^31-1");
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(start, 4))
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: unpacked k and v must be 16-byte aligned");
  if (tokens == 0 || c->batch == 0 || (!k && !v)) return WE_OK;
  DLK(we::launch_kv4_unpack(*c, k, v, dtype, tokens, start, we_ctx_dev_err(ctx), we_num_sms(ctx), we_ctx_stream(ctx)),
      "kv4 unpack");
  return WE_OK;
}

int we_kv4_attention(we_ctx* ctx, const we_kv4_cache* c, const void* q, int32_t dtype, int64_t tokens, int64_t heads,
                     int64_t q_stride, float scale, void* out, int32_t out_dtype, int64_t out_stride) {
  if (!ctx) return WE_EINVAL;
  int rc = cache_check(ctx, c);
  if (rc != WE_OK) return rc;
  if (!act_dtype_ok(dtype) || !act_dtype_ok(out_dtype))
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: q and out must be f32 or bf16");
  if (heads <= 0 || heads % c->kv_heads) return we_ctx_fail(ctx, WE_EINVAL, "heads must be a multiple of kvHeads");
  if (tokens < 0 || tokens > 0x7fffffff / heads) return we_ctx_fail(ctx, WE_EINVAL, "kv4: tokens * heads must be in 0..2^31-1");
  if ((q_stride && q_stride < heads * c->dim) || (out_stride && out_stride < heads * c->dim))
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: a token stride is shorter than a token's heads");
  if (!std::isfinite(scale)) return we_ctx_fail(ctx, WE_EINVAL, "kv4: scale must be finite");
  if (tokens == 0 || c->batch == 0) return WE_OK;
  if (!q || !out) return we_ctx_fail(ctx, WE_EINVAL, "kv4: missing q or out");
  if (!aligned(q, dsize(dtype)) || !aligned(out, dsize(out_dtype)))
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: q and out must be aligned to their element size");
  we::Kv4AttnArgs a{*c,
                    q,
                    out,
                    tokens,
                    heads,
                    q_stride ? q_stride : heads * c->dim,
                    out_stride ? out_stride : heads * c->dim,
                    scale != 0.f ? scale : 1.f / sqrtf((float)c->dim),
                    dtype,
                    out_dtype};
  int64_t part_bytes, units;
  we::kv4_attention_scratch(a, we_num_sms(ctx), &part_bytes, &units);
  if (heads / c->kv_heads * tokens > 0x7fffffff / 16 || a.c.kv_heads * ((heads / c->kv_heads * tokens + 7) / 8) > 65535)
    return we_ctx_fail(ctx, WE_EINVAL, "kv4: too many query rows in one call");
  void* part = nullptr;
  uint32_t* done = nullptr;
  if (units > 0) {
    done = we_ctx_counters(ctx, units);
    if (!done) return we_ctx_fail(ctx, WE_EINVAL, "kv4: too many sequences and heads to split in one call");
    if ((rc = we_ctx_scratch_take(ctx, (size_t)part_bytes, &part)) != WE_OK) return rc;
  }
  const cudaError_t e = we::launch_kv4_attention(a, part, done, we_ctx_dev_err(ctx), we_num_sms(ctx), we_ctx_stream(ctx));
  if (part) we_ctx_scratch_put(ctx, part);
  DLK(e, "kv4 attention");
  return WE_OK;
}

int we_kv4_advance(we_ctx* ctx, const we_kv4_cache* c, int64_t tokens) {
  if (!ctx) return WE_EINVAL;
  int rc = cache_check(ctx, c);
  if (rc != WE_OK) return rc;
  if (tokens < 0 || tokens > 0x7fffffff) return we_ctx_fail(ctx, WE_EINVAL, "kv4: tokens must be in 0..2^31-1");
  if (tokens == 0 || c->batch == 0) return WE_OK;
  DLK(we::launch_kv4_advance(*c, tokens, we_ctx_stream(ctx)), "kv4 advance");
  return WE_OK;
}

int we_cross_attention(we_ctx* ctx, const we_cross_desc* desc) {
  if (!ctx) return WE_EINVAL;
  if (!desc) return we_ctx_fail(ctx, WE_EINVAL, "cross attention: no description");
  we_cross_desc d = *desc;
  if (!act_dtype_ok(d.dtype) || !act_dtype_ok(d.out_dtype))
    return we_ctx_fail(ctx, WE_EINVAL, "cross attention: q/k/v and out must be f32 or bf16");
  if (d.kv_heads <= 0 || d.heads <= 0 || d.heads % d.kv_heads)
    return we_ctx_fail(ctx, WE_EINVAL, "heads must be a multiple of kvHeads");
  if (d.dim <= 0 || d.dim > 256) return we_ctx_fail(ctx, WE_EINVAL, "dim must be in 1..256");
  if (d.batch < 0 || d.tq < 0 || d.tk < 0) return we_ctx_fail(ctx, WE_EINVAL, "cross attention: negative size");
  if (d.batch > 65535 || d.heads > 65535 || d.tq > MAX_KEYS || d.tk > MAX_KEYS)
    return we_ctx_fail(ctx, WE_EINVAL, "cross attention: at most 65535 batch entries and heads, " + std::to_string(MAX_KEYS) + " tokens");
  const int64_t qw = d.heads * d.dim, kw = d.kv_heads * d.dim;
  if ((d.q_stride && d.q_stride < qw) || (d.out_stride && d.out_stride < qw) || (d.k_stride && d.k_stride < kw) ||
      (d.v_stride && d.v_stride < kw))
    return we_ctx_fail(ctx, WE_EINVAL, "cross attention: a token stride is shorter than a token's heads");
  if (!std::isfinite(d.scale)) return we_ctx_fail(ctx, WE_EINVAL, "cross attention: scale must be finite");
  if (d.batch == 0 || d.tq == 0) return WE_OK;
  if (!d.q || !d.out || (d.tk > 0 && (!d.k || !d.v)))
    return we_ctx_fail(ctx, WE_EINVAL, "cross attention: missing buffer");
  const size_t es = dsize(d.dtype);
  if (!aligned(d.q, es) || !aligned(d.k, es) || !aligned(d.v, es) || !aligned(d.out, dsize(d.out_dtype)) ||
      !aligned(d.key_lengths, 4))
    return we_ctx_fail(ctx, WE_EINVAL, "cross attention: a buffer is not aligned to its element size");
  if (!d.q_stride) d.q_stride = qw;
  if (!d.out_stride) d.out_stride = qw;
  if (!d.k_stride) d.k_stride = kw;
  if (!d.v_stride) d.v_stride = kw;
  if (d.scale == 0.f) d.scale = 1.f / sqrtf((float)d.dim);
  const int64_t group = d.heads / d.kv_heads;
  if (d.tq > 0x7fffffff / group) return we_ctx_fail(ctx, WE_EINVAL, "cross attention: tq * heads / kv_heads must fit 31 bits");
  // From 9 rows (tokens x heads of a group) on the tcgen05 kernel: its steps cost the same for 1 to 128 rows, the tiles' for
  // 1 to 8. us, tiles / tcgen05: 8 x 4096 keys, 24 heads, 8 rows 73.7 / 80.7, 9 rows 93.0 / 80.9; 4 x 1500 keys, 4 groups of
  // 4 heads, 8 rows 10.1 / 11.4, 16 rows 19.1 / 12.6. Calls of few heads and many keys would take tiles up to 16 rows: 2 x 512
  // keys, 16 heads, 9 rows 8.5 / 9.5 (dim 64: 6.9 / 8.6), 1500 keys 10.9 / 13.9 (8.5 / 12.3), 77 keys 8.1 / 7.2 (6.4 / 6.3), and
  // with 32 rows 15.8 / 11.4, 21.3 / 15.4 and 14.7 / 7.3.
  if (d.tq * group >= 9 && we::cross_flash_supported(d)) {
    const cudaError_t e = we::launch_cross_flash(d, we_ctx_dev_err(ctx), we_num_sms(ctx), we_ctx_stream(ctx));
    if (e != cudaErrorNotSupported) {
      DLK(e, "cross attention");
      return WE_OK;
    }
  }
  // a call of many query rows goes in pieces whose tiles fit a grid
  const int64_t most = std::max<int64_t>(1, 65535 / d.kv_heads * 8 / group);
  const we_cross_desc whole = d;
  for (int64_t b = 0; b < (whole.tq > most ? whole.batch : 1); b++)
    for (int64_t t = 0; t < whole.tq; t += most) {
      if (whole.tq > most) {  // then entry by entry: a piece's rows follow each other
        d = whole;
        d.batch = 1;
        d.tq = std::min(most, whole.tq - t);
        d.q = static_cast<const char*>(whole.q) + (b * whole.tq + t) * whole.q_stride * es;
        d.out = static_cast<char*>(whole.out) + (b * whole.tq + t) * whole.out_stride * dsize(d.out_dtype);
        d.k = static_cast<const char*>(whole.k) + b * whole.tk * whole.k_stride * es;
        d.v = static_cast<const char*>(whole.v) + b * whole.tk * whole.v_stride * es;
        if (whole.key_lengths) d.key_lengths = whole.key_lengths + b;
        if (whole.key_mask) d.key_mask = whole.key_mask + b * whole.tk;
      }
      int64_t part_bytes, units, grid_y;
      we::cross_tile_scratch(d, we_num_sms(ctx), &part_bytes, &units, &grid_y);
      if (grid_y > 65535) return we_ctx_fail(ctx, WE_EINVAL, "cross attention: too many heads in one call");
      void* part = nullptr;
      uint32_t* done = nullptr;
      if (units > 0) {
        done = we_ctx_counters(ctx, units);
        if (!done) return we_ctx_fail(ctx, WE_EINVAL, "cross attention: too many rows to split in one call");
        int rc = we_ctx_scratch_take(ctx, (size_t)part_bytes, &part);
        if (rc != WE_OK) return rc;
      }
      const cudaError_t e = we::launch_cross_tile(d, part, done, we_num_sms(ctx), we_ctx_stream(ctx));
      if (part) we_ctx_scratch_put(ctx, part);
      DLK(e, "cross attention");
    }
  return WE_OK;
}

}  // extern "C"
