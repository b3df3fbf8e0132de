// kv8.hip -- the 8-bit key / value cache: rows quantised as they are written, read back, and the attention over it (gfx950).
#include "q8.hpp"

using namespace wj;

namespace {

struct Kv8Args {
  wj_kv8 c;
  wj_kv8_batch b;
};

// What a sequence of the call owns.  first .. first + n - 1: its rows of the row arrays; pos0: position of the first of them
struct Span { int slot, first, n, len, pos0; };
__device__ __forceinline__ Span span_of(const Kv8Args& a, int b) {
  Span s;
  s.slot = a.b.slots_dev[b];
  s.first = a.b.starts_dev[b];
  const int last = min(a.b.starts_dev[b + 1], a.b.rows);
  if (s.first < 0) s.first = a.b.rows;                 // not a span of the arrays: no rows
  s.n = max(0, last - s.first);
  s.len = a.b.lens_dev[b];
  s.pos0 = s.len - s.n;
  if (s.slot < 0 || s.slot >= a.c.slots) s.slot = -1;
  return s;
}

// One wave per (row, head, K or V): the maximum over the lanes, then the codes.
__global__ __launch_bounds__(256) void kv8_write_kernel(const Kv8Args a, int dtype, const void* __restrict__ k, int64_t ldk,
                                                        const void* __restrict__ v, int64_t ldv) {
  const Span s = span_of(a, blockIdx.y);
  if (s.slot < 0) return;
  const int lane = threadIdx.x & 63, dim = a.c.dim, per = 2 * a.c.heads;
  const int64_t tasks = (int64_t)s.n * per;
  for (int64_t task = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); task < tasks; task += (int64_t)gridDim.x * 4) {
    const int t = (int)(task / per), which = (int)(task - (int64_t)t * per), head = which >> 1, pos = s.pos0 + t;
    if (pos < 0 || pos >= a.c.ctx) continue;
    const bool is_v = which & 1;
    const void* src = is_v ? v : k;
    const int64_t at = (int64_t)(s.first + t) * (is_v ? ldv : ldk) + head * dim;
    const int64_t row = ((int64_t)s.slot * a.c.heads + head) * a.c.ctx + pos;
    const float x0 = ld_any(src, dtype, at + lane), x1 = dim == 128 ? ld_any(src, dtype, at + 64 + lane) : 0.f;
    const RowQuant q(wave_max(fmaxf(mag(x0), mag(x1))));
    int8_t* codes = (is_v ? a.c.v_dev : a.c.k_dev) + row * dim;
    codes[lane] = (int8_t)q.code(x0);
    if (dim == 128) codes[64 + lane] = (int8_t)q.code(x1);
    if (lane == 0) (is_v ? a.c.v_scale_dev : a.c.k_scale_dev)[row] = q.scale;
  }
}

__global__ __launch_bounds__(256) void kv8_read_kernel(const Kv8Args a, int dtype, void* __restrict__ k, int64_t ldk, void* __restrict__ v,
                                                       int64_t ldv) {
  const Span s = span_of(a, blockIdx.y);
  const int lane = threadIdx.x & 63, dim = a.c.dim, per = 2 * a.c.heads;
  const int64_t tasks = (int64_t)s.n * per;
  for (int64_t task = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); task < tasks; task += (int64_t)gridDim.x * 4) {
    const int t = (int)(task / per), which = (int)(task - (int64_t)t * per), head = which >> 1, pos = s.pos0 + t;
    const bool is_v = which & 1, there = s.slot >= 0 && pos >= 0 && pos < a.c.ctx;
    const int64_t at = (int64_t)(s.first + t) * (is_v ? ldv : ldk) + head * dim;
    const int64_t row = there ? ((int64_t)s.slot * a.c.heads + head) * a.c.ctx + pos : 0;
    const int8_t* codes = (is_v ? a.c.v_dev : a.c.k_dev) + row * dim;
    const float scale = (is_v ? a.c.v_scale_dev : a.c.k_scale_dev)[row];
    for (int d = lane; d < dim; d += 64) st_any(is_v ? v : k, dtype, at + d, there ? (float)codes[d] * scale : 0.f);
  }
}

// One wave per (row, query head): 64 positions at a time, one per lane for the scores, then the dimensions over the lanes for the values.
__global__ __launch_bounds__(64) void kv8_attention_simple_kernel(const Kv8Args a, int dtype, const void* __restrict__ q, int64_t ldq,
                                                                  void* __restrict__ out, int64_t ldo, int n_heads, float scale, int causal) {
  __shared__ float qs[128], ps[64];
  const Span s = span_of(a, blockIdx.z);
  const int lane = threadIdx.x, head = blockIdx.y, kvh = head / (n_heads / a.c.heads), dim = a.c.dim;
  for (int t = blockIdx.x; t < s.n; t += gridDim.x) {
    const int64_t at = (int64_t)(s.first + t) * ldq + head * dim;
    __syncthreads();
    for (int d = lane; d < dim; d += 64) qs[d] = ld_any(q, dtype, at + d) * scale;
    const int keys = s.slot < 0 ? 0 : min(a.c.ctx, causal ? min(s.len, s.pos0 + t + 1) : s.len);
    const int64_t row0 = ((int64_t)max(s.slot, 0) * a.c.heads + kvh) * a.c.ctx;
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int base = 0; base < keys; base += 64) {
      __syncthreads();
      const bool in = base + lane < keys;
      const int64_t row = row0 + (in ? base + lane : 0);
      float dot = 0.f;
      for (int d = 0; d < dim; ++d) dot = fmaf(qs[d], (float)a.c.k_dev[row * dim + d], dot);
      const float sc = in ? dot * a.c.k_scale_dev[row] : -INFINITY;
      const float m_new = fmaxf(m, wave_max(sc));
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = expf(m - m_use), p = in ? expf(sc - m_use) : 0.f;
      l = l * alpha + wave_sum(p);
      m = m_new;
      ps[lane] = in ? p * a.c.v_scale_dev[row] : 0.f;
      __syncthreads();
      o0 *= alpha; o1 *= alpha;
      const int n = min(64, keys - base);
      for (int j = 0; j < n; ++j) {
        const int8_t* vr = a.c.v_dev + (row0 + base + j) * dim;
        o0 = fmaf(ps[j], (float)vr[lane], o0);
        if (dim == 128) o1 = fmaf(ps[j], (float)vr[64 + lane], o1);
      }
    }
    const int64_t to = (int64_t)(s.first + t) * ldo + head * dim;
    const float inv = keys > 0 ? 1.f / l : 0.f;
    st_any(out, dtype, to + lane, keys > 0 ? o0 * inv : 0.f);
    if (dim == 128) st_any(out, dtype, to + 64 + lane, keys > 0 ? o1 * inv : 0.f);
  }
}

int check_kv8(const char* who, wj_ctx* ctx, const wj_kv8* c, const wj_kv8_batch* b, int dtype) {
  WJ_REQUIRE(ctx && c && b, "%s: NULL argument", who);
  WJ_REQUIRE(known_dtype(dtype), "%s: unknown dtype %d", who, dtype);
  WJ_REQUIRE(c->dim == 64 || c->dim == 128, "%s: head dimension %d (64 and 128 are built)", who, c->dim);
  WJ_REQUIRE(c->slots >= 0 && c->ctx >= 0 && c->heads >= 1 && c->heads <= 65535, "%s: a cache of %d slots, %d heads, %d positions", who, c->slots, c->heads, c->ctx);
  WJ_REQUIRE(b->seqs >= 0 && b->seqs <= 65535 && b->rows >= 0 && b->max_new >= 0 && b->max_len >= 0, "%s: a batch of %d sequences (at most 65535), %d rows", who,
             b->seqs, b->rows);
  WJ_REQUIRE(b->seqs == 0 || (b->slots_dev && b->starts_dev && b->lens_dev), "%s: NULL batch array", who);
  const bool empty = (int64_t)c->slots * c->ctx == 0;
  WJ_REQUIRE(empty || (c->k_dev && c->k_scale_dev && c->v_dev && c->v_scale_dev), "%s: NULL cache array", who);
  WJ_REQUIRE(aligned_to(c->k_dev, 16) && aligned_to(c->v_dev, 16) && aligned_to(c->k_scale_dev, 4) && aligned_to(c->v_scale_dev, 4),
             "%s: the cache's codes are not 16-byte aligned (scales: 4)", who);
  return WJ_OK;
}

}  // namespace

extern "C" {

int wj_kv8_write(wj_ctx* ctx, const wj_kv8* cache, const wj_kv8_batch* batch, int dtype, const void* k_dev, int64_t ldk, const void* v_dev,
                 int64_t ldv, void* stream) {
  if (int rc = check_kv8("wj_kv8_write", ctx, cache, batch, dtype)) return rc;
  if (batch->seqs == 0 || batch->rows == 0 || (int64_t)cache->slots * cache->ctx == 0) return WJ_OK;
  WJ_REQUIRE(k_dev && v_dev, "wj_kv8_write: NULL argument");
  WJ_REQUIRE(ldk >= 0 && ldv >= 0, "wj_kv8_write: negative stride");
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  const int64_t tasks = (int64_t)(batch->max_new > 0 ? batch->max_new : 1) * 2 * cache->heads;
  const unsigned gx = (unsigned)(tasks + 3 < 4 * 4096 ? (tasks + 3) / 4 : 4096);
  hipLaunchKernelGGL(kv8_write_kernel, dim3(gx, batch->seqs), dim3(256), 0, ctx->pick(stream), Kv8Args{*cache, *batch}, dtype, k_dev, ldk, v_dev, ldv);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}

int wj_kv8_read(wj_ctx* ctx, const wj_kv8* cache, const wj_kv8_batch* batch, int dtype, void* k_dev, int64_t ldk, void* v_dev, int64_t ldv,
                void* stream) {
  if (int rc = check_kv8("wj_kv8_read", ctx, cache, batch, dtype)) return rc;
  if (batch->seqs == 0 || batch->rows == 0) return WJ_OK;
  WJ_REQUIRE((int64_t)cache->slots * cache->ctx > 0, "wj_kv8_read: an empty cache");
  WJ_REQUIRE(k_dev && v_dev, "wj_kv8_read: NULL argument");
  WJ_REQUIRE(batch->rows == 1 || (ldk >= cache->heads * cache->dim && ldv >= cache->heads * cache->dim), "wj_kv8_read: output rows overlap");
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  const int64_t tasks = (int64_t)(batch->max_new > 0 ? batch->max_new : 1) * 2 * cache->heads;
  const unsigned gx = (unsigned)(tasks + 3 < 4 * 4096 ? (tasks + 3) / 4 : 4096);
  hipLaunchKernelGGL(kv8_read_kernel, dim3(gx, batch->seqs), dim3(256), 0, ctx->pick(stream), Kv8Args{*cache, *batch}, dtype, k_dev, ldk, v_dev, ldv);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}

int64_t wj_kv8_attention_workspace(wj_ctx* ctx, const wj_kv8* cache, const wj_kv8_batch* batch, int n_heads) {
  (void)ctx; (void)cache; (void)batch; (void)n_heads;
  return 0;
}

int wj_kv8_attention(wj_ctx* ctx, const wj_kv8* cache, const wj_kv8_batch* batch, int dtype, const void* q_dev, int64_t ldq, void* out_dev,
                     int64_t ldo, int n_heads, float scale, int causal, void* workspace_dev, int64_t workspace_bytes, void* stream) {
  if (int rc = check_kv8("wj_kv8_attention", ctx, cache, batch, dtype)) return rc;
  WJ_REQUIRE(n_heads >= 1 && n_heads % cache->heads == 0 && n_heads / cache->heads <= 16, "wj_kv8_attention: %d query heads on %d key / value heads (a multiple, at most 16 each)",
             n_heads, cache->heads);
  if (batch->seqs == 0 || batch->rows == 0) return WJ_OK;
  WJ_REQUIRE((int64_t)cache->slots * cache->ctx > 0, "wj_kv8_attention: an empty cache");
  WJ_REQUIRE(q_dev && out_dev, "wj_kv8_attention: NULL argument");
  WJ_REQUIRE(ldq >= 0 && (batch->rows == 1 || ldo >= n_heads * cache->dim), "wj_kv8_attention: output rows overlap");
  WJ_REQUIRE(workspace_bytes >= wj_kv8_attention_workspace(ctx, cache, batch, n_heads), "wj_kv8_attention: workspace too small");
  DeviceScope dev;
  WJ_HIP(dev.enter(ctx->device));
  (void)workspace_dev;
  hipLaunchKernelGGL(kv8_attention_simple_kernel, dim3(batch->max_new > 0 ? batch->max_new : 1, n_heads, batch->seqs), dim3(64), 0, ctx->pick(stream),
                     Kv8Args{*cache, *batch}, dtype, q_dev, ldq, out_dev, ldo, n_heads, scale, causal);
  WJ_LAUNCH_CHECK();
  return WJ_OK;
}

}  // extern "C"
