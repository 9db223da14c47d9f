// C entry points of the sequence operators (include/ivh.h): every argument that the host can see
// is checked before anything is enqueued.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "../../include/ivh.h"
#include "capi_guard.hpp"
#include "seq_ops.hpp"

namespace {

using ivh::check_launch;
using ivh::guard;

constexpr float kLog2E = 1.4426950408889634f;

void need(bool ok, const char * what)
{
  if (!ok) throw std::invalid_argument(what);
}

void check_type(int type) { need(type == IVH_F16 || type == IVH_BF16, "type must be IVH_F16 or IVH_BF16"); }

// Operands are device memory of the current device, and the stream is one of its own: a kernel
// that reads another GPU's memory, or pageable host memory, faults.
void check_device(void * stream, std::initializer_list<const void *> ptrs)
{
  auto chk = [](hipError_t e) {
    if (e != hipSuccess) throw std::runtime_error(std::string("HIP error: ") + hipGetErrorString(e));
  };
  int dev = 0;
  chk(hipGetDevice(&dev));
  if (stream) {
    hipDevice_t own = 0;
    chk(hipStreamGetDevice(static_cast<hipStream_t>(stream), &own));
    need(own == dev, "the stream belongs to another device than the current one");
  }
  for (const void * p : ptrs) {
    if (!p) continue;
    hipPointerAttribute_t a;
    if (hipPointerGetAttributes(&a, p) != hipSuccess) {
      (void)hipGetLastError();
      throw std::invalid_argument("an operand is not device memory");
    }
    need(a.type != hipMemoryTypeUnregistered, "an operand is not device memory");
    need(a.type == hipMemoryTypeHost || a.device == dev, "an operand lies on another device than the current one");
  }
}

// rows of `dim` elements that start at multiples of `elems` elements
void check_rows(const void * ptr, int64_t token, int64_t head, int elems, const char * what)
{
  if (!ptr) throw std::invalid_argument(std::string(what) + ": null operand");
  if (token < 0 || head < 0 || token % elems || head % elems || reinterpret_cast<uintptr_t>(ptr) % (2 * elems))
    throw std::invalid_argument(std::string(what) + ": rows must start at multiples of " + std::to_string(2 * elems) + " bytes");
}

// output rows do not overlap
void check_apart(int64_t tokens, int64_t heads, int64_t dim, int64_t token, int64_t head, const char * what)
{
  const bool inner = (heads == 1 || head >= dim) && (tokens == 1 || token >= (heads - 1) * head + dim);
  const bool outer = (tokens == 1 || token >= dim) && (heads == 1 || head >= (tokens - 1) * token + dim);
  if (tokens > 0 && !inner && !outer) throw std::invalid_argument(std::string(what) + ": output rows overlap");
}

ivh::RotParams rotation(const ivh_rotation & r, int dim, const int32_t * pos, int64_t pos_axis, const float * freq, bool may_be_none)
{
  ivh::RotParams o;
  if (may_be_none && r.rot == 0) return o;
  need(r.rot >= 8 && r.rot <= dim && r.rot % 8 == 0, "rotation: rot must be a multiple of 8, at most dim");
  need(r.axes >= 1 && r.axes <= 4, "rotation: 1 to 4 axes");
  int64_t sum = 0;
  for (int i = 0; i < 4; ++i) {
    need(r.section[i] >= 0 && (i < r.axes || r.section[i] == 0), "rotation: bad section");
    sum += r.section[i];
  }
  need(sum == r.rot / 2, "rotation: the axes' sections must sum to rot / 2");
  need(pos_axis >= 0, "rotation: bad stride of positions");
  need(pos && freq, "rotation: null positions or frequencies");
  need(reinterpret_cast<uintptr_t>(pos) % 4 == 0 && reinterpret_cast<uintptr_t>(freq) % 4 == 0, "rotation: misaligned positions or frequencies");
  o.rot = r.rot;
  o.half = r.rot / 2;
  o.axes = r.axes;
  for (int i = 0; i < 4; ++i) o.sec[i] = r.section[i];
  o.adjacent = r.adjacent != 0;
  o.dealt = r.dealt != 0;
  o.pos = pos;
  o.pos_axis = pos_axis;
  o.freq = freq;
  return o;
}

constexpr int kMaxTokens = 1 << 26, kMaxBatch = 1 << 20, kMaxHeads = 1 << 22;  // the last: sequences times heads
// of contiguous rows: a larger window hides nothing either; with it a place less the window stays within 32 bits
constexpr int kMaxWindow = INT32_MAX - 2 * kMaxTokens;

void check_counts(int batch, int tokens)
{
  need(batch >= 0 && batch <= kMaxBatch, "batch must be in [0, 2^20]");
  need(tokens >= 0 && tokens <= kMaxTokens, "tokens must be in [0, 2^26]");
}

ivh::CacheParams cache(const ivh_cache_desc & d)
{
  check_type(d.type);
  need(d.bits == 8 || d.bits == 16, "cache: bits must be 8 or 16");
  need(d.heads >= 1 && d.heads <= 4096, "cache: heads must be in [1, 4096]");
  need(d.dim >= 16 && d.dim <= 256 && d.dim % 16 == 0, "cache: dim must be a multiple of 16, at most 256");
  need(d.page == 16 || d.page == 32 || d.page == 64 || d.page == 128, "cache: page must be 16, 32, 64 or 128 tokens");
  need(d.pages >= 1 && d.table_width >= 1, "cache: no pages");
  need((int64_t)d.table_width * d.page <= (1LL << 30), "cache: a sequence holds at most 2^30 tokens");
  ivh::CacheParams c;
  c.type = d.type;
  c.bits = d.bits;
  c.heads = d.heads;
  c.dim = d.dim;
  c.page = d.page;
  c.pages = d.pages;
  c.width = d.table_width;
  return c;
}

void bind(ivh::CacheParams & c, const void * kc, const void * vc, const float * ks, const float * vs, const int32_t * cu,
          const int32_t * lens, const int32_t * table, int batch, int tokens)
{
  need(kc && vc && cu && lens && table, "cache: null operand");
  need(c.bits == 16 || (ks && vs), "cache: 8-bit pages need their scales");
  need(reinterpret_cast<uintptr_t>(kc) % 16 == 0 && reinterpret_cast<uintptr_t>(vc) % 16 == 0, "cache: pages must start at multiples of 16 bytes");
  need((reinterpret_cast<uintptr_t>(cu) | reinterpret_cast<uintptr_t>(lens) | reinterpret_cast<uintptr_t>(table) |
        reinterpret_cast<uintptr_t>(ks) | reinterpret_cast<uintptr_t>(vs)) % 4 == 0, "cache: misaligned operand");
  c.kc = const_cast<void *>(kc);
  c.vc = const_cast<void *>(vc);
  c.ks = const_cast<float *>(ks);
  c.vs = const_cast<float *>(vs);
  c.cu = cu;
  c.lens = lens;
  c.table = table;
  c.batch = batch;
  c.tokens = tokens;
}

ivh::PagedParams paged(const ivh_paged_attn_desc * d, int batch, int tokens, size_t * bytes)
{
  need(d, "null descriptor");
  ivh::PagedParams p;
  p.c = cache(d->cache);
  check_counts(batch, tokens);
  need(d->heads >= 1 && d->heads % d->cache.heads == 0, "heads must be a multiple of the cache's heads");
  need((int64_t)tokens * d->heads <= kMaxTokens && (int64_t)batch * d->cache.heads <= kMaxHeads, "too many rows for a call");
  need(std::isfinite(d->scale * kLog2E), "scale must be finite");
  need(d->window >= 0 && d->sinks >= 0, "window and sinks must not be negative");
  need(d->max_new >= 0 && d->max_len >= 0, "max_new and max_len must not be negative");
  p.c.batch = batch;
  p.c.tokens = tokens;
  p.heads = d->heads;
  p.group = d->heads / d->cache.heads;
  p.scale_log2 = d->scale * kLog2E;
  p.window = d->window;
  p.sinks = d->sinks;
  const int max_new = d->max_new ? d->max_new : tokens;
  const int max_len = d->max_len ? d->max_len : d->cache.table_width * d->cache.page;
  *bytes = batch && tokens ? ivh::paged_split(p, max_new, max_len) : 0;
  return p;
}

}  // namespace

extern "C" {

int ivh_rope(const ivh_rope_desc * d, const void * x, const int32_t * pos, const float * freq, void * y, int tokens, void * stream)
{
  return guard([&] {
    need(d, "null descriptor");
    check_type(d->type);
    need(tokens >= 0 && tokens <= kMaxTokens, "tokens must be in [0, 2^26]");
    need(d->heads >= 1 && d->heads <= 4096, "heads must be in [1, 4096]");
    need(d->dim >= 8 && d->dim <= 1024 && d->dim % 8 == 0, "dim must be a multiple of 8, at most 1024");
    if (tokens == 0) return;
    ivh::RopeParams p;
    p.r = rotation(d->rotation, d->dim, pos, d->pos_axis, freq, false);
    check_rows(x, d->x_token, d->x_head, 4, "rope input");
    check_rows(y, d->y_token, d->y_head, 4, "rope output");
    check_apart(tokens, d->heads, d->dim, d->y_token, d->y_head, "rope");
    check_device(stream, {x, pos, freq, y});
    p.type = d->type;
    p.heads = d->heads;
    p.dim = d->dim;
    p.tokens = tokens;
    p.x = x;
    p.y = y;
    p.x_token = d->x_token;
    p.x_head = d->x_head;
    p.y_token = d->y_token;
    p.y_head = d->y_head;
    ivh::launch_rope(p, static_cast<hipStream_t>(stream));
    check_launch("rope");
  });
}

int ivh_cache_bytes(const ivh_cache_desc * d, size_t * pages, size_t * scales)
{
  return guard([&] {
    need(d, "null descriptor");
    const ivh::CacheParams c = cache(*d);
    if (pages) *pages = (size_t)c.pages * c.heads * c.page * c.dim * (c.bits / 8);
    if (scales) *scales = c.bits == 8 ? (size_t)c.pages * c.heads * sizeof(float) : 0;
  });
}

int ivh_kv_append(const ivh_append_desc * d, const void * k, const void * v, const int32_t * pos, const float * freq,
                  const int32_t * cu, const int32_t * lens, const int32_t * table, void * kc, void * vc, float * ks, float * vs,
                  int batch, int tokens, void * stream)
{
  return guard([&] {
    need(d, "null descriptor");
    ivh::AppendParams p;
    p.c = cache(d->cache);
    check_counts(batch, tokens);
    if (batch == 0 || tokens == 0) return;
    p.r = rotation(d->rotation, d->cache.dim, pos, d->pos_axis, freq, true);
    check_rows(k, d->k_token, d->k_head, 4, "keys");
    check_rows(v, d->v_token, d->v_head, 4, "values");
    bind(p.c, kc, vc, ks, vs, cu, lens, table, batch, tokens);
    check_device(stream, {k, v, pos, freq, cu, lens, table, kc, vc, ks, vs});
    p.k = k;
    p.v = v;
    p.k_token = d->k_token;
    p.k_head = d->k_head;
    p.v_token = d->v_token;
    p.v_head = d->v_head;
    ivh::launch_kv_append(p, static_cast<hipStream_t>(stream));
    check_launch("kv append");
  });
}

int ivh_paged_attention_workspace(const ivh_paged_attn_desc * d, int batch, int tokens, size_t * bytes)
{
  return guard([&] {
    need(bytes, "null bytes");
    paged(d, batch, tokens, bytes);
  });
}

int ivh_paged_attention(const ivh_paged_attn_desc * d, const void * q, const void * kc, const void * vc, const float * ks,
                        const float * vs, const int32_t * cu, const int32_t * lens, const int32_t * table, void * o, int batch,
                        int tokens, void * workspace, size_t workspace_bytes, void * stream)
{
  return guard([&] {
    size_t bytes = 0;
    ivh::PagedParams p = paged(d, batch, tokens, &bytes);
    if (batch == 0 || tokens == 0) return;
    check_rows(q, d->q_token, d->q_head, 8, "queries");
    check_rows(o, d->o_token, d->o_head, 8, "attention output");
    check_apart(tokens, d->heads, d->cache.dim, d->o_token, d->o_head, "attention");
    bind(p.c, kc, vc, ks, vs, cu, lens, table, batch, tokens);
    need(bytes == 0 || (workspace && workspace_bytes >= bytes), "workspace too small (ivh_paged_attention_workspace)");
    need(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must start at a multiple of 16 bytes");
    check_device(stream, {q, kc, vc, ks, vs, cu, lens, table, o, bytes ? workspace : nullptr});
    p.q = q;
    p.o = o;
    p.q_token = d->q_token;
    p.q_head = d->q_head;
    p.o_token = d->o_token;
    p.o_head = d->o_head;
    p.ws = static_cast<float *>(workspace);
    ivh::launch_paged_attention(p, static_cast<hipStream_t>(stream));
    check_launch("paged attention");
  });
}

int ivh_attention(const ivh_attn_desc * d, const void * q, const void * k, const void * v, const int32_t * cu_q,
                  const int32_t * cu_k, void * o, int batch, int tokens_q, int tokens_k, void * stream)
{
  return guard([&] {
    need(d, "null descriptor");
    check_type(d->type);
    check_counts(batch, tokens_q);
    check_counts(batch, tokens_k);
    need(d->heads >= 1 && d->heads <= 4096 && d->kv_heads >= 1 && d->heads % d->kv_heads == 0,
         "heads must be a multiple of the key heads, at most 4096");
    need((int64_t)batch * d->heads <= kMaxHeads, "too many rows for a call");
    need(d->dim >= 8 && d->dim <= 256 && d->dim % 8 == 0, "dim must be a multiple of 8, at most 256");
    need(std::isfinite(d->scale * kLog2E), "scale must be finite");
    need(d->window >= 0 && d->sinks >= 0 && d->max_q >= 0, "window, sinks and max_q must not be negative");
    if (batch == 0 || tokens_q == 0) return;
    check_rows(q, d->q_token, d->q_head, 8, "queries");
    if (tokens_k > 0) {
      check_rows(k, d->k_token, d->k_head, 8, "keys");
      check_rows(v, d->v_token, d->v_head, 8, "values");
    }
    check_rows(o, d->o_token, d->o_head, 8, "attention output");
    need(d->k_token < (1 << 23) && d->v_token < (1 << 23), "key and value rows must lie less than 2^23 elements apart");
    check_apart(tokens_q, d->heads, d->dim, d->o_token, d->o_head, "attention");
    need(cu_q && cu_k, "null sequence offsets");
    need((reinterpret_cast<uintptr_t>(cu_q) | reinterpret_cast<uintptr_t>(cu_k)) % 4 == 0, "misaligned sequence offsets");
    check_device(stream, {q, k, v, cu_q, cu_k, o});
    ivh::RaggedParams p;
    p.type = d->type;
    p.heads = d->heads;
    p.group = d->heads / d->kv_heads;
    p.dim = d->dim;
    p.batch = batch;
    p.tokens_q = tokens_q;
    p.tokens_k = tokens_k;
    p.max_q = d->max_q ? d->max_q : tokens_q;
    p.causal = d->causal != 0;
    p.window = std::min(d->window, kMaxWindow);
    p.sinks = d->sinks;
    p.scale_log2 = d->scale * kLog2E;
    p.q = q;
    p.k = k;
    p.v = v;
    p.o = o;
    p.cu_q = cu_q;
    p.cu_k = cu_k;
    p.q_token = d->q_token;
    p.q_head = d->q_head;
    p.k_token = d->k_token;
    p.k_head = d->k_head;
    p.v_token = d->v_token;
    p.v_head = d->v_head;
    p.o_token = d->o_token;
    p.o_head = d->o_head;
    ivh::launch_ragged_attention(p, static_cast<hipStream_t>(stream));
    check_launch("attention");
  });
}

}  // extern "C"
