// Span attention on bf16 (attention.h), and its C entry.
#include "attention.h"

int fa::attn::run_bf16(const Params& p, hipStream_t s) { return launch_type<false>(p, s); }

extern "C" size_t fa_span_attention_workspace_bytes(int batch, int queries, int keys, int heads, int head_dim) {
  if (batch < 1 || queries < 1 || keys < 1 || heads < 1 || head_dim < 1 || head_dim > 256) return 0;
  return fa::attn::workspace(batch, queries, keys, heads, head_dim);
}

extern "C" int fa_span_attention(const fa_span_args* a, fa_stream_t stream) {
  using namespace fa;
  const char* who = "fa_span_attention";
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->dtype != FA_DTYPE_BF16 && a->dtype != FA_DTYPE_F16)
    return host::fail(FA_ERR_INVALID_ARG, "%s: dtype %d: q, k and v are bf16 or fp16", who, a->dtype);
  if (a->batch < 0 || a->queries < 0 || a->keys < 0 || a->batch > (1 << 24) || a->queries > (1 << 30) || a->keys > (1 << 30))
    return host::fail(FA_ERR_INVALID_ARG, "%s: batch=%d, queries=%d, keys=%d", who, a->batch, a->queries, a->keys);
  if (a->kv_heads < 1 || a->heads < 1 || a->heads > (1 << 16) || a->heads % a->kv_heads)
    return host::fail(FA_ERR_INVALID_ARG, "%s: heads=%d is no multiple of kv_heads=%d", who, a->heads, a->kv_heads);
  if (a->head_dim < 8 || a->head_dim > 256 || a->head_dim % 8)
    return host::fail(FA_ERR_INVALID_ARG, "%s: head_dim=%d is no multiple of 8 in [8, 256]", who, a->head_dim);
  if (!(a->softcap >= 0.f) || !(a->softcap < INFINITY) || !(a->scale >= 0.f) || !(a->scale < INFINITY))
    return host::fail(FA_ERR_INVALID_ARG, "%s: scale=%g and softcap=%g must be finite and >= 0", who, a->scale,
                      a->softcap);
  if (a->batch == 0 || a->queries == 0) return FA_OK;
  if (!a->q || !a->out || (a->keys > 0 && (!a->k || !a->v)))
    return host::fail(FA_ERR_INVALID_ARG, "%s: q, k, v or out is NULL", who);
  const void* ptrs[] = {a->q, a->k, a->v, a->out};
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % 16)
      return host::fail(FA_ERR_INVALID_ARG, "%s: q, k, v or out is not 16-byte aligned", who);
  if (reinterpret_cast<uintptr_t>(a->spans) % 4 || reinterpret_cast<uintptr_t>(a->slopes) % 4)
    return host::fail(FA_ERR_INVALID_ARG, "%s: spans or slopes is not 4-byte aligned", who);
  for (int i = 0; i < 3; i++)
    if (a->q_stride[i] % 8 || a->k_stride[i] % 8 || a->v_stride[i] % 8)
      return host::fail(FA_ERR_INVALID_ARG, "%s: strides must be multiples of 8", who);
  // a tile's rows are addressed with 32-bit offsets
  if (a->k_stride[1] < 0 || a->v_stride[1] < 0 || a->k_stride[1] > (1 << 23) || a->v_stride[1] > (1 << 23))
    return host::fail(FA_ERR_UNSUPPORTED, "%s: token strides of k and v must be in [0, 2^23]", who);
  attn::Params p{};
  p.q = static_cast<const unsigned char*>(a->q);
  p.k = static_cast<const unsigned char*>(a->k);
  p.v = static_cast<const unsigned char*>(a->v);
  p.qb = a->q_stride[0], p.qt = a->q_stride[1], p.qh = a->q_stride[2];
  p.kb = a->k_stride[0], p.kt = (int)a->k_stride[1], p.kh = a->k_stride[2];
  p.vb = a->v_stride[0], p.vt = (int)a->v_stride[1], p.vh = a->v_stride[2];
  p.spans = a->spans, p.slopes = a->slopes;
  p.out = static_cast<unsigned char*>(a->out);
  p.B = a->batch, p.Tq = a->queries, p.Tk = a->keys, p.H = a->heads, p.G = a->heads / a->kv_heads, p.hd = a->head_dim;
  p.scale = a->softcap > 0.f ? 2.f * attn::LOG2E * a->scale / a->softcap : a->scale * attn::LOG2E;
  p.over = a->softcap > 0.f ? a->scale / a->softcap : 0.f;
  p.cap = a->softcap * attn::LOG2E;
  p.flat = a->scale == 0.f;
  if (p.flat) p.scale = 1.f;
  if (!(p.scale < INFINITY) || !(p.cap < INFINITY))
    return host::fail(FA_ERR_INVALID_ARG, "%s: scale=%g over softcap=%g leaves the fp32 range", who, a->scale, a->softcap);
  const size_t need = attn::workspace(a->batch, a->queries, a->keys, a->heads, a->head_dim);
  p.S = 1;
  if (a->workspace && need) {
    if (a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16)
      return host::fail(FA_ERR_INVALID_ARG, "%s: workspace of %zu bytes at %p, needs %zu, 16-byte aligned", who,
                        a->workspace_bytes, a->workspace, need);
    const int64_t units = attn::units_of(a->batch, a->queries, a->heads);
    p.S = attn::splits_for(units, a->keys, a->head_dim);
    p.least = attn::LEAST;
    p.used = static_cast<int*>(a->workspace);
    p.arrived = reinterpret_cast<uint64_t*>(static_cast<unsigned char*>(a->workspace) + attn::used_bytes(units));
    p.part = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(p.arrived) + attn::arrived_bytes(units));
    p.nonce = p.S <= attn::FUSED ? host::launch_nonce() : 0;
  }
  const int rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  return a->dtype == FA_DTYPE_F16 ? attn::run_f16(p, (hipStream_t)stream) : attn::run_bf16(p, (hipStream_t)stream);
}
