// The paged K/V cache: rows into pages with the position's rotation on the way (fa_paged_append), pages back to rows
// (fa_paged_load). The attention over it is in paged_attn.hip.
//
// A page holds 32 tokens, per K/V head k[hd / 8][32][8] and v[4][hd][8]: the operand orders of the attention's MFMAs, so that
// its copies are whole lines and each lane finds its 16 bytes side by side (keys: 8 dims of a token, values: 8 tokens of a dim).
//
// Rotation of pair j at position p: angle p f_j. Its turns, p f_j / 2 pi, are taken in 64 bits (53 bits hold them to 2^-30 at
// 2^23 turns) and reduced to [-1/2, 1/2] exactly; sine and cosine and the products are fp32, the result is rounded once.
// The bound is bytes: rows in and out once. A position's angles serve all heads: a workgroup takes a window of tokens, puts their
// sines and cosines into LDS and then goes over the heads, 16 bytes of each half of the pairs a thread.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"

namespace fa {
namespace paged {

constexpr int PT = 32;  // tokens of a page

struct RowArgs {
  const unsigned short* q;
  unsigned short* qo;
  int64_t qs[3];
  unsigned short *k, *v;
  int64_t ks[4], vs[4];
  unsigned short *pk, *pv;
  const int* table;
  int64_t ts;
  const int *start, *count;
  const double* freqs;
  int B, T, HQ, H, hd, pages, width, rot, adjacent, zero, windows;
};

template <bool F16>
__device__ __forceinline__ float lo(unsigned u) {
  return F16 ? h_lo(u) : bf_lo(u);
}
template <bool F16>
__device__ __forceinline__ float hi(unsigned u) {
  return F16 ? h_hi(u) : bf_hi(u);
}
template <bool F16>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  return F16 ? pack_f16x2(a, b) : pack_bf16x2(a, b);
}

// Page i of sample b, or -1.
__device__ __forceinline__ int page_of(const RowArgs& a, int b, int64_t i) {
  if (i < 0 || i >= a.width) return -1;
  const int p = a.table[b * a.ts + i];
  return (unsigned)p < (unsigned)a.pages ? p : -1;
}

// WIN: tokens of a workgroup's window, 8 aligned ones, whose values leave as whole pieces of 8 tokens, or 1.
template <bool F16, int WIN>
__global__ void __launch_bounds__(256) append_kernel(RowArgs a) {
  extern __shared__ float2 turn[];  // [WIN][rot / 2] cosine, sine
  const int b = blockIdx.x / a.windows, w = blockIdx.x - b * a.windows, i = threadIdx.x;
  const int first = a.start[b], half = a.rot >> 1;
  const int n = first < 0 ? 0 : a.count ? max(0, min(a.count[b], a.T)) : a.T;
  const int64_t s = max(first, 0), p0 = (s & -WIN) + (int64_t)w * WIN;  // the window's first position
  if (p0 - s >= a.T) return;
  const int page = page_of(a, b, p0 / PT), slot = (int)(p0 & (PT - 1));
  for (int e = i; e < WIN * half; e += 256) {
    const int x = e / half, j = e - x * half;
    const double t = (double)(p0 + x) * a.freqs[j] * 0.15915494309189535;  // 1 / 2 pi
    float sn, cs;
    sincospif(2.f * (float)(t - rint(t)), &sn, &cs);
    turn[e] = float2{cs, sn};
  }
  __syncthreads();

  // A head's pieces, 8 pairs or 8 dims that do not turn: dims d1 .. d1 + 7 and, of pairs, d1 + half .. of the result.
  const int pairs = a.rot >> 4, each = pairs + ((a.hd - a.rot) >> 3), step = gridDim.y * 256;
  auto first_dim = [&](int c) { return c < pairs ? 8 * c : a.rot + 8 * (c - pairs); };
  auto piece = [&](const unsigned short* in, int c, int x, u32x4& one, u32x4& two) {  // of token x of the window
    const int d = first_dim(c);
    if (c >= pairs) {
      one = *reinterpret_cast<const u32x4*>(in + d);
      return;
    }
    const u32x4 f = *reinterpret_cast<const u32x4*>(in + (a.adjacent ? 2 * d : d));
    const u32x4 g = *reinterpret_cast<const u32x4*>(in + (a.adjacent ? 2 * d + 8 : d + half));
    const float2* t = turn + x * half + d;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      float lo0, hi0, lo1, hi1;  // pairs 2 k and 2 k + 1
      if (a.adjacent) {
        const unsigned u0 = k < 2 ? f[2 * (k & 1)] : g[2 * (k & 1)], u1 = k < 2 ? f[2 * (k & 1) + 1] : g[2 * (k & 1) + 1];
        lo0 = lo<F16>(u0), hi0 = hi<F16>(u0), lo1 = lo<F16>(u1), hi1 = hi<F16>(u1);
      } else {
        lo0 = lo<F16>(f[k]), hi0 = lo<F16>(g[k]), lo1 = hi<F16>(f[k]), hi1 = hi<F16>(g[k]);
      }
      const float2 t0 = t[2 * k], t1 = t[2 * k + 1];
      one[k] = pack2<F16>(lo0 * t0.x - hi0 * t0.y, lo1 * t1.x - hi1 * t1.y);
      two[k] = pack2<F16>(hi0 * t0.x + lo0 * t0.y, hi1 * t1.x + lo1 * t1.y);
    }
  };
  // queries: neighbouring lanes along the dims, whose rows are read and written in runs
  for (int u = blockIdx.y * 256 + i; u < WIN * a.HQ * each; u += step) {
    const int y = u / each, c = u - y * each, x = y / a.HQ, h = y - x * a.HQ;
    const int64_t row = p0 + x - s;
    if (row < 0 || row >= a.T) continue;
    u32x4 one = u32x4{0, 0, 0, 0}, two = one;
    if (row < n) piece(a.q + b * a.qs[0] + row * a.qs[1] + h * a.qs[2], c, x, one, two);
    unsigned short* to = a.qo + (((size_t)b * a.T + row) * a.HQ + h) * a.hd + first_dim(c);
    *reinterpret_cast<u32x4*>(to) = one;
    if (c < pairs) *reinterpret_cast<u32x4*>(to + half) = two;
  }
  if (page < 0) return;
  // keys: along the tokens, whose pieces lie side by side in the page
  for (int u = blockIdx.y * 256 + i; u < WIN * a.H * each; u += step) {
    const int x = u % WIN, y = u / WIN, h = y / each, c = y - h * each;
    const int64_t row = p0 + x - s;
    if (row < 0 || row >= n) continue;
    u32x4 one, two;
    piece(a.k + b * a.ks[0] + row * a.ks[1] + h * a.ks[2], c, x, one, two);
    unsigned short* to = a.pk + ((size_t)page * a.H + h) * PT * a.hd + first_dim(c) * PT + (slot + x) * 8;
    *reinterpret_cast<u32x4*>(to) = one;
    if (c < pairs) *reinterpret_cast<u32x4*>(to + half * PT) = two;
  }

  // values: [head][8 dims]
  const int chunks = a.hd >> 3, from = (int)max((int64_t)0, s - p0), to = (int)min((int64_t)WIN, s + n - p0);
  for (int u = blockIdx.y * 256 + i; u < a.H * chunks; u += step) {
    const int h = u / chunks, d = (u - h * chunks) * 8;
    const unsigned short* in = a.v + b * a.vs[0] + (p0 - s) * a.vs[1] + h * a.vs[2] + d;
    unsigned short* out = a.pv + (((size_t)page * a.H + h) * (PT / 8) + (slot >> 3)) * a.hd * 8 + d * 8 + (slot & 7);
    if (WIN == 8 && from <= 0 && to >= 8) {
      u32x4 x[8], y;
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = *reinterpret_cast<const u32x4*>(in + j * a.vs[1]);
#pragma unroll
      for (int e = 0; e < 8; e++) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const unsigned u0 = x[2 * j][e >> 1], u1 = x[2 * j + 1][e >> 1];
          y[j] = e & 1 ? (u0 >> 16) | (u1 & 0xffff0000u) : (u0 & 0xffffu) | (u1 << 16);
        }
        *reinterpret_cast<u32x4*>(out + e * 8) = y;
      }
    } else {
      for (int j = from; j < to; j++) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(in + j * a.vs[1]);
#pragma unroll
        for (int e = 0; e < 8; e++) out[e * 8 + j] = (unsigned short)(x[e >> 1] >> (16 * (e & 1)));
      }
    }
  }
}

// One page of one head; KVEC: dims of k are contiguous and its rows 16-byte aligned, VVEC: tokens of v.
template <bool KVEC, bool VVEC>
__global__ void __launch_bounds__(256) load_kernel(RowArgs a) {
  const int h = blockIdx.x % a.H, y = blockIdx.x / a.H, b = y / a.windows, w = y - b * a.windows;
  const int64_t n = max((int64_t)0, min((int64_t)min(a.count[b], a.T), (int64_t)a.width * PT));
  const int64_t t0 = (int64_t)w * PT, end = a.zero ? a.T : n;  // of what is written
  if (t0 >= end) return;
  const int page = page_of(a, b, w);
  const size_t unit = ((size_t)max(page, 0) * a.H + h) * PT * a.hd;
  const int pieces = a.hd * PT / 8;
  for (int u = threadIdx.x; u < pieces; u += 256) {  // keys: 8 dims of a token
    const int x = u & (PT - 1), d = (u / PT) * 8;
    const int64_t t = t0 + x;
    if (t >= end) continue;
    u32x4 v = u32x4{0, 0, 0, 0};
    if (page >= 0 && t < n) v = *reinterpret_cast<const u32x4*>(a.pk + unit + (size_t)u * 8);
    unsigned short* to = a.k + b * a.ks[0] + t * a.ks[1] + h * a.ks[2] + d * a.ks[3];
    if constexpr (KVEC) {
      *reinterpret_cast<u32x4*>(to) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) to[e * a.ks[3]] = (unsigned short)(v[e >> 1] >> (16 * (e & 1)));
    }
  }
  for (int u = threadIdx.x; u < pieces; u += 256) {  // values: 8 tokens of a dim
    const int d = u % a.hd;
    const int64_t t = t0 + (u / a.hd) * 8;
    if (t >= end) continue;
    u32x4 v = u32x4{0, 0, 0, 0};
    if (page >= 0 && t < n) v = *reinterpret_cast<const u32x4*>(a.pv + unit + (size_t)u * 8);
    unsigned short* to = a.v + b * a.vs[0] + t * a.vs[1] + h * a.vs[2] + d * a.vs[3];
    if (VVEC && t + 8 <= n) {
      *reinterpret_cast<u32x4*>(to) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (t + e < end) to[e * a.vs[1]] = t + e < n ? (unsigned short)(v[e >> 1] >> (16 * (e & 1))) : (unsigned short)0;
    }
  }
}

int check_pool(const void* k, const void* v, const int* table, int batch, int heads, int hd, int pages, int width, int64_t stride,
               const char* who) {
  if (batch < 1 || heads < 1 || pages < 1 || width < 1 || batch > (1 << 20) || heads > (1 << 16) || width > (1 << 26) ||
      (int64_t)pages * heads > (int64_t)1 << 31)
    return host::fail(FA_ERR_INVALID_ARG, "%s: batch=%d, kv_heads=%d, pages=%d, table_pages=%d", who, batch, heads, pages, width);
  if (hd != 64 && hd != 96 && hd != 128 && hd != 256)
    return host::fail(FA_ERR_INVALID_ARG, "%s: head_dim=%d is none of 64, 96, 128, 256", who, hd);
  if (!k || !v || !table) return host::fail(FA_ERR_INVALID_ARG, "%s: the pool or the table is NULL", who);
  if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16)
    return host::fail(FA_ERR_INVALID_ARG, "%s: the pool is not 16-byte aligned", who);
  if (reinterpret_cast<uintptr_t>(table) % 4) return host::fail(FA_ERR_INVALID_ARG, "%s: table is not 4-byte aligned", who);
  if (batch > 1 && stride < width)
    return host::fail(FA_ERR_INVALID_ARG, "%s: table_stride=%lld is below table_pages=%d", who, (long long)stride, width);
  return FA_OK;
}

namespace {

int set_up(RowArgs& p, const fa_paged_rows_args* a, bool append, const char* who) {
  int rc = check_pool(a->pool_k, a->pool_v, a->table, a->batch, a->kv_heads, a->head_dim, a->pages, a->table_pages, a->table_stride,
                      who);
  if (rc != FA_OK) return rc;
  if (a->dtype != FA_DTYPE_BF16 && a->dtype != FA_DTYPE_F16)
    return host::fail(FA_ERR_INVALID_ARG, "%s: dtype %d: rows and pages are bf16 or fp16", who, a->dtype);
  if (a->tokens < 0 || a->tokens > (1 << 30)) return host::fail(FA_ERR_INVALID_ARG, "%s: tokens=%d", who, a->tokens);
  if (a->tokens && (!a->k || !a->v || (append ? !a->start : !a->count))) return host::fail(FA_ERR_INVALID_ARG, "%s: a pointer is NULL", who);
  const unsigned align = append ? 16 : 2;
  if (reinterpret_cast<uintptr_t>(a->k) % align || reinterpret_cast<uintptr_t>(a->v) % align)
    return host::fail(FA_ERR_INVALID_ARG, "%s: k or v is not %u-byte aligned", who, align);
  if (reinterpret_cast<uintptr_t>(a->start) % 4 || reinterpret_cast<uintptr_t>(a->count) % 4)
    return host::fail(FA_ERR_INVALID_ARG, "%s: start or count is not 4-byte aligned", who);
  p.k = static_cast<unsigned short*>(a->k), p.v = static_cast<unsigned short*>(a->v);
  p.pk = static_cast<unsigned short*>(a->pool_k), p.pv = static_cast<unsigned short*>(a->pool_v);
  for (int i = 0; i < 4; i++) p.ks[i] = a->k_stride[i], p.vs[i] = a->v_stride[i];
  p.table = a->table, p.ts = a->table_stride, p.start = a->start, p.count = a->count;
  p.B = a->batch, p.T = a->tokens, p.H = a->kv_heads, p.hd = a->head_dim, p.pages = a->pages, p.width = a->table_pages;
  return FA_OK;
}

}  // namespace
}  // namespace paged
}  // namespace fa

extern "C" int fa_paged_append(const fa_paged_rows_args* a, fa_stream_t stream) {
  using namespace fa;
  const char* who = "fa_paged_append";
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  paged::RowArgs p{};
  int rc = paged::set_up(p, a, true, who);
  if (rc != FA_OK) return rc;
  for (int i = 0; i < 3; i++)
    if (a->k_stride[i] % 8 || a->v_stride[i] % 8 || (a->q && a->q_stride[i] % 8))
      return host::fail(FA_ERR_INVALID_ARG, "%s: strides must be multiples of 8", who);
  if (a->k_stride[3] != 1 || a->v_stride[3] != 1) return host::fail(FA_ERR_INVALID_ARG, "%s: dims must be contiguous", who);
  if (a->rotary < 0 || a->rotary > a->head_dim || a->rotary % 16)
    return host::fail(FA_ERR_INVALID_ARG, "%s: rotary=%d must be a multiple of 16 up to head_dim=%d", who, a->rotary, a->head_dim);
  if (a->rotary && (!a->freqs || reinterpret_cast<uintptr_t>(a->freqs) % 8))
    return host::fail(FA_ERR_INVALID_ARG, "%s: freqs is NULL or not 8-byte aligned", who);
  if (a->q) {
    if (!a->q_out || reinterpret_cast<uintptr_t>(a->q) % 16 || reinterpret_cast<uintptr_t>(a->q_out) % 16)
      return host::fail(FA_ERR_INVALID_ARG, "%s: q_out is NULL, or q or q_out not 16-byte aligned", who);
    if (a->heads < 1 || a->heads > (1 << 16)) return host::fail(FA_ERR_INVALID_ARG, "%s: heads=%d", who, a->heads);
    p.q = static_cast<const unsigned short*>(a->q), p.qo = static_cast<unsigned short*>(a->q_out), p.HQ = a->heads;
    for (int i = 0; i < 3; i++) p.qs[i] = a->q_stride[i];
  }
  p.freqs = a->freqs, p.rot = a->rotary, p.adjacent = a->adjacent;
  if (a->tokens == 0) return FA_OK;
  const int win = a->tokens >= 8 ? 8 : 1;
  p.windows = (a->tokens + win - 2) / win + 1;  // of any alignment
  if ((int64_t)p.windows * a->batch > host::MAX_GRID) return host::fail(FA_ERR_INVALID_ARG, "%s: too many rows for one call", who);
  rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  // Workgroups of a window: a thread has up to three pieces (four prompts of 2011 tokens, 16 and 4 heads of 128 dims: 27.4 us in one
  // workgroup of eight pieces a thread, 24.5 in three, 26.5 in eight), or one where windows alone do not fill the chip.
  const int units = (p.HQ + p.H) * ((p.rot >> 4) + ((p.hd - p.rot) >> 3)) * win, most = (units + 255) / 256;
  const int slices = std::min(64, std::max((most + 2) / 3, std::min<int>(most, 1024 / std::min<int64_t>(1024, (int64_t)p.windows * p.B))));
  const dim3 grid(p.windows * p.B, slices);
  const unsigned lds = win * (p.rot / 2) * sizeof(float2);
  const bool f16 = a->dtype == FA_DTYPE_F16;
  void (*k)(paged::RowArgs) = f16 ? (win == 8 ? paged::append_kernel<true, 8> : paged::append_kernel<true, 1>)
                                  : (win == 8 ? paged::append_kernel<false, 8> : paged::append_kernel<false, 1>);
  hipLaunchKernelGGL(k, grid, dim3(256), lds, (hipStream_t)stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return host::fail(FA_ERR_LAUNCH, "%s: %s", who, hipGetErrorString(e));
  return FA_OK;
}

extern "C" int fa_paged_load(const fa_paged_rows_args* a, fa_stream_t stream) {
  using namespace fa;
  const char* who = "fa_paged_load";
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  paged::RowArgs p{};
  int rc = paged::set_up(p, a, false, who);
  if (rc != FA_OK) return rc;
  p.zero = a->zero_rest;
  if (a->tokens == 0) return FA_OK;
  p.windows = (a->tokens + paged::PT - 1) / paged::PT;
  const int64_t grid = (int64_t)p.windows * p.B * p.H;
  if (grid > host::MAX_GRID) return host::fail(FA_ERR_INVALID_ARG, "%s: too many rows for one call", who);
  rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  auto whole = [](const long long* s, int one, int x, int y, int z, const void* at) {
    return s[one] == 1 && s[x] % 8 == 0 && s[y] % 8 == 0 && s[z] % 8 == 0 && reinterpret_cast<uintptr_t>(at) % 16 == 0;
  };
  const bool kvec = whole(a->k_stride, 3, 0, 1, 2, a->k), vvec = whole(a->v_stride, 1, 0, 2, 3, a->v);
  void (*k)(paged::RowArgs) = kvec ? (vvec ? paged::load_kernel<true, true> : paged::load_kernel<true, false>)
                                   : (vvec ? paged::load_kernel<false, true> : paged::load_kernel<false, false>);
  hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return host::fail(FA_ERR_LAUNCH, "%s: %s", who, hipGetErrorString(e));
  return FA_OK;
}
