// Attention of each sample's newest tokens over the 8-bit cache (fa_kv8_attention); the cache's layout is in kv8.hip.
//
// Row (t, h) of sample b is the query of token t < n at position i = len - n + t. It sees keys j < i + 1 (causal)
// or j < len:  s_j = q . k_j scale, capped to cap tanh(s_j / cap), less slope_h |i - j|;  o = sum_j softmax(s)_j v_j.
//
// What bounds it is reading the cache once: 2 hd bytes a key and K/V head. The rows that share a K/V head (G heads of
// each token) are the 16 columns of the MFMAs, so a key is read and converted once for all of them. A wave takes
// blocks of 32 keys on its own with a running maximum and sum: S^T = K Q^T (16x16x32, two tiles of 16 keys), softmax
// down the columns, O^T += V^T P^T. The tiles' rows are dealt so that the softmax leaves P exactly where the next
// product wants it: row m of key tile t is key 8 (m / 4) + 4 t + m % 4, so lane quarter q ends with keys 8 q .. 8 q + 7.
// Each wave copies its blocks to LDS on its own (no registers, no barrier): the keys' next block is asked for as soon as
// this one's codes are in registers, the values' likewise, so a whole block is on its way at any time. Keys are split
// over the waves of a workgroup and, where rows are few, over workgroups (the sums then meet in
// the workspace). They are dealt block by block, so that the waves read one contiguous stretch of memory together: with a
// stretch for each wave, equally far apart, all of them met in the same memory channels (2 x 131072 keys: 35.8 us instead of 33.0).
//
// Codes are exact in bf16 and fp16. Q K^T runs in q's type; P is rounded to fp16 (2^-12, half the step of an fp16
// result, a sixteenth of bf16's) for the product with the values' codes; scales, softmax and sums are fp32. Weights are taken
// against a reference 2^15 below the maximum: fp16 then holds those above 2^-29 of the largest with all its bits and the rest to 2^-40
// of it, where against the maximum itself 131072 keys of 2^-26 each, 2^-9 of the sum, were lost.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"
#include "newest.h"

namespace fa {
namespace kv8 {

using newest::BT;
using newest::Place;
using newest::Span;
using newest::W;
using newest::lds_wait;
using newest::span_of;
using newest::splits_used;
using newest::vm_wait;
constexpr float LOG2E = newest::LOG2E;

struct AttnArgs : newest::Args {
  const unsigned char *k, *v;
  const float *ks, *vs;
};

// The reference of weights whose scores (base 2) have the maximum `top`; past 2^22, where the difference would round, itself.
__device__ __forceinline__ float reference(float top) { return fabsf(top) < 4194304.f ? top - 15.f : top; }
// Both sums, of weighted values and of weights, are kept times 2^-35. With weights of up to 2^15 a key adds at most 2^-20 of its
// value: a million keys of the largest values stay in the fp32 range, and those of the smallest scale (2^-100) above its end.
constexpr float SMALL = 0x1p-35f;

template <bool F16>
__device__ __forceinline__ u32x4 cvt8(unsigned lo, unsigned hi) {  // eight e4m3 codes -> eight bf16 / fp16, exact
  if constexpr (F16) {
    return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true))};
  } else {
    return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))};
  }
}

// 0xff in the bytes below n (n <= 0: none, n >= 4: all)
__device__ __forceinline__ unsigned bytes_below(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u; }
// bit 7 of each byte that is the NaN code of either sign
__device__ __forceinline__ unsigned nan_bytes(unsigned c) { return ((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

template <int HD>
using Lds = newest::Lds<HD, 2 * BT * HD>;  // of a wave: a block of keys and one of values

template <bool F16, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(64 * W, HD == 256 ? 2 : HD == 128 ? 3 : 4) attn_kernel(AttnArgs a) {
  constexpr int KS = (HD + 63) / 64, NT = HD / 16, NC = BT * HD / 1024;  // NC: copies of a block
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const Place here = newest::place_of(a);
  if (!here.there) return;
  const int b = here.b, h = here.h, rt = here.rt, split = here.split;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const Span sp = span_of(a, b);

  const int rr = rt * 16 + r, t = rr / a.G, head = h * a.G + rr % a.G, pos = sp.len - sp.n + t;
  const bool valid = rr < a.T * a.G && t < sp.n && pos >= 0;
  int limit = valid ? (a.causal ? pos + 1 : sp.len) : 0;
  int hi = limit, lo = valid ? limit : 0x7fffffff;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    hi = max(hi, __shfl_xor(hi, o));
    lo = min(lo, __shfl_xor(lo, o));
  }
  hi = __builtin_amdgcn_readfirstlane(hi);  // keys that any row sees
  lo = __builtin_amdgcn_readfirstlane(lo);  // keys that every row sees (rows that are not there do not count)
  if (!valid) limit = hi;
  const int nb = (hi + BT - 1) / BT;
  const int used = splits_used(a, nb);
  if (split >= used) return;
  const int at = split * W + wave, all = used * W;

  u32x4 qf[KS][2];
#pragma unroll
  for (int i = 0; i < KS; i++)
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int d = 64 * i + 16 * q + 8 * s;
      qf[i][s] = u32x4{0, 0, 0, 0};
      if (valid && d < HD)
        qf[i][s] = *reinterpret_cast<const u32x4*>(a.q + (b * a.qb + t * a.qt + head * a.qh + d) * 2);
    }
  const float slope = BIAS && valid ? a.slopes[head] * LOG2E : 0.f;

  const size_t unit = ((size_t)b * a.H + h) * a.nblk;
  unsigned char* kl = lds + wave * Lds<HD>::WAVE;
  unsigned char* vl = kl + BT * HD;
  const unsigned at_k = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)kl), at_v = at_k + BT * HD;
  auto copy = [&](const unsigned char* from, int blk, unsigned to) {
    const unsigned char* p = from + (unit + blk) * (BT * HD);
#pragma unroll
    for (int i = 0; i < NC; i++) copy_to_lds(p + i * 1024, lane * 16, to + i * 1024);
  };

  f32x4 O[NT];
#pragma unroll
  for (int j = 0; j < NT; j++) O[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;  // l: this lane's keys only
  if (at < nb) {
    copy(a.k, at, at_k);
    copy(a.v, at, at_v);
  }
  // The queries are waited for here: left to the compiler, that wait (for everything under way) stands in the loop.
#pragma unroll
  for (int i = 0; i < KS; i++) {
    asm volatile("" : "+v"(qf[i][0]));
    asm volatile("" : "+v"(qf[i][1]));
  }
  for (int blk = at; blk < nb; blk += all) {
    const bool more = blk + all < nb;
    vm_wait<NC>();  // the keys; the values are still on their way
    u32x4 kc[2][KS];
#pragma unroll
    for (int i = 0; i < KS; i++)
#pragma unroll
      for (int x = 0; x < 2; x++) {
        kc[x][i] = u32x4{0, 0, 0, 0};
        if (HD % 64 == 0 || 64 * i + 16 * q < HD)
          kc[x][i] = *reinterpret_cast<const u32x4*>(kl + ((4 * i + q) * BT + 8 * (r >> 2) + 4 * x + (r & 3)) * 16);
      }
    const float ksc = a.ks[unit + blk], vsc = a.vs[unit + blk] * SMALL;
    lds_wait();
    if (more) copy(a.k, blk + all, at_k);
    f32x4 s[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      s[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; i++) {
        const u32x4 c = kc[x][i], c0 = cvt8<F16>(c[0], c[1]), c1 = cvt8<F16>(c[2], c[3]);
        s[x] = F16 ? mfma16h(c0, qf[i][0], s[x]) : mfma16(c0, qf[i][0], s[x]);
        s[x] = F16 ? mfma16h(c1, qf[i][1], s[x]) : mfma16(c1, qf[i][1], s[x]);
      }
    }
    const int key0 = blk * BT + 8 * q;
    const bool mixed = blk * BT + BT > lo;
    const float mx = newest::scores<CAP, BIAS>(a, s, ksc, key0, mixed, limit, slope, pos);
    const float mn = fmaxf(m, reference(cols_max(mx)));
    const float ms = mn == -INFINITY ? 0.f : mn;
    if (__builtin_amdgcn_ballot_w64(mn != m)) {
      const float al = exp2_w(m - ms);  // 0 where there was nothing yet
      l *= al;
#pragma unroll
      for (int j = 0; j < NT; j++) O[j] *= al;
      m = mn;
    }
    u32x4 P;
#pragma unroll
    for (int x = 0; x < 2; x++) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[x][i] = exp2_w(s[x][i] - ms);
        l += s[x][i];
      }
      P[2 * x] = pack_f16x2(s[x][0], s[x][1]);
      P[2 * x + 1] = pack_f16x2(s[x][2], s[x][3]);
    }
    if (more) vm_wait<NC>();
    else vm_wait<0>();
    u32x2 vc[NT];  // keys key0 .. key0 + 7 of dim 16 j + r
#pragma unroll
    for (int j = 0; j < NT; j++) vc[j] = *reinterpret_cast<const u32x2*>(vl + (16 * j + r) * BT + 8 * q);
    lds_wait();
    if (more) copy(a.v, blk + all, at_v);
    // Values of keys that a row does not see must not reach it: its P is 0 there, but 0 x NaN is NaN. Codes behind the
    // last key that any row sees are cleared; where one between lo and hi is NaN, each column has its own product.
    bool apart = false;
    if (mixed) {
      const u32x2 some = u32x2{bytes_below(hi - key0), bytes_below(hi - key0 - 4)};
      const u32x2 each = u32x2{bytes_below(lo - key0), bytes_below(lo - key0 - 4)};
      unsigned bad = 0;
#pragma unroll
      for (int j = 0; j < NT; j++) {
        vc[j] &= some;
        bad |= (nan_bytes(vc[j][0]) & ~each[0]) | (nan_bytes(vc[j][1]) & ~each[1]);
      }
      apart = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
    }
    const f32x4 zero = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!apart) {
#pragma unroll
      for (int j = 0; j < NT; j++) O[j] += vsc * mfma16h(cvt8<true>(vc[j][0], vc[j][1]), P, zero);
    } else {
#pragma unroll 1
      for (int c = 0; c < 16; c++) {
        const int n = __builtin_amdgcn_readlane(limit, c) - key0;
        const unsigned own0 = bytes_below(n), own1 = bytes_below(n - 4);
#pragma unroll
        for (int j = 0; j < NT; j++) {
          const f32x4 o = mfma16h(cvt8<true>(vc[j][0] & own0, vc[j][1] & own1), P, zero);
          if (r == c) O[j] += vsc * o;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  newest::meet<F16, HD, Lds<HD>>(a, here, sp, used, lds, O, m, cols_sum(l) * SMALL);
}

template <bool F16, int HD>
__global__ void __launch_bounds__(256) join_kernel(AttnArgs a) {
  newest::join<F16, HD>(a);
}

// A wave takes about 2.3 us for a block of 256 dims that comes from memory (1.2 of 128 and less); more than one workgroup a CU
// (four) share its bandwidth. (Within 10 % of the best of eleven counts in nine of eleven shapes, 17 % in the others.)
int splits_for(int batch, int tokens, int heads, int kv_heads, int hd, int blocks) {
  return newest::splits_for(batch, tokens, heads, kv_heads, blocks, hd == 256 ? 2.3 : 1.2, hd == 256 ? 1.0 : 4.0);
}

template <bool F16, int HD>
int launch_attn(const AttnArgs& a, hipStream_t s) {
  const unsigned grid = newest::grid_of(a);
  if (!grid) return host::fail(FA_ERR_INVALID_ARG, "fa_kv8_attention: too many rows for one call");
  const bool cap = a.cap > 0.f, bias = a.slopes != nullptr;
  void (*k)(AttnArgs) = cap ? (bias ? attn_kernel<F16, HD, true, true> : attn_kernel<F16, HD, true, false>)
                            : (bias ? attn_kernel<F16, HD, false, true> : attn_kernel<F16, HD, false, false>);
  const unsigned lds = Lds<HD>::BYTES;
  const int rc = host::allow_lds(reinterpret_cast<const void*>(k), lds, "fa_kv8_attention");
  if (rc != FA_OK) return rc;
  hipLaunchKernelGGL(k, dim3(grid), dim3(64 * W), lds, s, a);
  if (a.S > newest::FUSED) hipLaunchKernelGGL((join_kernel<F16, HD>), dim3(newest::join_grid(a, HD)), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return host::fail(FA_ERR_LAUNCH, "fa_kv8_attention: %s", hipGetErrorString(e));
  return FA_OK;
}

template <bool F16>
int launch_attn(const AttnArgs& a, int hd, hipStream_t s) {
  if (hd == 64) return launch_attn<F16, 64>(a, s);
  if (hd == 96) return launch_attn<F16, 96>(a, s);
  if (hd == 128) return launch_attn<F16, 128>(a, s);
  return launch_attn<F16, 256>(a, s);
}

int check_cache(const void* k, const void* v, const void* ks, const void* vs, int batch, int heads, int hd, int blocks,
                const char* who);  // kv8.hip

}  // namespace kv8
}  // namespace fa

extern "C" size_t fa_kv8_attention_workspace_bytes(int batch, int tokens, int heads, int kv_heads, int head_dim, int blocks) {
  if (batch < 1 || tokens < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads || head_dim < 1 || blocks < 1) return 0;
  return fa::newest::workspace(fa::kv8::splits_for(batch, tokens, heads, kv_heads, head_dim, blocks), batch, tokens, heads, kv_heads,
                               head_dim);
}

extern "C" int fa_kv8_attention(const fa_kv8_attn_args* a, fa_stream_t stream) {
  using namespace fa;
  const char* who = "fa_kv8_attention";
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  int rc = kv8::check_cache(a->cache_k, a->cache_v, a->cache_ks, a->cache_vs, a->batch, a->kv_heads, a->head_dim, a->blocks, who);
  if (rc != FA_OK) return rc;
  rc = newest::check_call(a, who);
  if (rc != FA_OK || a->tokens == 0) return rc;
  kv8::AttnArgs p{};
  p.k = static_cast<const unsigned char*>(a->cache_k), p.v = static_cast<const unsigned char*>(a->cache_v);
  p.ks = a->cache_ks, p.vs = a->cache_vs;
  rc = newest::set_up(p, a, a->blocks, kv8::splits_for(a->batch, a->tokens, a->heads, a->kv_heads, a->head_dim, a->blocks), 1,
                      who);
  if (rc != FA_OK) return rc;
  rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  return a->dtype == FA_DTYPE_F16 ? kv8::launch_attn<true>(p, a->head_dim, (hipStream_t)stream)
                                  : kv8::launch_attn<false>(p, a->head_dim, (hipStream_t)stream);
}
