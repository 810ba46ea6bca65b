// Attention of each sample's newest tokens over a paged cache (fa_paged_attention); the pages' layout is in paged.hip.
//
// Row (t, h) of sample b is the query of token t < n at position i = len - n + t. It sees keys j < i + 1 (causal)
// or j < len:  s_j = q . k_j scale, capped to cap tanh(s_j / cap), less slope_h |i - j|;  o = sum_j softmax(s)_j v_j.
//
// What bounds it is reading the cache once: 4 hd bytes a key and K/V head. The rows that share a K/V head are the 16 columns of the
// MFMAs. A wave takes pages on its own with a running maximum and sum: S^T = K Q^T (16x16x32, two tiles of 16 keys), softmax
// down the columns, O^T += V^T P^T; row m of key tile t is key 8 (m / 4) + 4 t + m % 4, so lane quarter q ends with keys
// 8 q .. 8 q + 7, the next product's operand. Each wave copies its pages to LDS on its own (no registers, no barrier): the next
// page's keys are asked for as soon as this one's are in registers, the values' likewise. How pages are dealt to waves and
// workgroups, and how their sums meet: newest.h.
//
// With many rows (a piece of a prompt) each workgroup takes its pages from the L2 again, at what a CU copies from there (110 GB/s): a wave then
// has two tiles of rows for each page (tiles_for). Not kept: workgroups of 64 rows whose waves walk together over pages that are copied once
// (293 tokens x 8 heads over up to 4011 keys 38 us with single tiles, 52 with four splits and 117 unsplit that way; 1024 tokens of 32
// heads over 8192 keys 306, and 239 with two tiles a wave).
//
// Rounding: scores are exact products summed in fp32, softmax and sums are fp32. bf16: the weights go into the second
// product as two bf16 (2^-16 of each is lost; as one, 2^-9), and are taken against a reference 2^17 above
// the maximum, so that 131072 keys cannot leave the fp32 range whatever the values. fp16: the weights are rounded once (2^-12), against a
// reference 2^15 below the maximum: those above 2^-29 of the largest keep all their bits. The result's own rounding is 2^-12 as well: of
// the 2-norm 1.8e-4 to 2.1e-4 are off by it alone, 2.0e-4 to 2.6e-4 with the weights'. A second part takes its time in pieces of prompts, whose
// MFMAs count: 1024 tokens over 8192 keys 245 us in bf16, 220 in fp16; in fp16 with two parts 293 tokens over up to 4011 keys 37.4 -> 40.8 us,
// 4 x 256 of 256 dims over 4096 137 -> 146, 48 single tokens over up to 8192 28.7 -> 28.8, capped and biased 29.0 -> 30.0.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"
#include "newest.h"

namespace fa {
namespace paged {

using newest::BT;
using newest::Place;
using newest::Span;
using newest::W;
using newest::lds_wait;
using newest::vm_wait;

struct AttnArgs : newest::Args {
  const unsigned char *k, *v;
  const int* table;
  int64_t ts;
  int pages;
};

constexpr float FAR = 4194304.f;  // from here on numbers are half a unit and more apart
template <bool F16>
__device__ __forceinline__ float reference(float top) {
  return fabsf(top) < FAR ? top + (F16 ? -15.f : 17.f) : top;  // past it the difference would round
}
template <bool F16>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  return F16 ? mfma16h(a, b, c) : mfma16(a, b, c);
}
// The halves of words 0 .. 3 (keys 0 .. 7) below n.
__device__ __forceinline__ u32x4 halves_below(int n) {
  u32x4 x;
#pragma unroll
  for (int j = 0; j < 4; j++) x[j] = n >= 2 * j + 2 ? ~0u : n == 2 * j + 1 ? 0xffffu : 0u;
  return x;
}

// A page of keys lies in LDS with its tokens in the order in which the two MFMAs' rows take them (16 lanes read 256 bytes in one run;
// in the page's own order they met in half of the banks): slot 16 x + m holds token 8 (m / 4) + 4 x + m % 4. A copy's lane i
// fetches what belongs into slot i of its 1 KB, four neighbours 64 bytes in one run.
__device__ __forceinline__ unsigned key_offset(int lane) {
  return (lane >> 5) * 512 + (8 * ((lane & 15) >> 2) + 4 * ((lane >> 4) & 1) + (lane & 3)) * 16;
}

// What a wave keeps of its tile of 16 rows: row r is column r of the MFMAs, lane r + 16 q.
template <bool F16, int HD, bool CAP, bool BIAS>
struct Tile {
  static constexpr int KS = HD / 32, NT = HD / 16;
  int pos, limit, lo, hi;  // keys that the row sees, that every row does (those that are not there do not count), that any does
  float slope, m, l;       // m: the weights' reference; l: their sum over this lane's keys
  uint64_t far;            // lanes of rows whose reference is past FAR
  u32x4 q[KS];
  f32x4 O[NT];

  __device__ __forceinline__ void begin(const AttnArgs& a, const Place& at, const Span& sp, int rt) {
    const int lane = threadIdx.x & 63, row = rt * 16 + (lane & 15), t = row / a.G, head = at.h * a.G + row % a.G;
    pos = sp.len - sp.n + t;
    const bool valid = row < a.T * a.G && t < sp.n && pos >= 0;
    limit = valid ? (a.causal ? pos + 1 : sp.len) : 0;
    hi = limit, lo = valid ? limit : 0x7fffffff;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      hi = max(hi, __shfl_xor(hi, o));
      lo = min(lo, __shfl_xor(lo, o));
    }
    hi = __builtin_amdgcn_readfirstlane(hi);
    lo = __builtin_amdgcn_readfirstlane(lo);
    if (!valid) limit = hi;
#pragma unroll
    for (int i = 0; i < KS; i++) {
      q[i] = u32x4{0, 0, 0, 0};
      if (valid)
        q[i] = *reinterpret_cast<const u32x4*>(a.q + (at.b * a.qb + t * a.qt + head * a.qh + 32 * i + 8 * (lane >> 4)) * 2);
    }
    slope = BIAS && valid ? a.slopes[head] * newest::LOG2E : 0.f;
    m = -INFINITY, l = 0.f, far = 0;
#pragma unroll
    for (int j = 0; j < NT; j++) O[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Waits for the queries: left to the compiler, that wait (for everything under way) stands in the loop.
  __device__ __forceinline__ void arrive() {
#pragma unroll
    for (int i = 0; i < KS; i++) asm volatile("" : "+v"(q[i]));
    asm volatile("" : "+v"(slope));
  }

  // The products s of block `blk`'s keys -> its weights P (and what they left off, R; bf16 only) against the new reference.
  __device__ __forceinline__ void weigh(const AttnArgs& a, f32x4* s, int blk, bool gone, u32x4& P, u32x4& R) {
    const int key0 = blk * BT + 8 * ((threadIdx.x & 63) >> 4);
    const bool mixed = blk * BT + BT > (gone ? 0 : lo);
    const int own = gone ? 0 : limit;
    float mx, f = 1.f;  // scores are s f
    if (!CAP && !BIAS && a.scale > 0.f) {
      f = a.scale;  // goes into the exponent's one instruction
      if (mixed) {
        asm volatile("");  // a branch: as selects the masks cost every block
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (key0 + 4 * x + i >= own) s[x][i] = -INFINITY;
      }
      mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[x][i]);
      mx *= f;
    } else {
      mx = newest::scores<CAP, BIAS>(a, s, 1.f, key0, mixed, own, slope, pos);
    }
    const float mn = fmaxf(m, reference<F16>(cols_max(mx)));
    float ms = mn == -INFINITY ? 0.f : mn;
    if (__builtin_amdgcn_ballot_w64(mn != m) | far) {
      const float al = exp2_w(m - ms);  // 0 where there was nothing yet
      l *= al;
#pragma unroll
      for (int j = 0; j < NT; j++) O[j] *= al;
      m = mn;
      // The reference is a rounded product, and what the rounding took off stands in the fused exponents below: up to 2^6 at 2^30, where the
      // largest weight would vanish or overflow. Of rows past FAR (each by itself: another's scores do not change its roundings) s
      // becomes the difference of rounded products, 0 for the largest, in units of f. (The test makes pieces of prompts 1 to 4 % longer; no
      // test here and a second walk over the pages of waves that met such a row cost as much, as the compiler lays it out.)
      if constexpr (!CAP && !BIAS) {
        const bool own = fabsf(ms) >= FAR;
        far = __builtin_amdgcn_ballot_w64(own);
        if (__builtin_expect(far != 0, 0)) {
          const float unit = 1.f / f;
#pragma unroll
          for (int x = 0; x < 2; x++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              float product = s[x][i] * f;
              asm volatile("" : "+v"(product));  // not to be fused with the difference
              s[x][i] = own ? (product - ms) * unit : s[x][i];
            }
          ms = own ? 0.f : ms;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[x][i] = exp2_w(!CAP && !BIAS ? fmaf(s[x][i], f, -ms) : s[x][i] - ms);
        l += s[x][i];
      }
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float p0 = s[x][2 * i], p1 = s[x][2 * i + 1];
        if constexpr (F16) {
          P[2 * x + i] = pack_f16x2(p0, p1);
        } else {  // the upper halves as they are, and the rest
          P[2 * x + i] = __builtin_amdgcn_perm(as_u32(p1), as_u32(p0), 0x07060302u);
          R[2 * x + i] = pack_bf16x2(p0 - as_f32(as_u32(p0) & 0xffff0000u), p1 - as_f32(as_u32(p1) & 0xffff0000u));
        }
      }
    }
  }
};

// Values that are not finite, out of v: where +inf (or NaN) stood, plus is 1, where -inf (or NaN), minus.
template <bool F16>
__device__ __forceinline__ u32x4 finite_part(u32x4 v, u32x4& plus, u32x4& minus) {
  constexpr unsigned INF = F16 ? 0x7c00u : 0x7f80u, ONE = F16 ? 0x3c00u : 0x3f80u, BOTH = 0x10001u;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const unsigned w = v[i], size = w & 0x7fff7fffu;
    const unsigned nan = (size + (0x7fffu - INF) * BOTH) & 0x80008000u, inf = (size + (0x8000u - INF) * BOTH) & 0x80008000u;
    plus[i] = (((inf & ~w) | nan) >> 15) * ONE;
    minus[i] = (((inf & w) | nan) >> 15) * ONE;
    v[i] = w & ~((inf >> 15) * 0xffffu);
  }
  return v;
}

// Page `blk` of the sample for a wave's MB tiles, its keys and values at kl and vl in LDS; gone: it is no page, and nobody sees its keys.
// keys_read and values_read run once the one and the other are in registers, values_there before these are read.
template <int MB, bool F16, int HD, bool CAP, bool BIAS, class A, class B, class C>
__device__ __forceinline__ void step(Tile<F16, HD, CAP, BIAS>* t, const AttnArgs& a, const unsigned char* kl, const unsigned char* vl, int blk,
                                     bool gone, A&& keys_read, B&& values_there, C&& values_read) {
  constexpr int KS = HD / 32, NT = HD / 16;
  const int lane = threadIdx.x & 63, r = lane & 15, qq = lane >> 4;
  u32x4 kc[2][KS];
#pragma unroll
  for (int i = 0; i < KS; i++)
#pragma unroll
    for (int x = 0; x < 2; x++) kc[x][i] = *reinterpret_cast<const u32x4*>(kl + ((4 * i + qq) * BT + 16 * x + r) * 16);
  keys_read();
  f32x4 s[MB][2];
#pragma unroll
  for (int n = 0; n < MB; n++)
#pragma unroll
    for (int x = 0; x < 2; x++) {
      s[n][x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; i++) s[n][x] = mma<F16>(kc[x][i], t[n].q[i], s[n][x]);
    }
  u32x4 P[MB], R[MB];
#pragma unroll
  for (int n = 0; n < MB; n++) t[n].weigh(a, s[n], blk, gone, P[n], R[n]);
  int lo = t[0].lo, hi = t[0].hi;
#pragma unroll
  for (int n = 1; n < MB; n++) lo = min(lo, t[n].lo), hi = max(hi, t[n].hi);
  values_there();
  u32x4 vc[NT];  // keys key0 .. key0 + 7 of dim 16 j + r
#pragma unroll
  for (int j = 0; j < NT; j++) vc[j] = *reinterpret_cast<const u32x4*>(vl + (qq * HD + 16 * j + r) * 16);
  values_read();
  // Values of keys that a row does not see must not reach it: its P is 0 there, but 0 x NaN is NaN. Those behind the last key that
  // any row sees are cleared. Where one between low and high is not finite, the product is taken without such values, and rows that see
  // them get their infinities: products of ones count these (both for a NaN). With 256 dims each column has a product of its own.
  const int key0 = blk * BT + 8 * qq, low = gone ? 0 : lo, high = gone ? 0 : hi;
  bool apart = false;
  if (blk * BT + BT > low) {
    const u32x4 some = halves_below(high - key0), each = halves_below(low - key0);
    unsigned bad = 0;
#pragma unroll
    for (int j = 0; j < NT; j++) {
      vc[j] &= some;
#pragma unroll
      for (int i = 0; i < 4; i++) bad |= not_finite<F16>(vc[j][i]) & ~each[i];
    }
    apart = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
  }
  if constexpr (HD == 256) {  // (products of ones took registers: 4 x 256 tokens of 8 heads over 4096 keys 154 us, 140 so)
    static_assert(MB == 1, "one tile of 256 dims");
    if (apart) {
      const int own = gone ? 0 : t->limit;
#pragma unroll 1
      for (int c = 0; c < 16; c++) {
        const u32x4 mine = halves_below(__builtin_amdgcn_readlane(own, c) - key0);
#pragma unroll
        for (int j = 0; j < NT; j++) {
          f32x4 o = mma<F16>(vc[j] & mine, P[0], t->O[j]);
          if constexpr (!F16) o = mma<F16>(vc[j] & mine, R[0], o);
          if (r == c) t->O[j] = o;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      return;
    }
  } else if (apart) {
    u32x4 sees[MB];
#pragma unroll
    for (int n = 0; n < MB; n++) sees[n] = halves_below((gone ? 0 : t[n].limit) - key0) & (F16 ? 0x3c003c00u : 0x3f803f80u);
#pragma unroll
    for (int j = 0; j < NT; j++) {
      u32x4 plus, minus;
      vc[j] = finite_part<F16>(vc[j], plus, minus);
#pragma unroll
      for (int n = 0; n < MB; n++) {
        const f32x4 p = mma<F16>(plus, sees[n], f32x4{0.f, 0.f, 0.f, 0.f}), m = mma<F16>(minus, sees[n], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int i = 0; i < 4; i++) t[n].O[j][i] += (p[i] > 0.f ? INFINITY : 0.f) + (m[i] > 0.f ? -INFINITY : 0.f);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int n = 0; n < MB; n++) {
      t[n].O[j] = mma<F16>(vc[j], P[n], t[n].O[j]);
      if constexpr (!F16) t[n].O[j] = mma<F16>(vc[j], R[n], t[n].O[j]);
    }
}

// The pages of a sample that a wave goes over, blk, blk + step, .., one after the other: 64 are held in the lanes (looked up one by one, by
// scalar loads, each step waited for the one of the step after it: LDS reads and scalar loads share a counter).
struct Pages {
  const int* table;
  int pages, nb, blk, step, left, held;
  __device__ __forceinline__ Pages(const AttnArgs& a, int b, int nb, int first, int step)
      : table(a.table + b * a.ts), pages(a.pages), nb(nb), blk(first), step(step), left(0), held(0) {}
  // The next one's number, 0 behind the last; where there are no more in the lanes, all copies under way are waited for.
  __device__ __forceinline__ int next() {
    if (left == 0) {
      const int64_t mine = blk + (int64_t)step * (threadIdx.x & 63);
      held = mine < nb ? table[mine] : 0;
      asm volatile("" : "+v"(held));
      left = 64;
    }
    blk += step;
    return __builtin_amdgcn_readlane(held, 64 - left--);
  }
  __device__ __forceinline__ bool there(int pg) const { return (unsigned)pg < (unsigned)pages; }
  __device__ __forceinline__ size_t read(int pg) const { return there(pg) ? pg : 0; }  // the first one, where there is none
};

template <int HD>
using Lds = newest::Lds<HD, 2 * BT * HD * 2>;  // of a wave: a page of keys and one of values

template <bool F16, int HD, bool CAP, bool BIAS, int MB>
__global__ void __launch_bounds__(64 * W, HD == 256 ? 1 : HD == 128 || MB > 1 ? 2 : HD == 96 ? 3 : 4) attn_kernel(AttnArgs a) {
  constexpr int PAGE = BT * HD * 2, NC = PAGE / 1024;  // NC: copies of a page
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const Place here = newest::place_of(a);
  if (!here.there) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span sp = newest::span_of(a, here.b);
  if (here.split > 0 && here.split >= newest::splits_used(a, (sp.len + BT - 1) / BT)) return;  // of a short sample: 48 of 1 to 8192 keys 34.4 us, 32.8 so
  Tile<F16, HD, CAP, BIAS> tile[MB];
  int hi = 0;
#pragma unroll
  for (int n = 0; n < MB; n++) {
    tile[n].begin(a, here, sp, here.rt * MB + n);
    hi = max(hi, tile[n].hi);
  }
  const int nb = (hi + BT - 1) / BT;
  const int used = newest::splits_used(a, nb);
  if (here.split >= used) return;
  const int at = here.split * W + wave, all = used * W;
  Pages pages(a, here.b, nb, at, all);
  unsigned char* kl = lds + wave * Lds<HD>::WAVE;
  unsigned char* vl = kl + PAGE;
  const unsigned at_k = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)kl), at_v = at_k + PAGE;
  const unsigned keys_at = key_offset(lane), values_at = lane * 16;
  auto copy = [&](const unsigned char* from, int pg, unsigned to, unsigned off) {
    const unsigned char* p = from + (pages.read(pg) * a.H + here.h) * PAGE;
#pragma unroll
    for (int i = 0; i < NC; i++) copy_to_lds(p + i * 1024, off, to + i * 1024);
  };
  int pg = pages.next();
  if (at < nb) {
    copy(a.k, pg, at_k, keys_at);
    copy(a.v, pg, at_v, values_at);
  }
#pragma unroll
  for (int n = 0; n < MB; n++) tile[n].arrive();
  for (int blk = at; blk < nb; blk += all) {
    const bool more = blk + all < nb;
    const int next = more ? pages.next() : 0;
    vm_wait<NC>();  // the keys; the values are still on their way
    step<MB>(
        tile, a, kl, vl, blk, !pages.there(pg),
        [&] {
          lds_wait();
          if (more) copy(a.k, next, at_k, keys_at);
        },
        [&] {
          if (more) vm_wait<NC>();
          else vm_wait<0>();
        },
        [&] {
          lds_wait();
          if (more) copy(a.v, next, at_v, values_at);
        });
    pg = next;
  }
#pragma unroll
  for (int n = 0; n < MB; n++) {
    Place at_n = here;
    at_n.rt = here.rt * MB + n;
    if (at_n.rt < a.RT) newest::meet<F16, HD, Lds<HD>>(a, at_n, sp, used, lds, tile[n].O, tile[n].m, cols_sum(tile[n].l));
  }
}

template <bool F16, int HD>
__global__ void __launch_bounds__(256) join_kernel(AttnArgs a) {
  newest::join<F16, HD>(a);
}

// Row tiles of a wave: two where there are many of them over many pages (us with one and with two; heads / K/V heads, dims): 1024 tokens
// over 8192 keys, 32 / 8, 128 319 and 239 (fp16 296 and 214), 96 234 and 205, 64 172 and 160; 512 over 4096, 32 / 8, 128 88 and 69; 1024 over 1024
// 44 and 39; 128 over 131072, 8 / 1 173 and 136; 8 x 512 over 2048, 16 / 4, 96 123.5 and 122.9. Fewer leave CUs idle: 293 over 4011, 1500 and 293, 8 / 1,
// 128 39 and 58; 4 x 50 over 1018 12 and 18; and two to four tiles in all read each page once or twice as it is: 32 x 8 over 4096, 32 / 8 98 and 107.
// (8 x 512 over 1024, 16 / 4, 96, on this side of it, 69 and 74.5.) 256 dims do not fit into the registers twice.
int tiles_for(int batch, int tokens, int heads, int kv_heads, int hd, int pages) {
  const int64_t rt = ((int64_t)tokens * (heads / kv_heads) + 15) / 16;
  return hd <= 128 && rt >= 8 && (double)rt * batch * kv_heads * pages >= 65536.0 ? 2 : 1;  // (past 64 bits at the limits)
}

// A wave takes about 2.3 us for a page of 256 dims (1.2 of 128 and less); more than one workgroup a CU (two) share its bandwidth. That
// is for samples that fill their tables. Where one tile of rows is all there is (single tokens), samples are of any age, and a
// full one that takes few splits is waited for: up to 8 splits of 4 pages a wave or more. (Samples of 1 to 8192 tokens by the estimate and so, then
// of 4096 each, us; samples x K/V heads, 4 of 128 dims: 384 64 and 47, 141 and 153; 256 74 and 37, 96 and 103; 192 38 and 29, 75 and 79; 128
// 28.6 and 21.5, 52 and 54; 256 dims: 64 42 and 33, 54 and 59; 48 36 and 27, 44 and 49. Past 64, where shorter samples are enough to fill the
// chip, the one gains more than the other loses; 32 and fewer take as many by the estimate. 16 splits for 192 32.5 instead of 33.)
int splits_for(int batch, int tokens, int heads, int kv_heads, int hd, int pages) {
  const int tiles = tiles_for(batch, tokens, heads, kv_heads, hd, pages);
  if (tiles > 1)
    return std::min(newest::FUSED, newest::splits_for(batch, tokens, heads, kv_heads, pages, 1.8, 2.0, tiles));  // a second kernel joins single tiles
  const int s = newest::splits_for(batch, tokens, heads, kv_heads, pages, hd == 256 ? 2.3 : 1.2, hd == 256 ? 1.0 : 2.0);
  const int64_t units = (int64_t)batch * kv_heads;
  if ((int64_t)tokens * (heads / kv_heads) > 16 || units < 64) return s;
  return (int)std::max<int64_t>(s, std::min<int64_t>({8, (pages + 4 * W - 1) / (4 * W), newest::MAX_PARTS / units}));
}

template <bool F16, int HD>
int launch_attn(const AttnArgs& a, hipStream_t s) {
  const unsigned grid = newest::grid_of(a);
  if (!grid) return host::fail(FA_ERR_INVALID_ARG, "fa_paged_attention: too many rows for one call");
  const bool cap = a.cap > 0.f, bias = a.slopes != nullptr;
  void (*k)(AttnArgs) = cap ? (bias ? attn_kernel<F16, HD, true, true, 1> : attn_kernel<F16, HD, true, false, 1>)
                            : (bias ? attn_kernel<F16, HD, false, true, 1> : attn_kernel<F16, HD, false, false, 1>);
  if constexpr (HD <= 128)
    if (a.RU < a.RT)
      k = cap ? (bias ? attn_kernel<F16, HD, true, true, 2> : attn_kernel<F16, HD, true, false, 2>)
              : (bias ? attn_kernel<F16, HD, false, true, 2> : attn_kernel<F16, HD, false, false, 2>);
  const unsigned lds = Lds<HD>::BYTES;
  const int rc = host::allow_lds(reinterpret_cast<const void*>(k), lds, "fa_paged_attention");
  if (rc != FA_OK) return rc;
  hipLaunchKernelGGL(k, dim3(grid), dim3(64 * W), lds, s, a);
  if (a.S > newest::FUSED) hipLaunchKernelGGL((join_kernel<F16, HD>), dim3(newest::join_grid(a, HD)), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return host::fail(FA_ERR_LAUNCH, "fa_paged_attention: %s", hipGetErrorString(e));
  return FA_OK;
}

template <bool F16>
int launch_attn(const AttnArgs& a, int hd, hipStream_t s) {
  if (hd == 64) return launch_attn<F16, 64>(a, s);
  if (hd == 96) return launch_attn<F16, 96>(a, s);
  if (hd == 128) return launch_attn<F16, 128>(a, s);
  return launch_attn<F16, 256>(a, s);
}

int check_pool(const void* k, const void* v, const int* table, int batch, int heads, int hd, int pages, int width, int64_t stride,
               const char* who);  // paged.hip

}  // namespace paged
}  // namespace fa

extern "C" size_t fa_paged_attention_workspace_bytes(int batch, int tokens, int heads, int kv_heads, int head_dim, int table_pages) {
  if (batch < 1 || tokens < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads || head_dim < 1 || table_pages < 1) return 0;
  return fa::newest::workspace(fa::paged::splits_for(batch, tokens, heads, kv_heads, head_dim, table_pages), batch, tokens, heads,
                               kv_heads, head_dim);
}

extern "C" int fa_paged_attention(const fa_paged_attn_args* a, fa_stream_t stream) {
  using namespace fa;
  const char* who = "fa_paged_attention";
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  int rc = paged::check_pool(a->pool_k, a->pool_v, a->table, a->batch, a->kv_heads, a->head_dim, a->pages, a->table_pages,
                             a->table_stride, who);
  if (rc != FA_OK) return rc;
  rc = newest::check_call(a, who);
  if (rc != FA_OK || a->tokens == 0) return rc;
  paged::AttnArgs p{};
  p.k = static_cast<const unsigned char*>(a->pool_k), p.v = static_cast<const unsigned char*>(a->pool_v);
  p.table = a->table, p.ts = a->table_stride, p.pages = a->pages;
  rc = newest::set_up(p, a, a->table_pages, paged::splits_for(a->batch, a->tokens, a->heads, a->kv_heads, a->head_dim, a->table_pages),
                      paged::tiles_for(a->batch, a->tokens, a->heads, a->kv_heads, a->head_dim, a->table_pages), who);
  if (rc != FA_OK) return rc;
  rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  return a->dtype == FA_DTYPE_F16 ? paged::launch_attn<true>(p, a->head_dim, (hipStream_t)stream)
                                  : paged::launch_attn<false>(p, a->head_dim, (hipStream_t)stream);
}
