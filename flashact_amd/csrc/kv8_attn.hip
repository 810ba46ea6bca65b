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

namespace fa {
namespace kv8 {

constexpr int BT = 32;
constexpr float LOG2E = 1.4426950408889634f;

struct AttnArgs {
  const unsigned char* q;
  int64_t qb, qt, qh;  // strides in elements
  const unsigned char *k, *v;
  const float *ks, *vs;
  const int *lens, *count;
  const float* slopes;
  unsigned char* out;
  float* part;  // [sample][head][row tile][split] {O[16][hd], {m, l}[16]}
  uint64_t *arrived, nonce;  // [sample][head][row tile][FUSED], where the last workgroup joins the splits
  int B, T, H, G, nblk, RT, RC, S, least, causal;  // RT row tiles of a head, RC of them side by side on an XCD
  float scale, over, cap;  // base 2: scale log2(e); capped, scale / cap and cap log2(e)
};

// The row tile's share of what its sample has cached.
struct Span {
  int len, n;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, int b) {
  const int cap = (int)min((int64_t)a.nblk * BT, (int64_t)0x7fffffff - 31);
  Span s;
  s.len = max(0, min(a.lens[b], cap));
  s.n = a.count ? max(0, min(a.count[b], a.T)) : a.T;
  return s;
}
// The reference of weights whose scores (base 2) have the maximum `top`; past 2^22, where the difference would round, itself.
__device__ __forceinline__ float reference(float top) { return fabsf(top) < 4194304.f ? top - 15.f : top; }
// Both sums, of weighted values and of weights, are kept times 2^-35. With weights of up to 2^15 a key adds at most 2^-20 of its
// value: a million keys of the largest values stay in the fp32 range, and those of the smallest scale (2^-100) above its end.
constexpr float SMALL = 0x1p-35f;
constexpr int W = 4;  // waves of a workgroup
// Splits that a row tile of nb blocks uses: each wave of each has a.least blocks or more.
constexpr int MAX_SPLITS = 256;
// Up to so many are joined by the last workgroup (32 requests of 50 to 16384 keys on 16 splits: 20.6 us, 22.6 with a kernel), more
// by a kernel with workgroups enough to read them.
constexpr int FUSED = 16;
__device__ __forceinline__ int splits_used(const AttnArgs& a, int nb) {
  const unsigned per = W * a.least;
  return max(1, min(a.S, (int)((nb + per - 1) / per)));
}

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

template <bool F16>
__device__ __forceinline__ void store_row4(unsigned char* out, size_t at, f32x4 v) {
  if constexpr (F16)
    *reinterpret_cast<u32x2*>(out + at * 2) = u32x2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
  else
    *reinterpret_cast<u32x2*>(out + at * 2) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

// 1 / l of a row: no keys give zeros, NaN stays.
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Waits until at most N copies to LDS (or loads) of this wave are outstanding.
template <int N>
__device__ __forceinline__ void vm_wait() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
  asm volatile("" ::: "memory");
}
// this wave's LDS reads have returned
__device__ __forceinline__ void lds_wait() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <int HD>
struct Lds {
  static constexpr int PITCH = HD + 4;                               // of the waves' sums
  static constexpr int WAVE = 2 * BT * HD;                           // a block of keys and one of values
  static constexpr int SUM = W * 16 * PITCH * 4 > W * WAVE ? W * 16 * PITCH * 4 : W * WAVE;
  static constexpr int BYTES = SUM + 2 * W * 16 * 4;
};

template <bool F16, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(64 * W, HD == 256 ? 2 : HD == 128 ? 3 : 4) attn_kernel(AttnArgs a) {
  constexpr int KS = (HD + 63) / 64, NT = HD / 16, NC = BT * HD / 1024;  // NC: copies of a block
  constexpr int PITCH = Lds<HD>::PITCH;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  float* osum = reinterpret_cast<float*>(lds);
  float* wm = reinterpret_cast<float*>(lds + Lds<HD>::SUM);
  float* wl = wm + W * 16;

  // Row tiles of one (split, sample, head) share their keys: RC neighbours on one XCD. Splits are the slowest index: samples
  // that leave the later ones unused would else leave XCDs unused (64 samples of 1050 keys on 16 splits: 72 us instead
  // of 21); within a split the runs of row tiles are turned, so that the splits of one meet on different XCDs.
  const unsigned xcd = blockIdx.x & 7, y = blockIdx.x >> 3, yr = y / (unsigned)a.RC, u = yr * 8 + xcd;
  const unsigned runs = (a.RT + a.RC - 1) / a.RC, all_runs = a.B * a.H * runs;
  const int split = u / all_runs;
  unsigned turned = u - split * all_runs + (all_runs >= 8 ? (split * (all_runs - 1)) & 7 : 0);
  if (turned >= all_runs) turned -= all_runs;
  const int bh = turned / runs, b = bh / (unsigned)a.H, h = bh - b * a.H;
  const int rt = (turned - bh * runs) * a.RC + y - yr * a.RC;
  if (split >= a.S || rt >= a.RT) return;
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
    // scores in base 2
    const int key0 = blk * BT + 8 * q;
    const bool mixed = blk * BT + BT > lo;
    if constexpr (CAP) {
      float most = 0.f;
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s[x][i] *= ksc * a.over;
          most = fmaxf(most, fabsf(s[x][i]));
        }
      if (__builtin_amdgcn_ballot_w64(most > kTanhNear) == 0) {
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int i = 0; i < 4; i++) s[x][i] = a.cap * tanh_near(s[x][i]);
      } else {
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int i = 0; i < 4; i++) s[x][i] = a.cap * tanh_own(s[x][i], s[x][i] * (2.f * LOG2E));
      }
    } else {
      const float f = ksc * a.scale;
      s[0] *= f;
      s[1] *= f;
    }
    float mx = -INFINITY;
    if constexpr (BIAS) {
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[x][i] -= slope * fabsf((float)(pos - (key0 + 4 * x + i)));
    }
    if (mixed) {
      asm volatile("");  // a branch: as selects the masks cost every block
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (key0 + 4 * x + i >= limit) s[x][i] = -INFINITY;
    }
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[x][i]);
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

  // the waves' sums
  l = cols_sum(l) * SMALL;
  __syncthreads();  // the blocks in LDS are done with
  if (q == 0) {
    wm[wave * 16 + r] = m;
    wl[wave * 16 + r] = l;
  }
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; w++) M = fmaxf(M, wm[w * 16 + r]);
  const float mine = m == -INFINITY ? 0.f : exp2_w(m - M);
  constexpr int ONE = 16 * HD + 32;
  const rsrc_t part = make_rsrc(a.part + ((size_t)bh * a.RT + rt) * a.S * ONE, 0xffffffffu);  // the tile's splits
#pragma unroll
  for (int j = 0; j < NT; j++)
    *reinterpret_cast<f32x4*>(osum + (wave * 16 + r) * PITCH + 16 * j + 4 * q) = mine * O[j];
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * HD / 4; e += 64 * W) {
    const int row = e / (HD / 4), d = e % (HD / 4) * 4, g = rt * 16 + row;
    if (g >= a.T * a.G) continue;
    float rm = -INFINITY, rl = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) rm = fmaxf(rm, wm[w * 16 + row]);
#pragma unroll
    for (int w = 0; w < W; w++) rl += wm[w * 16 + row] == -INFINITY ? 0.f : wl[w * 16 + row] * exp2_w(wm[w * 16 + row] - rm);
    f32x4 o = *reinterpret_cast<const f32x4*>(osum + row * PITCH + d);
#pragma unroll
    for (int w = 1; w < W; w++) o += *reinterpret_cast<const f32x4*>(osum + (w * 16 + row) * PITCH + d);
    if (used > 1) {
      stb128<kCpSc1>(part, (split * ONE + row * HD + d) * 4, __builtin_bit_cast(u32x4, o));
      if (d == 0) stb64<kCpSc1>(part, (split * ONE + 16 * HD + 2 * row) * 4, __builtin_bit_cast(u32x2, f32x2{rm, rl}));
    } else {
      const int tt = g / a.G;
      if (tt >= sp.n || sp.len - sp.n + tt < 0) o = f32x4{0.f, 0.f, 0.f, 0.f}, rl = 0.f;
      store_row4<F16>(a.out, ((size_t)b * a.T + tt) * a.H * a.G * HD + (size_t)(h * a.G + g % a.G) * HD + d,
                      o * inverse(rl));
    }
  }
  if (used == 1 || a.S > FUSED) return;
  // The last of the tile's workgroups joins its splits, in their order. (One token of 983 keys on eight splits: 9.4 us, 9.7 with
  // a second kernel to join, 11.4 with a counter per tile by compare and exchange, which eight that arrive together retry; 48
  // requests: 24.1, 26.1 with the kernel.)
  if (!arrived_last(a.arrived + ((size_t)bh * a.RT + rt) * FUSED, a.nonce, split, used, reinterpret_cast<int*>(wm))) return;
  f32x2* ml = reinterpret_cast<f32x2*>(lds);
  static_assert(16 * FUSED <= 64 * W, "a split's row a thread");
  const int rows = min(16, a.T * a.G - rt * 16), own = threadIdx.x;
  f32x2 mine_ml = f32x2{-INFINITY, 0.f};
  if (own < 16 * used) mine_ml = __builtin_bit_cast(f32x2, ldb64<kCpSc1>(part, ((own >> 4) * ONE + 16 * HD + 2 * (own & 15)) * 4));
  constexpr int PER = HD / 4;  // quads of dims of a row
  for (int base = 0; base < rows * PER; base += 64 * W) {
    const int e = base + threadIdx.x, row = e / PER, g = rt * 16 + row, tt = g / a.G;
    const bool there = e < rows * PER;
    f32x4 x[FUSED];
#pragma unroll
    for (int s = 0; s < FUSED; s++)
      if (s < used && there) x[s] = __builtin_bit_cast(f32x4, ldb128<kCpSc1>(part, (s * ONE + e * 4) * 4));
    if (base == 0) {
      if (own < 16 * FUSED) ml[own] = mine_ml;
      __syncthreads();
    }
    if (!there) continue;
    float rm = -INFINITY, rl = 0.f;
#pragma unroll
    for (int s = 0; s < FUSED; s++) rm = fmaxf(rm, ml[s * 16 + row][0]);
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < FUSED; s++)
      if (s < used) {
        const f32x2 v = ml[s * 16 + row];
        const float w = v[0] == -INFINITY ? 0.f : exp2_w(v[0] - rm);
        rl += w * v[1];
        o += w * x[s];
      }
    if (tt >= sp.n || sp.len - sp.n + tt < 0) o = f32x4{0.f, 0.f, 0.f, 0.f}, rl = 0.f;
    store_row4<F16>(a.out, ((size_t)b * a.T + tt) * a.H * a.G * HD + (size_t)(h * a.G + g % a.G) * HD + e % PER * 4, o * inverse(rl));
  }
}

// The splits' sums, in a fixed order, where there are more than FUSED. One workgroup: 64 dims (96) of
// one row; nothing to do where its sample used one split. Threads are quads of dims x groups of splits, so that 16 splits are
// read side by side (2 x 131072 keys on 128 splits: 32.3 us, 32.8 with all 256 dims in one workgroup).
template <bool F16, int HD>
__global__ void __launch_bounds__(256) join_kernel(AttnArgs a) {
  constexpr int DIMS = HD % 64 == 0 ? 64 : HD, SLOTS = DIMS / 4, GROUPS = 256 / SLOTS, RUNS = HD / DIMS;
  __shared__ float wt[MAX_SPLITS], red[8];
  __shared__ f32x4 sums[GROUPS][SLOTS];
  const int rows = a.T * a.G, unit = blockIdx.x / RUNS, run = blockIdx.x % RUNS;
  const int g = unit % rows, bh = unit / rows, h = bh % a.H, b = bh / a.H;
  const int rt = g >> 4, row = g & 15, t = g / a.G;
  const Span sp = span_of(a, b);
  int hi = 0;  // as the attention found it: the keys that the tile's last row sees
  if (rt * 16 / a.G < sp.n) {
    const int last = min(min(rt * 16 + 15, rows - 1) / a.G, sp.n - 1), pos = sp.len - sp.n + last;
    hi = pos < 0 ? 0 : a.causal ? pos + 1 : sp.len;
  }
  const int used = splits_used(a, (hi + BT - 1) / BT);
  if (used == 1) return;
  constexpr int ONE = 16 * HD + 32;
  const float* part = a.part + ((size_t)bh * a.RT + rt) * a.S * ONE;
  const int i = threadIdx.x, wave = i >> 6;
  const f32x2 ml = i < used ? *reinterpret_cast<const f32x2*>(part + (size_t)i * ONE + 16 * HD + 2 * row) : f32x2{-INFINITY, 0.f};
  const float ms = ml[0], ls = ml[1];
  float x = wave_max(ms);
  if ((i & 63) == 0) red[wave] = x;
  __syncthreads();
  const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float w = ms == -INFINITY ? 0.f : exp2_w(ms - M);
  wt[i] = w;
  x = wave_sum(w * ls);
  if ((i & 63) == 0) red[4 + wave] = x;
  __syncthreads();
  float L = red[4] + red[5] + red[6] + red[7];
  const int d = run * DIMS + (i % SLOTS) * 4, grp = i / SLOTS;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  if (grp < GROUPS) {
#pragma unroll 8
    for (int s = grp; s < used; s += GROUPS) o += wt[s] * *reinterpret_cast<const f32x4*>(part + (size_t)s * ONE + row * HD + d);
    sums[grp][i % SLOTS] = o;
  }
  __syncthreads();
  if (i >= SLOTS) return;
  o = sums[0][i];
#pragma unroll
  for (int s = 1; s < GROUPS; s++) o += sums[s][i];
  if (t >= sp.n || sp.len - sp.n + t < 0) o = f32x4{0.f, 0.f, 0.f, 0.f}, L = 0.f;
  store_row4<F16>(a.out, ((size_t)b * a.T + t) * a.H * a.G * HD + (size_t)(h * a.G + g % a.G) * HD + d, o * inverse(L));
}

// Splits of all row tiles together: they bound the workspace (68 MB with 256 dims), where whole rounds of workgroups alone would ask
// for gigabytes beside a small cache. 2049 tokens of 8 heads of 256 dims over 8192 keys 354 us, unbounded (135 MB) 440, over 32768 keys
// 1360 and 1275; 4152 of 128 dims 244 and 276, 1143 and 1085; 4 x 2080 of 64 dims over 16384 keys 643 and 603.
constexpr int MAX_PARTS = 4096;

// Splits of the keys across workgroups. A wave takes about 2.3 us for a block of 256 dims that comes from memory (1.2 of 128
// and less) and one to begin and end, more than one (four) workgroups a CU share its bandwidth, and joining the splits costs
// 3 us: the number with the least estimate, for samples that fill the cache (their lengths are on the GPU), is taken (within
// 10 % of the best of eleven counts in nine of eleven shapes, 17 % in the others). Shorter ones use fewer.
int splits_for(int batch, int tokens, int heads, int kv_heads, int hd, int blocks) {
  const int64_t rt = ((int64_t)tokens * (heads / kv_heads) + 15) / 16, units = rt * batch * kv_heads;
  const double block = hd == 256 ? 2.3 : 1.2, resident = hd == 256 ? 1.0 : 4.0;
  const int64_t most = std::min<int64_t>({(blocks + W - 1) / W, MAX_SPLITS, std::max<int64_t>(1, MAX_PARTS / units)});
  int best = 1;
  double least = 1e300;
  auto consider = [&](int64_t S) {
    if (S < 1 || S > most) return;
    const int64_t each = (blocks + W * S - 1) / (W * S);
    const double t = (block * each + 1.0) * std::max(1.0, (units * S + 255) / 256 / resident) + (S > 1 ? 3.0 : 0.0);
    if (t < least) best = (int)S, least = t;
  };
  for (int64_t S = 1; S <= most; S += std::max<int64_t>(1, S / 4)) consider(S);
  for (int64_t n = 1; n <= 4; n *= 2) consider(256 * n / units);  // whole rounds of workgroups
  return best;
}

size_t arrived_bytes(size_t tiles) { return (tiles * FUSED * sizeof(uint64_t) + 255) / 256 * 256; }

size_t attn_workspace(int batch, int tokens, int heads, int kv_heads, int hd, int blocks) {
  const int S = splits_for(batch, tokens, heads, kv_heads, hd, blocks);
  if (S == 1) return 0;
  const size_t rt = ((size_t)tokens * (heads / kv_heads) + 15) / 16;
  return (S <= FUSED ? arrived_bytes(rt * batch * kv_heads) : 0) + rt * batch * kv_heads * S * (16 * hd + 32) * sizeof(float);
}

template <bool F16, int HD>
int launch_attn(const AttnArgs& a, hipStream_t s) {
  const int runs = (a.RT + a.RC - 1) / a.RC;
  const int64_t grid = ((int64_t)a.B * a.H * a.S * runs + 7) / 8 * 8 * a.RC;
  if (grid > 0x7fffffff) return host::fail(FA_ERR_INVALID_ARG, "fa_kv8_attention: too many rows for one call");
  const bool cap = a.cap > 0.f, bias = a.slopes != nullptr;
  void (*k)(AttnArgs) = cap ? (bias ? attn_kernel<F16, HD, true, true> : attn_kernel<F16, HD, true, false>)
                            : (bias ? attn_kernel<F16, HD, false, true> : attn_kernel<F16, HD, false, false>);
  const unsigned lds = Lds<HD>::BYTES;
  const int rc = host::allow_lds(reinterpret_cast<const void*>(k), lds, "fa_kv8_attention");
  if (rc != FA_OK) return rc;
  hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(64 * W), lds, s, a);
  if (a.S > FUSED)
    hipLaunchKernelGGL((join_kernel<F16, HD>), dim3((unsigned)(a.B * a.H * a.T * a.G * (HD % 64 == 0 ? HD / 64 : 1))), dim3(256), 0, s, a);
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
  return fa::kv8::attn_workspace(batch, tokens, heads, kv_heads, head_dim, blocks);
}

extern "C" int fa_kv8_attention(const fa_kv8_attn_args* a, fa_stream_t stream) {
  using namespace fa;
  const char* who = "fa_kv8_attention";
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  int rc = kv8::check_cache(a->cache_k, a->cache_v, a->cache_ks, a->cache_vs, a->batch, a->kv_heads, a->head_dim, a->blocks, who);
  if (rc != FA_OK) return rc;
  if (a->dtype != FA_DTYPE_BF16 && a->dtype != FA_DTYPE_F16)
    return host::fail(FA_ERR_INVALID_ARG, "%s: dtype %d: q is bf16 or fp16", who, a->dtype);
  if (a->heads < 1 || a->heads > (1 << 16) || a->heads % a->kv_heads)
    return host::fail(FA_ERR_INVALID_ARG, "%s: heads=%d is no multiple of kv_heads=%d", who, a->heads, a->kv_heads);
  if (a->tokens < 0 || (int64_t)a->tokens * a->heads > (1 << 24))
    return host::fail(FA_ERR_INVALID_ARG, "%s: tokens=%d x heads=%d outside [0, 2^24]", who, a->tokens, a->heads);
  if (!(a->softcap >= 0.f) || !(a->softcap < INFINITY) || !(fabsf(a->scale) < INFINITY))
    return host::fail(FA_ERR_INVALID_ARG, "%s: scale=%g and softcap=%g must be finite, softcap >= 0", who, a->scale,
                      a->softcap);
  if (a->tokens == 0) return FA_OK;
  if (!a->q || !a->out || !a->lens) return host::fail(FA_ERR_INVALID_ARG, "%s: q, out or lens is NULL", who);
  if (reinterpret_cast<uintptr_t>(a->q) % 16 || reinterpret_cast<uintptr_t>(a->out) % 16)
    return host::fail(FA_ERR_INVALID_ARG, "%s: q or out is not 16-byte aligned", who);
  if (reinterpret_cast<uintptr_t>(a->lens) % 4 || reinterpret_cast<uintptr_t>(a->count) % 4 ||
      reinterpret_cast<uintptr_t>(a->slopes) % 4)
    return host::fail(FA_ERR_INVALID_ARG, "%s: lens, count or slopes is not 4-byte aligned", who);
  for (int i = 0; i < 3; i++)
    if (a->q_stride[i] % 8)
      return host::fail(FA_ERR_INVALID_ARG, "%s: q_stride[%d]=%lld is no multiple of 8", who, i, a->q_stride[i]);
  const size_t need = kv8::attn_workspace(a->batch, a->tokens, a->heads, a->kv_heads, a->head_dim, a->blocks);
  if (need && (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return host::fail(FA_ERR_INVALID_ARG, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, need,
                      a->workspace ? a->workspace_bytes : (size_t)0);
  kv8::AttnArgs p{};
  p.q = static_cast<const unsigned char*>(a->q);
  p.qb = a->q_stride[0], p.qt = a->q_stride[1], p.qh = a->q_stride[2];
  p.k = static_cast<const unsigned char*>(a->cache_k), p.v = static_cast<const unsigned char*>(a->cache_v);
  p.ks = a->cache_ks, p.vs = a->cache_vs;
  p.lens = a->lens, p.count = a->count, p.slopes = a->slopes;
  p.out = static_cast<unsigned char*>(a->out), p.part = static_cast<float*>(a->workspace);
  p.B = a->batch, p.T = a->tokens, p.H = a->kv_heads, p.G = a->heads / a->kv_heads, p.nblk = a->blocks;
  p.RT = (p.T * p.G + 15) / 16;
  p.S = kv8::splits_for(a->batch, a->tokens, a->heads, a->kv_heads, a->head_dim, a->blocks);
  if (p.S > 1 && p.S <= kv8::FUSED) {
    p.nonce = host::launch_nonce();
    p.arrived = static_cast<uint64_t*>(a->workspace);
    p.part = reinterpret_cast<float*>(static_cast<unsigned char*>(a->workspace) + kv8::arrived_bytes((size_t)p.RT * p.B * p.H));
  }
  // All row tiles of a (split, sample, head) run on one XCD where these divide evenly over the 8, else in runs short enough
  // that there are 32 or more (200 tokens of 8 heads over 1100 keys of one sample 38 -> 21 us; 17.3 -> 17.5 for 4 samples of 50).
  const int64_t groups = (int64_t)p.B * p.H * p.S, runs = groups % 8 ? std::min<int64_t>((31 + groups) / groups, p.RT) : 1;
  p.RC = (int)((p.RT + runs - 1) / runs);
  p.least = (int64_t)p.RT * p.B * p.H >= 64 ? 4 : 1;

  p.causal = a->causal;
  p.scale = a->scale * kv8::LOG2E;
  p.over = a->softcap > 0.f ? a->scale / a->softcap : 0.f;
  p.cap = a->softcap * kv8::LOG2E;
  if (!(fabsf(p.scale) < INFINITY) || !(fabsf(p.over) < INFINITY) || !(p.cap < INFINITY))
    return host::fail(FA_ERR_INVALID_ARG, "%s: scale=%g over softcap=%g leaves the fp32 range", who, a->scale, a->softcap);
  rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  return a->dtype == FA_DTYPE_F16 ? kv8::launch_attn<true>(p, a->head_dim, (hipStream_t)stream)
                                  : kv8::launch_attn<false>(p, a->head_dim, (hipStream_t)stream);
}
