// Attention in which every query has its own span of keys (fa_span_attention): packed prompts, prefixes, windows.
//
//   s_ij = q_i . k_j scale, capped to cap tanh(s / cap), less slope_h |i + Tk - Tq - j|;  o_i = sum_j softmax_j(s_ij) v_j
//   over the keys first_i <= j < last_i; a query whose span is empty gets zeros.
//
// One pass over the keys with a running maximum and sum. The waves of a workgroup take 16 or 32 queries of one head each and
// walk together over the tiles of KT keys between the first key that any of them sees and the last; tiles that all queries of
// a wave see whole skip the masks. S^T = K Q^T and O^T += V^T P^T on the 16x16x32 MFMA: a lane holds one query's column, the
// softmax needs two cross-lane steps, and P^T is already the second product's operand (slot 8 q + j of a 32-key step is key
// 4 q + j of its first 16 for j < 4, key 16 + 4 q + j - 4 beyond), which the values' transposing LDS read matches.
// Where that leaves CUs idle, the keys are split over workgroups too, whose sums meet in a workspace.
// Keys and values of the next tiles are copied to LDS (no registers) while this one is worked on, one barrier a tile. With
// many queries the MFMAs are the bound, next to the LDS reads that feed them (each operand of 1 KB serves 16 or 32 queries)
// and, capped, the three exponentials a score; with few it is one wave's chain of a tile's steps, about 3000 cycles.
// 8191 tokens of 16 heads of 128 dims over 4 K/V heads, causal behind a tenth, capped: 373 us, 745 TFLOP/s.
//
// Rounding: the scores' products are exact in fp32, softmax and sums are fp32, P is rounded to the values' type for the
// second product (bf16 values have a range that fp16 weights times fp16 values would not hold), the result once.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"

namespace fa {
namespace attn {

struct Params {
  const unsigned char *q, *k, *v;
  int64_t qb, qt, qh, kb, vb, kh, vh;  // strides in elements; the token strides of k and v fit 32 bits
  int kt, vt;
  const int* spans;  // [B][Tq][2] or NULL: all keys
  const float* slopes;
  unsigned char* out;  // [B][Tq][H][hd]
  int B, Tq, Tk, H, G, hd, ntile, stages;
  // base 2: scale log2(e); capped, 2 log2(e) scale / cap for tanh_far, scale / cap for tanh_near, and cap log2(e)
  float scale, over, cap;
  int flat;  // the scale is zero: see where the queries are loaded
  // where keys are split over workgroups: into up to S parts of `least` steps or more; the parts that each (tile, sample,
  // head) was split into, and their sums, 64 rows of {O[hd], m, l} each as a wave's lanes hold them
  int S, least;
  int* used;
  float* part;
  uint64_t *arrived, nonce;  // [tile, sample, head][FUSED], where the last workgroup joins the parts
};

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_SPLITS = 256, LEAST = 8;
// Up to so many parts are joined by the last workgroup (1024 queries over 4096 keys 43 -> 37 us, 50 over 1018 with 256 dims 24 -> 23),
// more by a kernel with workgroups enough to read them.
constexpr int FUSED = 4;

// Chunk c (16 bytes) of row `row` lies in LDS slot c ^ turn of the row's CH slots: the same chunk of 16 rows (a key operand)
// and the same pair of chunks of 8 rows (a value operand) meet in different banks.
template <int CH>
__device__ __forceinline__ int turn(int row) {
  if constexpr (CH == 8) return (row & 6) | ((row >> 3) & 1);
  else if constexpr (CH == 12) return ((row >> 1) & 2) | ((row >> 3) & 1);
  else return ((row & 7) << 1) | ((row >> 3) & 1);
}

// Waits until at most N copies or loads of this wave are outstanding.
template <int N>
__device__ __forceinline__ void vm_wait() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
  asm volatile("" ::: "memory");
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
// Four rows of 16 two-byte elements, held by 16 lanes as 8-byte pieces (lane 4 a + p: row a, elements 4 p .. 4 p + 3) ->
// lane i gets element i of the four rows.
__device__ __forceinline__ u32x2 read_turned(const unsigned char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4*)(const_cast<unsigned char*>(p))));
}

template <bool F16>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  return F16 ? pack_f16x2(a, b) : pack_bf16x2(a, b);
}
template <bool F16>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  return F16 ? mfma16h(a, b, c) : mfma16(a, b, c);
}
// sign bit of each half whose fraction is not zero
template <bool F16>
__device__ __forceinline__ unsigned fraction(unsigned x) {
  return F16 ? ((x & 0x03ff03ffu) + 0x7fff7fffu) & 0x80008000u : ((x & 0x007f007fu) + 0x7fff7fffu) & 0x80008000u;
}
// the halves whose sign bit is set, whole
__device__ __forceinline__ unsigned spread(unsigned sign) { return sign | (sign - (sign >> 15)); }

typedef int i32x2 __attribute__((ext_vector_type(2), aligned(4)));

// The least of a row of 16 lanes, in each of them (DPP row_ror).
__device__ __forceinline__ int rows_least(int v) {
  v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, false));
  v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x124, 0xF, 0xF, false));
  v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x122, 0xF, 0xF, false));
  return min(v, __builtin_amdgcn_update_dpp(0, v, 0x121, 0xF, 0xF, false));
}

// The reference of weights whose scores (base 2) have the maximum `top`. In fp16 the largest starts at 2^12 and may grow to 2^15:
// those above 2^-26 of it keep all their bits and the rest is held to 2^-37 of it, where with the maximum at one 65536 keys of
// 2^-26 each were lost. Past 2^22, where the difference would round, it is the maximum. bf16 has the range of fp32.
constexpr float FAR = 4194304.f;  // from here on numbers are half a unit and more apart
template <bool F16>
__device__ __forceinline__ float reference(float top) { return F16 && fabsf(top) < FAR ? top - 12.f : top; }

constexpr int part_floats(int nt) { return nt * 256 + 32; }  // of 16 rows

template <bool F16, int HD, int QB, int NW, int SP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(64 * NW * SP, 2) span_kernel(Params p) {
  constexpr int KT = HD == 256 ? 32 : 64, CH = HD / 8, NK = HD / 32, NT = HD / 16, MT = KT / 16;
  constexpr int TILE = KT * HD * 2, COPIES = KT * CH / 64, PER = COPIES / NW;  // bytes, copies of a tile of keys: all, a wave's
  constexpr unsigned ONE = F16 ? 0x3c00u : 0x3f80u;
  constexpr float PASS = F16 ? 15.f : 8.f;  // how far weights may grow, as powers of two, before the reference follows
  // 4096 for a NaN, 64 for an infinity, 1 for a negative one: the 32 keys of a step sum up without mixing
  constexpr unsigned NANS = (F16 ? 0x6c00u : 0x4580u) * 0x10001u, UPS = (F16 ? 0x5400u : 0x4280u) * 0x10001u;
  constexpr unsigned DOWNS = ONE * 0x10001u;
  static_assert(KT * CH % 64 == 0 && COPIES % NW == 0, "whole copies, as many of each wave");
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];  // p.stages buffers of {keys, values}
  const int lane = threadIdx.x & 63, all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = SP > 1 ? all_waves % NW : all_waves, grp = SP > 1 ? all_waves / NW : 0;  // grp: whose tiles of keys
  const int r = lane & 15, q = lane >> 4;

  // Heads (of all samples) go to XCDs in runs where they divide evenly, so that those that share keys meet in one L2;
  // the last tiles, which see most under a causal span, start first.
  const unsigned heads = p.B * p.H, units = heads * p.ntile, split = SP > 1 ? blockIdx.x / units : 0;
  const unsigned id = SP > 1 ? blockIdx.x - split * units : blockIdx.x;
  unsigned bh, tile;
  if (heads % 8 == 0) {
    const unsigned per = heads / 8, j = id >> 3;
    tile = j / per;
    bh = (id & 7) * per + (j - tile * per);
  } else {
    tile = id / heads;
    bh = id - tile * heads;
  }
  const int b = bh / (unsigned)p.H, h = bh - b * p.H, kvh = h / p.G;
  const int row0 = (p.ntile - 1 - (int)tile) * (16 * QB * NW) + wave * 16 * QB;

  // this lane's queries and the tile's extent; rows behind the last load what it loads and see nothing
  int first[QB], last[QB], lo = 0x7fffffff, hi = 0, all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
  for (int x = 0; x < QB; x++) first[x] = 0, last[x] = p.Tk;
  if (p.spans) {
#pragma unroll
    for (int x = 0; x < QB; x++) {
      const i32x2 s = *reinterpret_cast<const i32x2*>(p.spans + ((size_t)b * p.Tq + min(row0 + 16 * x + r, p.Tq - 1)) * 2);
      first[x] = s[0], last[x] = s[1];
    }
  }
#pragma unroll
  for (int x = 0; x < QB; x++) {
    const bool there = row0 + 16 * x + r < p.Tq;
    first[x] = max(first[x], 0), last[x] = there ? min(last[x], p.Tk) : 0;
    if (first[x] < last[x]) {
      lo = min(lo, first[x]), hi = max(hi, last[x]);
      all_lo = max(all_lo, first[x]), all_hi = min(all_hi, last[x]);
    } else {
      first[x] = last[x] = 0;
      if (there) all_hi = 0;  // a row that sees nothing: every tile is masked
    }
  }
  lo = rows_least(lo), hi = -rows_least(-hi), all_lo = -rows_least(-all_lo), all_hi = rows_least(all_hi);
  int* ext = reinterpret_cast<int*>(lds + p.stages * SP * 2 * TILE);  // the workgroup walks over the keys of all its waves
  if (lane == 0 && grp == 0) {
    ext[2 * wave] = lo;
    ext[2 * wave + 1] = hi;
  }
  // dims behind hd are zero in LDS: the copies never write them
  if (p.hd < HD)
    for (int i = threadIdx.x; i < p.stages * SP * 2 * TILE / 16; i += 64 * NW * SP) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
  u32x4 qf[QB][NK];
#pragma unroll
  for (int x = 0; x < QB; x++)
#pragma unroll
    for (int i = 0; i < NK; i++) {
      const int row = min(row0 + 16 * x + r, p.Tq - 1), d = 32 * i + 8 * q;
      qf[x][i] = u32x4{0, 0, 0, 0};
      if (d < p.hd) qf[x][i] = *reinterpret_cast<const u32x4*>(p.q + (b * p.qb + row * p.qt + h * p.qh + d) * 2);
    }
  const float slope = BIAS ? p.slopes[h] * LOG2E : 0.f;
  __syncthreads();
  int k0 = 0x7fffffff, k1 = 0;
#pragma unroll
  for (int w = 0; w < NW; w++) k0 = min(k0, ext[2 * w]), k1 = max(k1, ext[2 * w + 1]);
  k1 = __builtin_amdgcn_readfirstlane(k1);
  k0 = min(__builtin_amdgcn_readfirstlane(k0), k1);  // a workgroup whose queries see nothing: 0, 0
  int used = 1;
  if constexpr (SP > 1) {
    if (p.S > 1) {
      const int steps = (k1 - k0 + KT * SP - 1) / (KT * SP), parts = max(1, min(p.S, steps / p.least));
      const int per = (steps + parts - 1) / parts;
      used = steps > 0 ? (steps + per - 1) / per : 1;
      if (split == 0 && threadIdx.x == 0) p.used[bh * p.ntile + tile] = used;
      if ((int)split >= used) return;
      k0 += (int)split * per * (KT * SP);
      k1 = min(k1, k0 + per * (KT * SP));
    }
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);

  const unsigned char* kg = p.k + (b * p.kb + kvh * p.kh) * 2;
  const unsigned char* vg = p.v + (b * p.vb + kvh * p.vh) * 2;
  const unsigned lbase = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)lds);
  // Keys [key, key + KT); behind the last one it is repeated, and dims behind hd are left out.
  unsigned koff[PER], voff[PER];  // of the lane's chunks in a whole tile
#pragma unroll
  for (int n = 0; n < PER; n++) {
    const int slot = (n * NW + wave) * 64 + lane, row = slot / CH, c = (slot % CH) ^ turn<CH>(row);
    koff[n] = row * (unsigned)(p.kt * 2) + c * 16;
    voff[n] = row * (unsigned)(p.vt * 2) + c * 16;
  }
  auto copy_tile = [&](int key, int buf) {
    const unsigned char* kp = kg + (int64_t)key * p.kt * 2;
    const unsigned char* vp = vg + (int64_t)key * p.vt * 2;
    const unsigned to = lbase + (buf * SP + grp) * 2 * TILE + wave * 1024;
    if (p.hd == HD && key + KT <= p.Tk) {
#pragma unroll
      for (int n = 0; n < PER; n++) {
        copy_to_lds(kp, koff[n], to + n * NW * 1024);
        copy_to_lds(vp, voff[n], to + n * NW * 1024 + TILE);
      }
      return;
    }
    int ln = lane;
    asm volatile("" : "+v"(ln));  // worked out here each time: no registers to keep it in
#pragma unroll
    for (int n = 0; n < PER; n++) {
      const int slot = (n * NW + wave) * 64 + ln, row = slot / CH, c = (slot % CH) ^ turn<CH>(row);
      const unsigned at = min(row, p.Tk - 1 - key);
      if (c * 8 < p.hd) {
        copy_to_lds(kp, at * (unsigned)(p.kt * 2) + c * 16, to + n * NW * 1024);
        copy_to_lds(vp, at * (unsigned)(p.vt * 2) + c * 16, to + n * NW * 1024 + TILE);
      }
    }
  };

  f32x4 O[QB][NT];
  float m[QB], l[QB];
  uint64_t far[QB];  // lanes of rows whose reference is past FAR
#pragma unroll
  for (int x = 0; x < QB; x++) {
    m[x] = -INFINITY, l[x] = 0.f, far[x] = 0;
#pragma unroll
    for (int j = 0; j < NT; j++) O[x][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // p.stages - 1 tiles are on their way
  constexpr int STEP = KT * SP;
  const int ahead = (p.stages - 1) * STEP;
  for (int i = 0; i < p.stages - 1; i++)
    if (k0 + i * STEP + grp * KT < k1) copy_tile(k0 + i * STEP + grp * KT, i);
  // The queries are waited for here: left to the compiler, that wait (for everything under way) stands in the loop.
#pragma unroll
  for (int x = 0; x < QB; x++)
#pragma unroll
    for (int i = 0; i < NK; i++) asm volatile("" : "+v"(qf[x][i]));
  // A scale of zero would take masked scores (-inf) to NaN as the unit of a tile's scores. It leaves of a query only what is not
  // finite (0 x inf is NaN), so the query is what is scaled, and the unit becomes one.
  if (p.flat) {
#pragma unroll
    for (int x = 0; x < QB; x++)
#pragma unroll
      for (int i = 0; i < NK; i++)
#pragma unroll
        for (int n = 0; n < 4; n++) qf[x][i][n] = spread(not_finite<F16>(qf[x][i][n])) & 0x7fff7fffu;
  }
  int buf = 0, free = p.stages - 1;
  for (int step = k0; step < k1; step += STEP) {
    const int key = step + grp * KT;
    const int later = min(p.stages - 2, max(k1 - 1 - key, 0) / STEP);  // tiles behind this one that are on their way
    if (later == 2) vm_wait<4 * PER>();  // this wave's share of this one has landed
    else if (later == 1) vm_wait<2 * PER>();
    else vm_wait<0>();
    __syncthreads();  // everyone's has, and the tile before is no longer read
    if (key + ahead < k1) copy_tile(key + ahead, free);
    const unsigned char* kl = lds + (buf * SP + grp) * 2 * TILE;
    const unsigned char* vl = kl + TILE;
    free = buf;
    buf = buf + 1 == p.stages ? 0 : buf + 1;
    if (key + KT <= lo || key >= hi) continue;  // nothing in it for this wave
    const bool mixed = key < all_lo || key + KT > all_hi;

    // LDS reads are asked for a step ahead of the products that use them, and kept there (sched_barrier): left alone, the
    // compiler saves registers by reading just before each use, and every product waits for the LDS.
    auto key_operand = [&](int t, u32x4(&kf)[NK]) {
#pragma unroll
      for (int i = 0; i < NK; i++)
        kf[i] = *reinterpret_cast<const u32x4*>(kl + ((16 * t + r) * CH + ((4 * i + q) ^ turn<CH>(16 * t + r))) * 16);
    };
    // dims 16 j .. of 32 keys from 32 u: two turned reads of four keys each (lane >> 2 = 4 q + r / 4)
    auto value = [&](int u, int j, int ln) {
      u32x2 w[2];
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int row = 32 * u + 16 * half + (ln >> 2), c = 2 * j + ((ln & 3) >> 1);
        w[half] = read_turned(vl + (row * CH + (c ^ turn<CH>(row))) * 16 + (ln & 1) * 8);
      }
      return u32x4{w[0][0], w[0][1], w[1][0], w[1][1]};
    };
    // One block of queries: two key operands a step, whose products do not wait for one another.
    constexpr int KG = QB == 1 ? 2 : 1;
    f32x4 s[QB][MT];
    u32x4 kf[2 * KG < MT ? 2 * KG : MT][NK];
#pragma unroll
    for (int t = 0; t < KG; t++) key_operand(t, kf[t]);
#pragma unroll
    for (int t = 0; t < MT; t += KG) {
#pragma unroll
      for (int n = 0; n < KG; n++)
        if (t + KG + n < MT) key_operand(t + KG + n, kf[(t + KG + n) % (2 * KG)]);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);  // products first: the other wave's softmax fills what they leave (397 -> 381 us)
#pragma unroll
      for (int n = 0; n < KG * QB; n++) s[n % QB][t + n / QB] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NK; i++)
#pragma unroll
        for (int n = 0; n < KG * QB; n++)
          s[n % QB][t + n / QB] = mma<F16>(kf[(t + n / QB) % (2 * KG)][i], qf[n % QB][i], s[n % QB][t + n / QB]);
    }
    __builtin_amdgcn_s_setprio(0);
    constexpr int NG = HD == 128 && QB == 2 ? 2 : NT % 4 ? 3 : 4, STEPS = KT / 32 * (NT / NG);  // value operands a step
    u32x4 vf[2][NG];
#pragma unroll
    for (int n = 0; n < NG; n++) vf[0][n] = value(0, n, lane);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 P[QB][KT / 32];
#pragma unroll
    for (int x = 0; x < QB; x++) {
      // relative to the lane's first key of the tile
      const int f = first[x] - key - 4 * q, e = last[x] - key - 4 * q;
      const float away = BIAS ? (float)(row0 + 16 * x + r + p.Tk - p.Tq - key - 4 * q) : 0.f;
      // s becomes the score in units of `post`: as it is, capped the tanh, with a bias its base-2 logarithm's worth whole
      const float post = BIAS ? 1.f : CAP ? p.cap : p.scale;
      if constexpr (CAP) {
        float most = 0.f;
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) most = fmaxf(most, fabsf(s[x][t][i]));
        if (__builtin_amdgcn_ballot_w64(most * p.over > kTanhNear) == 0) {
#pragma unroll
          for (int t = 0; t < MT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[x][t][i] = tanh_near(s[x][t][i] * p.over);
        } else {
#pragma unroll
          for (int t = 0; t < MT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[x][t][i] = tanh_own(s[x][t][i] * p.over, s[x][t][i] * p.scale);
        }
      }
      if constexpr (BIAS) {
        const float unit = CAP ? p.cap : p.scale;
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) s[x][t][i] = s[x][t][i] * unit - slope * fabsf(away - (16 * t + i));
      }
      float mx = -INFINITY;
      if (mixed) {
        asm volatile("");  // a branch: as selects the masks cost every tile
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (16 * t + i < f || 16 * t + i >= e) s[x][t][i] = -INFINITY;
      }
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[x][t][i]);
      mx = cols_max(mx) * post;  // post >= 0
      // The reference that weights are taken against follows the maximum only where they would pass 2^PASS: what
      // counts is that no weight overflows, and most tiles leave the sums as they are.
      float ms = m[x] == -INFINITY ? 0.f : m[x];
      if (__builtin_amdgcn_ballot_w64(mx - m[x] > PASS) | far[x]) {
        // each row's by itself: another's keys do not change its roundings
        const float mn = mx - m[x] > PASS ? reference<F16>(mx) : m[x], al = m[x] == mn ? 1.f : exp2_w(m[x] - mn);  // 0 where there was nothing yet
        l[x] *= al;
#pragma unroll
        for (int j = 0; j < NT; j++) O[x][j] *= al;
        m[x] = mn;
        // The reference is a rounded product, and what the rounding took off stands in the fused exponents below: up to 2^6 at 2^30, where
        // the largest weight would vanish or overflow. Of rows past FAR s becomes the difference of rounded products, 0 for the
        // largest, in units of `post`. (The test costs 1 %: 8191 tokens 372.9 and 376.6 us.)
        ms = mn == -INFINITY ? 0.f : mn;
        if constexpr (!BIAS) {
          const bool own = fabsf(ms) >= FAR;
          far[x] = __builtin_amdgcn_ballot_w64(own);
          if (__builtin_expect(far[x] != 0, 0)) {
            const float unit = 1.f / post;
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
              for (int i = 0; i < 4; i++) {
                float product = s[x][t][i] * post;
                asm volatile("" : "+v"(product));  // not to be fused with the difference
                s[x][t][i] = own ? (product - ms) * unit : s[x][t][i];
              }
            ms = own ? 0.f : ms;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < MT; t++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s[x][t][i] = exp2_w(fmaf(s[x][t][i], post, -ms));
          l[x] += s[x][t][i];
        }
        P[x][t >> 1][2 * (t & 1)] = pack2<F16>(s[x][t][0], s[x][t][1]);
        P[x][t >> 1][2 * (t & 1) + 1] = pack2<F16>(s[x][t][2], s[x][t][3]);
      }
    }
    bool apart = false;
    if (mixed) {
      // A value that a query does not see must not reach it, but 0 x NaN is NaN: where a masked tile holds values that are
      // not finite, they are left out of the product, and counted for the queries that see them.
      unsigned bad = 0;
      int ln = lane;
      asm volatile("" : "+v"(ln));
#pragma unroll
      for (int u = 0; u < KT / 32; u++)
#pragma unroll
        for (int j = 0; j < NT; j++) {
          const u32x4 w = value(u, j, ln);
#pragma unroll
          for (int n = 0; n < 4; n++) bad |= not_finite<F16>(w[n]);
          if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
      apart = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
    }
#pragma unroll
    for (int st = 0; st < STEPS; st++) {
      const int u = st / (NT / NG), j0 = st % (NT / NG) * NG;
      if (st + 1 < STEPS) {
#pragma unroll
        for (int n = 0; n < NG; n++) vf[(st + 1) & 1][n] = value((st + 1) / (NT / NG), (st + 1) % (NT / NG) * NG + n, lane);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (apart) {
#pragma unroll
        for (int x = 0; x < QB; x++) {
          int at = 32 * u + 4 * q;
          asm volatile("" : "+v"(at));  // nothing of this rare path is worked out ahead of the loop and kept
          u32x4 seen;                   // one for each key that the lane's query sees
#pragma unroll
          for (int w = 0; w < 4; w++) {
            const int j = key + at + 16 * (w >> 1) + 2 * (w & 1);
            seen[w] = (j >= first[x] && j < last[x] ? ONE : 0u) | (j + 1 >= first[x] && j + 1 < last[x] ? ONE << 16 : 0u);
          }
#pragma unroll
          for (int n = 0; n < NG; n++) {
            u32x4 odd;
#pragma unroll
            for (int w = 0; w < 4; w++) {
              const unsigned v = vf[st & 1][n][w], nan = spread(fraction<F16>(v)), minus = spread(v & 0x80008000u);
              odd[w] = spread(not_finite<F16>(v)) & ((nan & NANS) | (~nan & ((minus & DOWNS) | (~minus & UPS))));
              if (x == QB - 1) vf[st & 1][n][w] = v & ~spread(not_finite<F16>(v));
            }
            const f32x4 c = mma<F16>(odd, seen, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float rest = c[i] - 64.f * floorf(c[i] * (1.f / 64));
              O[x][j0 + n][i] += c[i] >= 4096.f ? NAN : (c[i] >= 64.f ? INFINITY : 0.f) - (rest >= 1.f ? INFINITY : 0.f);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int n = 0; n < NG; n++)
#pragma unroll
        for (int x = 0; x < QB; x++) O[x][j0 + n] = mma<F16>(vf[st & 1][n], P[x][u], O[x][j0 + n]);
    }
    __builtin_amdgcn_s_setprio(0);
  }

  __syncthreads();  // the tiles in LDS are done with
  // Rows leave through LDS, 16 bytes a lane along a row: a lane holds four dims of its row, and stores of 8 bytes to 16 rows
  // took the address unit 3500 cycles with 256 dims.
  constexpr int PITCH = HD * 2 + 16;
  static_assert(NW * SP * 16 * PITCH <= 2 * SP * 2 * TILE, "LDS");
  unsigned char* turn_rows = lds + all_waves * (16 * PITCH);
  auto put = [&](int j, f32x4 o) {
    *reinterpret_cast<u32x2*>(turn_rows + r * PITCH + (16 * j + 4 * q) * 2) = u32x2{pack2<F16>(o[0], o[1]), pack2<F16>(o[2], o[3])};
  };
  auto leave = [&](int x, int j0, auto tiles) {  // dims of tiles j0 .. j0 + tiles - 1
    constexpr int C = 2 * decltype(tiles)::value;
    wave_fence();
#pragma unroll
    for (int i = 0; i < (16 * C + 63) / 64; i++) {
      const int at = i * 64 + lane, rr = at / C, d = 16 * j0 + at % C * 8, row = row0 + 16 * x + rr;
      if ((16 * C % 64 == 0 || rr < 16) && row < p.Tq && d < p.hd)
        *reinterpret_cast<u32x4*>(p.out + ((((size_t)b * p.Tq + row) * p.H + h) * p.hd + d) * 2) =
            *reinterpret_cast<const u32x4*>(turn_rows + rr * PITCH + d * 2);
    }
    wave_fence();
  };
  if constexpr (SP > 1) {  // each of the two groups finishes half of the dims: it hands the sums of the others over, lane by lane
    static_assert(QB == 1 && SP == 2 && NT % 2 == 0, "one block of queries, two groups");
    constexpr int HALF = NT / 2, MINE = HALF * 256 + 128;
    static_assert(NW * 2 * MINE * 4 <= 2 * SP * 2 * TILE, "LDS");
    float* give = reinterpret_cast<float*>(lds) + (wave * 2 + grp) * MINE;
    const float* take = reinterpret_cast<const float*>(lds) + (wave * 2 + 1 - grp) * MINE;
    auto finish = [&](auto low) {  // low: this group's tiles start at 0
      constexpr int J0 = decltype(low)::value ? 0 : HALF, J1 = HALF - J0;
#pragma unroll
      for (int j = 0; j < HALF; j++) *reinterpret_cast<f32x4*>(give + (j * 64 + lane) * 4) = O[0][J1 + j];
      give[HALF * 256 + lane] = m[0];
      give[HALF * 256 + 64 + lane] = l[0];
      __syncthreads();
      const float m1 = take[HALF * 256 + lane], l1 = take[HALF * 256 + 64 + lane], mm = fmaxf(m[0], m1);
      const float f0 = m[0] == -INFINITY ? 0.f : exp2_w(m[0] - mm), f1 = m1 == -INFINITY ? 0.f : exp2_w(m1 - mm);
      float sum = cols_sum(l[0] * f0 + l1 * f1);
#pragma unroll
      for (int j = 0; j < HALF; j++)
        O[0][J0 + j] = O[0][J0 + j] * f0 + f1 * *reinterpret_cast<const f32x4*>(take + (j * 64 + lane) * 4);
      if (used > 1) {
        constexpr unsigned PART = NW * part_floats(NT) * 4;  // bytes
        const size_t unit = (size_t)bh * p.ntile + tile;
        const rsrc_t parts = make_rsrc(reinterpret_cast<unsigned char*>(p.part) + unit * p.S * PART, 0xffffffffu);
        const unsigned mine = wave * (part_floats(NT) * 4);
#pragma unroll
        for (int j = J0; j < J0 + HALF; j++) {
          const f32x4 o = O[0][j];
          stb128<kCpSc1>(parts, split * PART + mine + (j * 64 + lane) * 16, __builtin_bit_cast(u32x4, o));
        }
        if (J0 == 0 && lane < 16)
          stb64<kCpSc1>(parts, split * PART + mine + NT * 1024 + lane * 8, __builtin_bit_cast(u32x2, f32x2{mm, sum}));
        if (p.S > FUSED || !arrived_last(p.arrived + unit * FUSED, p.nonce, split, used, ext)) return;
        f32x2 ml[FUSED];
        float top = -INFINITY;
#pragma unroll
        for (int s = 0; s < FUSED; s++) {
          ml[s] = f32x2{-INFINITY, 0.f};
          if (s < used) ml[s] = __builtin_bit_cast(f32x2, ldb64<kCpSc1>(parts, s * PART + mine + NT * 1024 + r * 8));
          top = fmaxf(top, ml[s][0]);
        }
        sum = 0.f;
#pragma unroll
        for (int j = J0; j < J0 + HALF; j++) O[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < FUSED; s++)
          if (s < used) {
            const float w = ml[s][0] == -INFINITY ? 0.f : exp2_w(ml[s][0] - top);
            sum += w * ml[s][1];
#pragma unroll
            for (int j = J0; j < J0 + HALF; j++)
              O[0][j] += w * __builtin_bit_cast(f32x4, ldb128<kCpSc1>(parts, s * PART + mine + (j * 64 + lane) * 16));
          }
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      __syncthreads();
#pragma unroll
      for (int j = J0; j < J0 + HALF; j++) put(j, O[0][j] * inv);
      leave(0, J0, std::integral_constant<int, HALF>{});
    };
    if (grp == 0) finish(std::true_type{});
    else finish(std::false_type{});
  } else {
#pragma unroll
    for (int x = 0; x < QB; x++) {
      const float sum = cols_sum(l[x]), inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int j = 0; j < NT; j++) put(j, O[x][j] * inv);
      leave(x, 0, std::integral_constant<int, NT>{});
    }
  }
}

// Joins the parts of 16 rows; a wave takes every fourth tile of 16 dims.
template <bool F16, int HD>
__global__ void __launch_bounds__(256) join_kernel(Params p) {
  constexpr int NT = HD / 16, NJ = (NT + 3) / 4;
  __shared__ float wt[MAX_SPLITS][16];
  const unsigned unit = blockIdx.x >> 2, rows = blockIdx.x & 3, bh = unit / p.ntile, tile = unit - bh * p.ntile;
  const int used = p.used[unit];
  if (used == 1) return;
  const float* from = p.part + (size_t)unit * p.S * (4 * part_floats(NT)) + rows * part_floats(NT);
  const int stride = 4 * part_floats(NT), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, q = lane >> 4;
  float mm = -INFINITY;
  for (int s = 0; s < used; s++) mm = fmaxf(mm, from[(size_t)s * stride + NT * 256 + 2 * r]);
  float sum = 0.f;
  for (int s = 0; s < used; s++) {
    const float m = from[(size_t)s * stride + NT * 256 + 2 * r], l = from[(size_t)s * stride + NT * 256 + 2 * r + 1];
    const float w = m == -INFINITY ? 0.f : exp2_w(m - mm);
    sum += w * l;
    if (tid < 16) wt[s][r] = w;
  }
  __syncthreads();
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  f32x4 O[NJ];
#pragma unroll
  for (int i = 0; i < NJ; i++) O[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < used; s++) {
    const float w = wt[s][r];
#pragma unroll
    for (int i = 0; i < NJ; i++)
      if (NT % 4 == 0 || 4 * i + wave < NT)
        O[i] += w * *reinterpret_cast<const f32x4*>(from + (size_t)s * stride + ((4 * i + wave) * 64 + lane) * 4);
  }
  const int row = (p.ntile - 1 - (int)tile) * 64 + rows * 16 + r, b = bh / (unsigned)p.H, h = bh - b * p.H;
  if (row >= p.Tq) return;
  unsigned char* o = p.out + (((size_t)b * p.Tq + row) * p.H + h) * p.hd * 2;
#pragma unroll
  for (int i = 0; i < NJ; i++) {
    const int d = 16 * (4 * i + wave) + 4 * q;
    if (d < p.hd)
      *reinterpret_cast<u32x2*>(o + d * 2) =
          u32x2{pack2<F16>(O[i][0] * inv, O[i][1] * inv), pack2<F16>(O[i][2] * inv, O[i][3] * inv)};
  }
}

// Parts that keys are split into, for workgroups of 64 queries with two groups of waves: the least of (rounds of
// workgroups) x (steps of each, and two for its beginning and end), joining taken as three. A workgroup whose queries see
// fewer keys makes fewer parts, of LEAST steps or more (packed prompts of 2364 tokens: 60.5 us with 8, 62.6 with 4, 60.7 with 16).
// 64 queries over 65536 keys of 256 dims 1517 -> 109 us, one over 131072 of 128 dims 1424 -> 103, 1024 over 4096 59 -> 39;
// of the counts 1 .. 16 the rule's was within 3 % of the best in all of 14 shapes between.
inline int splits_for(int64_t units, int keys, int hd) {
  const int step = hd > 128 ? 64 : 128;
  const int64_t n = (keys + (int64_t)step - 1) / step, most = std::min<int64_t>({n / LEAST, MAX_SPLITS, 1024 / units});
  int best = 1;
  int64_t cost = (units + 255) / 256 * (n + 2);
  for (int64_t S = 2; S <= most; S++) {
    const int64_t t = (units * S + 255) / 256 * ((n + S - 1) / S + 2) + 3;
    if (t < cost) best = (int)S, cost = t;
  }
  return best;
}
inline int64_t units_of(int batch, int queries, int heads) { return ((int64_t)queries + 63) / 64 * batch * heads; }
// Few queries: see launch_dims.
inline bool few(int64_t units, int hd) { return units <= (hd > 128 ? 384 : 256); }
inline size_t used_bytes(int64_t units) { return ((size_t)units * 4 + 255) / 256 * 256; }
inline size_t arrived_bytes(int64_t units) { return ((size_t)units * FUSED * 8 + 255) / 256 * 256; }
inline size_t workspace(int batch, int queries, int keys, int heads, int hd) {
  const int64_t units = units_of(batch, queries, heads);
  const int S = few(units, hd) ? splits_for(units, keys, hd) : 1, nt = (hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : 256) / 16;
  return S == 1 ? 0 : used_bytes(units) + arrived_bytes(units) + (size_t)units * S * 4 * part_floats(nt) * 4;
}

template <bool F16, int HD, int QB, int NW, int SP>
int launch(Params p, hipStream_t s) {
  constexpr int KT = HD == 256 ? 32 : 64, STAGE = SP * 2 * KT * HD * 2, EXTRA = 2 * NW * 4;
  p.ntile = (p.Tq + 16 * QB * NW - 1) / (16 * QB * NW);
  const int64_t units = (int64_t)p.ntile * p.B * p.H, grid = units * (SP > 1 ? p.S : 1);
  if (grid > 0x7fffffff) return host::fail(FA_ERR_INVALID_ARG, "fa_span_attention: too many rows for one call");
  const bool cap = p.cap > 0.f, bias = p.slopes != nullptr;
  void (*k)(Params) =
      cap ? (bias ? span_kernel<F16, HD, QB, NW, SP, true, true> : span_kernel<F16, HD, QB, NW, SP, true, false>)
          : (bias ? span_kernel<F16, HD, QB, NW, SP, false, true> : span_kernel<F16, HD, QB, NW, SP, false, false>);
  // Up to four tiles in LDS: a workgroup of eight waves has a CU to itself, two of four waves share one.
  constexpr int STAGES = std::min(4, (NW * SP == 8 ? 160 : 80) * 1024 / (STAGE + EXTRA));
  static_assert(STAGES >= 2, "LDS");
  p.stages = STAGES;
  const unsigned lds = STAGES * STAGE + EXTRA;
  const int rc = host::allow_lds(reinterpret_cast<const void*>(k), lds, "fa_span_attention");
  if (rc != FA_OK) return rc;
  hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(64 * NW * SP), lds, s, p);
  if (SP > 1 && p.S > FUSED) hipLaunchKernelGGL((join_kernel<F16, HD>), dim3((unsigned)(4 * units)), dim3(256), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return host::fail(FA_ERR_LAUNCH, "fa_span_attention: %s", hipGetErrorString(e));
  return FA_OK;
}

template <bool F16, int HD>
int launch_dims(const Params& p, hipStream_t s) {
  // Few queries: workgroups of 64 in which two groups of waves share the keys, as a lone wave a SIMD waits for itself most of
  // the time (2048 tokens of 8 heads of 128 dims 46 -> 35 us; 304 workgroups, though, 66 -> 69, 384 of 96 dims 41 -> 48; with 256 dims up
  // to 384, where packed prompts of 2364 tokens gain, 83 -> 60 us, more than whole ones of 3000 lose, 140 -> 148). Many, past 512:
  // workgroups of 128 with two blocks a wave, which halve the LDS reads for each product (8192 tokens of 16 heads of 128
  // dims: 605 us instead of 765; 768 workgroups of 64: 72 instead of 90; 512: 57 instead of 53). 256 dims leave registers for one (two, at one wave a SIMD: 2374 instead of 1467), and two
  // workgroups of 64 on a CU go better than one of 128 (1467 instead of 1511).
  const int64_t small = units_of(p.B, p.Tq, p.H);
  if (few(small, HD)) return launch<F16, HD, 1, 4, 2>(p, s);
  if constexpr (HD == 256) return launch<F16, HD, 1, 4, 1>(p, s);
  else return small <= 512 ? launch<F16, HD, 1, 4, 1>(p, s) : launch<F16, HD, 2, 4, 1>(p, s);
}

template <bool F16>
int launch_type(const Params& p, hipStream_t s) {
  if (p.hd <= 64) return launch_dims<F16, 64>(p, s);
  if (p.hd <= 96) return launch_dims<F16, 96>(p, s);
  if (p.hd <= 128) return launch_dims<F16, 128>(p, s);
  return launch_dims<F16, 256>(p, s);
}

int run_bf16(const Params& p, hipStream_t s);
int run_f16(const Params& p, hipStream_t s);

}  // namespace attn
}  // namespace fa
