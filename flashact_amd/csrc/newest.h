// What the attentions of each sample's newest tokens over a cache share (kv8_attn.hip, paged_attn.hip): who sees what, and how the
// sums of waves and of workgroups meet.
//
// A workgroup of W waves takes one tile of 16 rows (t, h) of a sample and K/V head; its keys, in blocks of 32, are dealt to the
// waves of up to S workgroups. Each wave ends with O^T of its blocks (f32x4 O[j]: dims 16 j + 4 q .. of row r, lane r + 16 q), the
// reference m of its weights (base 2) and their sum l. All of it is summed in a fixed order: results do not depend on timing.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"

namespace fa {
namespace newest {

constexpr int BT = 32;  // keys of a block
constexpr int W = 4;    // waves of a workgroup
constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_SPLITS = 256;
// Up to so many are joined by the last workgroup (32 requests of 50 to 16384 keys on 16 splits: 20.6 us, 22.6 with a kernel), more
// by a kernel with workgroups enough to read them.
constexpr int FUSED = 16;

struct Args {
  const unsigned char* q;
  int64_t qb, qt, qh;  // strides in elements
  const int *lens, *count;
  const float* slopes;
  unsigned char* out;
  float* part;               // [sample][head][row tile][split] {O[16][hd], {m, l}[16]}
  uint64_t *arrived, nonce;  // [sample][head][row tile][FUSED], where the last workgroup joins the splits
  int B, T, H, G, nblk, RT, RU, RC, S, least, causal;  // RT row tiles of a head in RU workgroups, RC of these side by side on an XCD
  float scale, over, cap;  // base 2: scale log2(e); capped, scale / cap and cap log2(e)
};

// The row tile's share of what its sample has cached.
struct Span {
  int len, n;
};
__device__ __forceinline__ Span span_of(const Args& a, int b) {
  const int cap = (int)min((int64_t)a.nblk * BT, (int64_t)0x7fffffff - 31);
  Span s;
  s.len = max(0, min(a.lens[b], cap));
  s.n = a.count ? max(0, min(a.count[b], a.T)) : a.T;
  return s;
}
// Splits that a row tile of nb blocks uses: each wave of each has a.least blocks or more.
__device__ __forceinline__ int splits_used(const Args& a, int nb) {
  const unsigned per = W * a.least;
  return max(1, min(a.S, (int)((nb + per - 1) / per)));
}

// Which row tile of which sample and head, and which split of its keys, a workgroup takes.
struct Place {
  int split, bh, b, h, rt;  // rt: the workgroup's place along the rows, its row tile where it has one
  bool there;
};
__device__ __forceinline__ Place place_of(const Args& a) {
  // Row tiles of one (split, sample, head) share their keys: RC neighbours on one XCD. Splits are the slowest index: samples
  // that leave the later ones unused would else leave XCDs unused (64 samples of 1050 keys on 16 splits: 72 us instead
  // of 21); within a split the runs of row tiles are turned, so that the splits of one meet on different XCDs.
  const unsigned xcd = blockIdx.x & 7, y = blockIdx.x >> 3, yr = y / (unsigned)a.RC, u = yr * 8 + xcd;
  const unsigned runs = (a.RU + a.RC - 1) / a.RC, all_runs = a.B * a.H * runs;
  Place p;
  p.split = u / all_runs;
  unsigned turned = u - p.split * all_runs + (all_runs >= 8 ? (p.split * (all_runs - 1)) & 7 : 0);
  if (turned >= all_runs) turned -= all_runs;
  p.bh = turned / runs, p.b = p.bh / (unsigned)a.H, p.h = p.bh - p.b * a.H;
  p.rt = (turned - p.bh * runs) * a.RC + y - yr * a.RC;
  p.there = p.split < a.S && p.rt < a.RU;
  return p;
}

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

// Raw products of a lane's eight keys key0 .. key0 + 7 -> scores in base 2, -inf at `limit` and behind where the block is `mixed`; the
// largest of them. factor: the keys' scale.
template <bool CAP, bool BIAS>
__device__ __forceinline__ float scores(const Args& a, f32x4* s, float factor, int key0, bool mixed, int limit, float slope, int pos) {
  if constexpr (CAP) {
    float most = 0.f;
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[x][i] *= factor * a.over;
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
    const float f = factor * a.scale;
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
  return mx;
}

// LDS of a workgroup whose waves stage WAVE bytes each, and whose sums lie over the stages afterwards.
template <int HD, int STAGE>
struct Lds {
  static constexpr int PITCH = HD + 4;  // of the waves' sums
  static constexpr int WAVE = STAGE;
  static constexpr int SUM = W * 16 * PITCH * 4 > W * WAVE ? W * 16 * PITCH * 4 : W * WAVE;
  static constexpr int BYTES = SUM + 2 * W * 16 * 4;
};

// The waves' sums meet, and the splits' (`used` of them) where these are joined by the last workgroup. l: all lanes of a row hold
// the sum of the row's weights of this wave.
template <bool F16, int HD, class L>
__device__ __forceinline__ void meet(const Args& a, const Place& at, const Span& sp, int used, unsigned char* lds, const f32x4* O,
                                     float m, float l) {
  constexpr int NT = HD / 16, PITCH = L::PITCH;
  float* osum = reinterpret_cast<float*>(lds);
  float* wm = reinterpret_cast<float*>(lds + L::SUM);
  float* wl = wm + W * 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4, b = at.b, h = at.h, rt = at.rt, split = at.split;
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
  const rsrc_t part = make_rsrc(a.part + ((size_t)at.bh * a.RT + rt) * a.S * ONE, 0xffffffffu);  // the tile's splits
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
  if (!arrived_last(a.arrived + ((size_t)at.bh * a.RT + rt) * FUSED, a.nonce, split, used, reinterpret_cast<int*>(wm))) return;
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
__device__ __forceinline__ void join(const Args& a) {
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
inline unsigned join_grid(const Args& a, int hd) { return (unsigned)(a.B * a.H * a.T * a.G * (hd % 64 == 0 ? hd / 64 : 1)); }

// Splits of all row tiles together: they bound the workspace (68 MB with 256 dims), where whole rounds of workgroups alone would ask
// for gigabytes beside a small cache. 2049 tokens of 8 heads of 256 dims over 8192 keys 354 us, unbounded (135 MB) 440, over 32768 keys
// 1360 and 1275; 4152 of 128 dims 244 and 276, 1143 and 1085; 4 x 2080 of 64 dims over 16384 keys 643 and 603.
constexpr int MAX_PARTS = 4096;

// Splits of the keys across workgroups. A wave takes `block` us for a block that comes from memory and one to begin and end, more
// than `resident` workgroups a CU share its bandwidth, and joining the splits costs 3 us: the number with the least estimate, for
// samples that fill the cache (their lengths are on the GPU), is taken. Shorter ones use fewer.
inline int splits_for(int batch, int tokens, int heads, int kv_heads, int blocks, double block, double resident,
                      int tiles = 1) {
  const int64_t rt = ((int64_t)tokens * (heads / kv_heads) + 16 * tiles - 1) / (16 * tiles), units = rt * batch * kv_heads;
  const int64_t most = std::min<int64_t>({(blocks + W - 1) / W, MAX_SPLITS, std::max<int64_t>(1, MAX_PARTS / (units * tiles))});
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

inline size_t arrived_bytes(size_t tiles) { return (tiles * FUSED * sizeof(uint64_t) + 255) / 256 * 256; }

inline size_t workspace(int S, int batch, int tokens, int heads, int kv_heads, int hd) {
  if (S == 1) return 0;
  const size_t rt = ((size_t)tokens * (heads / kv_heads) + 15) / 16;
  return (S <= FUSED ? arrived_bytes(rt * batch * kv_heads) : 0) + rt * batch * kv_heads * S * (16 * hd + 32) * sizeof(float);
}

// What both entries check and set up; p.S is set and `need` is the workspace of that many splits. fa_kv8_attn_args and
// fa_paged_attn_args name the fields used here alike.
template <class A>
int check_call(const A* a, const char* who) {
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
  return FA_OK;
}

template <class A>
int set_up(Args& p, const A* a, int blocks, int splits, int tiles, const char* who) {
  const size_t need = workspace(splits, a->batch, a->tokens, a->heads, a->kv_heads, a->head_dim);
  if (need && (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return host::fail(FA_ERR_INVALID_ARG, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, need,
                      a->workspace ? a->workspace_bytes : (size_t)0);
  p.q = static_cast<const unsigned char*>(a->q);
  p.qb = a->q_stride[0], p.qt = a->q_stride[1], p.qh = a->q_stride[2];
  p.lens = a->lens, p.count = a->count, p.slopes = a->slopes;
  p.out = static_cast<unsigned char*>(a->out), p.part = static_cast<float*>(a->workspace);
  p.B = a->batch, p.T = a->tokens, p.H = a->kv_heads, p.G = a->heads / a->kv_heads, p.nblk = blocks;
  p.RT = (p.T * p.G + 15) / 16;
  p.RU = (p.RT + tiles - 1) / tiles;
  p.S = splits;
  if (p.S > 1 && p.S <= FUSED) {
    p.nonce = host::launch_nonce();
    p.arrived = static_cast<uint64_t*>(a->workspace);
    p.part = reinterpret_cast<float*>(static_cast<unsigned char*>(a->workspace) + arrived_bytes((size_t)p.RT * p.B * p.H));
  }
  // All row tiles of a (split, sample, head) run on one XCD where these divide evenly over the 8, else in runs short enough
  // that there are 32 or more (200 tokens of 8 heads over 1100 keys of one sample 38 -> 21 us; 17.3 -> 17.5 for 4 samples of 50).
  const int64_t groups = (int64_t)p.B * p.H * p.S, runs = groups % 8 ? std::min<int64_t>((31 + groups) / groups, p.RU) : 1;
  p.RC = (int)((p.RU + runs - 1) / runs);
  p.least = (int64_t)p.RU * p.B * p.H >= 64 ? 4 : 1;
  p.causal = a->causal;
  p.scale = a->scale * LOG2E;
  p.over = a->softcap > 0.f ? a->scale / a->softcap : 0.f;
  p.cap = a->softcap * LOG2E;
  if (!(fabsf(p.scale) < INFINITY) || !(fabsf(p.over) < INFINITY) || !(p.cap < INFINITY))
    return host::fail(FA_ERR_INVALID_ARG, "%s: scale=%g over softcap=%g leaves the fp32 range", who, a->scale, a->softcap);
  return FA_OK;
}

// Workgroups of a launch, or 0 where there are too many.
inline unsigned grid_of(const Args& a) {
  const int runs = (a.RU + a.RC - 1) / a.RC;
  const int64_t grid = ((int64_t)a.B * a.H * a.S * runs + 7) / 8 * 8 * a.RC;
  return grid > host::MAX_GRID ? 0 : (unsigned)grid;
}

}  // namespace newest
}  // namespace fa
