// Log probabilities of given tokens, with entropy and the best alternatives (fa_token_logprobs), out of logits read once.
//
//   z = scale x;  m = max z, s = sum e^(z - m), t = sum (z - m) e^(z - m):
//   log p_i = z_i - m - log s,  entropy = log s - t / s,  alternatives by (x descending, index ascending).
//
// Bound by reading the logits, once. A workgroup takes a part of a row, 16 values a thread at a time; every thread keeps its own
// running maximum (of x, exact) and sums. Few rows are split over up to 32 workgroups, whose sums the last one to arrive joins.
//
// The alternatives cost the pass over the row nothing: they are found behind it, from the threads' maxima. The k-th largest maximum of 64
// groups of threads is a bound that at least k values reach, and few more (24 for k = 20, whatever the row's length). The
// threads whose maximum reaches it read their values again, those that do are put side by side, and each counts how many are before it.
// Where ties leave too many (a row of equal values), the k-th largest value is found exactly by four counts of eight bits
// over the whole row, and equal ones are taken in the row's order.
// (Sorted lists kept by each wave during the pass, with insertions one by one, took 16 us instead of 9.5 for 8 of 262144 bf16 logits, and
// 35 instead of 17.6 for 20 of 48 rows of 99991: every step from a comparison to a scalar and back costs some 50 cycles.)
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"

namespace fa {
namespace tokens {

constexpr int W = 4;  // waves of a workgroup
constexpr int MAX_SPLITS = 32;
constexpr int MOST = 512;  // threads that look again, and values that they may find, for the short way
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LEAST = -1e30f;  // for -inf where it is multiplied by a weight of 0

struct Params {
  const unsigned char* x;
  int64_t xs;  // row stride, elements
  const void* tokens;
  int wide;  // tokens are 64-bit
  float scale, c;  // c: scale log2(e)
  int rows, V, top, S, per;  // per: vectors of a split
  float *logprob, *entropy;
  int* top_tokens;
  float* top_logprobs;
  float* part;  // [row][split] {m, s, t, 0, maximum[threads]}; without alternatives the first four
  uint64_t *arrived, nonce;  // [row][split]
};
__host__ __device__ constexpr int part_floats(bool top) { return top ? 4 + 64 * W : 4; }

template <int DT>
struct Vec {
  static constexpr int E = DT == FA_DTYPE_F32 ? 4 : 8, BYTES = DT == FA_DTYPE_F32 ? 4 : 2;
  static constexpr int U = 16 / E;  // vectors of a lane's batch
};
// Value i of a vector.
template <int DT>
__device__ __forceinline__ float value(u32x4 v, int i) {
  if constexpr (DT == FA_DTYPE_F32) return as_f32(v[i]);
  else if constexpr (DT == FA_DTYPE_F16) return i & 1 ? h_hi(v[i >> 1]) : h_lo(v[i >> 1]);
  else return i & 1 ? bf_hi(v[i >> 1]) : bf_lo(v[i >> 1]);
}
template <int DT>
__device__ __forceinline__ float value_at(const unsigned char* row, int i) {
  if constexpr (DT == FA_DTYPE_F32) return reinterpret_cast<const float*>(row)[i];
  else if constexpr (DT == FA_DTYPE_F16) return (float)reinterpret_cast<const _Float16*>(row)[i];
  else return as_f32((unsigned)reinterpret_cast<const unsigned short*>(row)[i] << 16);
}

// Unsigned numbers in the values' order (-0 as 0), and back. NaN is above all: it is sorted out by itself.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = as_u32(x + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned u) { return as_f32(u >> 31 ? u & 0x7fffffffu : ~u); }
constexpr unsigned NOTHING = 0x007fffffu;  // ordered(-inf)

struct Sums {
  float m, s, t;
};
// The lanes' sums as one, in every lane.
__device__ __forceinline__ Sums sum_lanes(Sums x, float c) {
  Sums y;
  y.m = wave_max(x.m);
  const float d = fmaxf((x.m - (y.m == -INFINITY ? 0.f : y.m)) * c, LEAST), a = exp2_w(d);
  // lane 0's: a fused product and sum in the first step may leave the lanes a last bit apart
  y.s = as_f32(__builtin_amdgcn_readfirstlane(as_u32(wave_sum(a * x.s))));
  y.t = as_f32(__builtin_amdgcn_readfirstlane(as_u32(wave_sum(a * (x.t + d * x.s)))));
  return y;
}

// Where a row lies: vectors of 16 aligned bytes, of which [whole_b, whole_e) lie in it whole. Up to 2 (E - 1) values at its ends do not
// belong to one of these.
template <int DT>
struct Row {
  static constexpr int E = Vec<DT>::E;
  const unsigned char* x;
  const u32x4* base;
  int off, V, whole_b, whole_e;

  __device__ __forceinline__ Row(const Params& p, int row) {
    x = p.x + (int64_t)row * p.xs * Vec<DT>::BYTES;
    off = (int)(reinterpret_cast<uintptr_t>(x) & 15) / Vec<DT>::BYTES;
    V = p.V;
    base = reinterpret_cast<const u32x4*>(x - off * Vec<DT>::BYTES);
    whole_b = off ? 1 : 0, whole_e = (off + V) / E;
  }
  __device__ __forceinline__ int index(int v, int i) const { return v * E - off + i; }  // of value i of vector v
  // Index of the i-th value at the ends, or -1: i < E those before the whole vectors, i < 2 E those behind them.
  __device__ __forceinline__ int end(int i) const {
    const int before = off ? min(E - off, V) : 0, at = i < E ? i : max(whole_e * E - off, before) + i - E;
    return i < E ? (i < before ? i : -1) : i < 2 * E && at < V ? at : -1;
  }
  // Vector v of all that hold one of the row's values; what is not in the row reads as -inf.
  __device__ __forceinline__ int vectors() const { return (off + V + E - 1) / E; }
  __device__ __forceinline__ u32x4 any(int v) const {
    u32x4 y = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < E; i++) {
      const int at = index(v, i);
      const unsigned low = DT == FA_DTYPE_F32 ? 0xff800000u : DT == FA_DTYPE_F16 ? 0xfc00u : 0xff80u;
      unsigned u = low;
      if (at >= 0 && at < V) u = DT == FA_DTYPE_F32 ? reinterpret_cast<const unsigned*>(x)[at] : reinterpret_cast<const unsigned short*>(x)[at];
      if constexpr (DT == FA_DTYPE_F32) y[i] = u;
      else y[i >> 1] |= u << (16 * (i & 1));
    }
    return y;
  }
};

struct Shared {
  Sums sums[W];
  float maxima[W][64];
  unsigned items, found, digit, above;
  unsigned item[MOST];
  uint64_t key[MOST];
  unsigned count[256];
  int flag;
};

// The workgroup's threads count their values' next eight bits, of those whose upper bits are `prefix`'s; four times, and the k-th
// largest value is known. Returns it (ordered) and how many are above it.
template <int DT>
__device__ __forceinline__ unsigned kth_of_row(const Row<DT>& r, int k, Shared& sh, int& above) {
  static_assert(64 * W == 256, "a thread a count");
  unsigned prefix = 0;
  above = 0;
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    sh.count[threadIdx.x] = 0;
    __syncthreads();
    for (int v = threadIdx.x; v < r.vectors(); v += 64 * W) {
      const u32x4 y = r.any(v);
#pragma unroll
      for (int i = 0; i < Vec<DT>::E; i++) {
        const float x = value<DT>(y, i);
        const unsigned u = ordered(x);
        if (x > -INFINITY && (shift == 24 || u >> (shift + 8) == prefix >> (shift + 8))) atomicAdd(&sh.count[u >> shift & 255], 1u);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int d = 255;
      for (; d > 0 && above + (int)sh.count[d] < k; d--) above += sh.count[d];
      sh.digit = d, sh.above = above;
    }
    __syncthreads();
    prefix |= sh.digit << shift;
    above = sh.above;
  }
  return prefix;
}

// The best `top` of a row, by the workgroup's threads. Maxima of the row's threads (thread t of split s has taken the whole vectors t + 256 i
// of the split's): this one's `own`, or, where there are splits, a share of all of them. m, logs: as the log probabilities need them.
// Loops stay loops: code that runs once costs its fetch.
template <int DT>
__device__ __forceinline__ void alternatives(const Params& p, const Row<DT>& r, int row, Shared& sh, float m, float logs, float own_max,
                                             const f32x4* maxima) {
  constexpr int E = Vec<DT>::E, T = 64 * W, QUADS = MAX_SPLITS / 4;
  const int t = threadIdx.x, lane = t & 63, k = p.top, edge = r.end(t);
  float high[QUADS], most = own_max;
  if (p.S > 1) {
    most = -INFINITY;
#pragma unroll
    for (int i = 0; i < QUADS; i++) {
      high[i] = fmaxf(fmaxf(maxima[i][0], maxima[i][1]), fmaxf(maxima[i][2], maxima[i][3]));
      most = fmaxf(most, high[i]);
    }
  }
  sh.maxima[t >> 6][lane] = most;
  if (t == 0) sh.items = sh.found = 0;
  __syncthreads();
  float g = sh.maxima[0][lane];
#pragma unroll
  for (int w = 1; w < W; w++) g = fmaxf(g, sh.maxima[w][lane]);
  // the largest group's maximum that k of them reach
  int reach = 0;
#pragma unroll 4
  for (int j = 0; j < 64; j++) reach += as_f32(__builtin_amdgcn_readlane(as_u32(g), j)) >= g;
  const float bound = wave_max(reach >= k ? g : -INFINITY);
  auto reaches = [&](float x) { return x >= bound && x > -INFINITY; };
  // who has to look again: threads, or four neighbours of a split
  auto look = [&](float x, int who) {
    if (reaches(x)) {
      const unsigned at = atomicAdd(&sh.items, 1u);
      if (at < MOST) sh.item[at] = who;
    }
  };
  const int side = p.S > 1 ? 4 : 1;
  if (p.S == 1) {
    look(own_max, t);
  } else {
#pragma unroll
    for (int i = 0; i < QUADS; i++) look(high[i], (4 * i + (t >> 6)) * 64 + lane);
  }
  auto found = [&](float x, int index) {
    if (reaches(x)) {
      const unsigned at = atomicAdd(&sh.found, 1u);
      if (at < MOST) sh.key[at] = (uint64_t)ordered(x) << 32 | ~(unsigned)index;
    }
  };
  if (edge >= 0) found(value_at<DT>(r.x, edge), edge);
  __syncthreads();
  const int items = sh.items, nv = r.vectors(), each = side * ((p.per + T - 1) / T);  // vectors of an item, at most
  unsigned floor = ordered(bound);
  int n = MOST + 1, fill = 0;  // values found, and further ones that equal `floor`
  if (items <= MOST) {
#pragma unroll 1
    for (unsigned e = t; e < (unsigned)(items * each); e += T) {
      const unsigned i = e / (unsigned)each, rest = e - i * each, who = sh.item[i] * side, s = who / T;
      const int v = max(s * p.per, (unsigned)r.whole_b) + who % T + rest % side + T * (rest / side);
      if (v >= min((int)(s + 1) * p.per, r.whole_e)) continue;
      const u32x4 y = r.base[v];
#pragma unroll
      for (int j = 0; j < E; j++) found(value<DT>(y, j), r.index(v, j));
    }
    __syncthreads();
    n = sh.found;
    if (n < k) floor = NOTHING, fill = k - n;  // all others are ruled out
  }
  if (n > MOST) {
    int above;
    floor = kth_of_row(r, k, sh, above);
    fill = k - above, n = above;
    if (t == 0) sh.found = 0;
    __syncthreads();
    for (int v = t; v < nv; v += T) {
      const u32x4 y = r.any(v);
#pragma unroll
      for (int j = 0; j < E; j++) {
        const float x = value<DT>(y, j);
        if (x > -INFINITY && ordered(x) > floor) sh.key[atomicAdd(&sh.found, 1u)] = (uint64_t)ordered(x) << 32 | ~(unsigned)r.index(v, j);
      }
    }
    __syncthreads();
  }
  int* const tokens = p.top_tokens + (size_t)row * k;
  float* const logprobs = p.top_logprobs + (size_t)row * k;
  for (int c = t; c < n; c += T) {
    const uint64_t own = sh.key[c];
    int before = 0;
#pragma unroll 4
    for (int j = 0; j < n; j++) before += sh.key[j] > own;
    if (before < k) {
      tokens[before] = (int)~(unsigned)own;
      logprobs[before] = (unordered((unsigned)(own >> 32)) - m) * p.scale - logs;
    }
  }
  // those that equal `floor`, in the row's order; where there are not enough (NaN), token -1
  if (fill == 0) return;
  int have = 0;
#pragma unroll 1
  for (int v0 = 0; v0 < nv && have < fill; v0 += T) {
    const int v = v0 + t;
    unsigned hits = 0;
    if (v < nv) {
      const u32x4 y = r.any(v);
#pragma unroll
      for (int i = 0; i < E; i++) {
        const float x = value<DT>(y, i);
        const int at = r.index(v, i);
        if (x == x && ordered(x) == floor && at >= 0 && at < p.V) hits |= 1u << i;
      }
    }
    int before = have, all = 0;  // of lower lanes, of the wave
#pragma unroll
    for (int i = 0; i < E; i++) {
      const uint64_t b = __builtin_amdgcn_ballot_w64(hits >> i & 1);
      before += __builtin_amdgcn_mbcnt_hi((unsigned)(b >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)b, 0));
      all += __builtin_popcountll(b);
    }
    if (lane == 0) sh.count[t >> 6] = all;
    __syncthreads();
    for (int w = 0; w < W; w++) {
      if (w < t >> 6) before += sh.count[w];
      have += sh.count[w];
    }
    for (; hits; hits &= hits - 1, before++)
      if (before < fill) {
        tokens[n + before] = r.index(v, __builtin_ctz(hits));
        logprobs[n + before] = (unordered(floor) - m) * p.scale - logs;
      }
    __syncthreads();
  }
  for (int i = n + have + t; i < k; i += T) tokens[i] = -1, logprobs[i] = -INFINITY - logs;
}

template <int DT, bool TOP>
__global__ void __launch_bounds__(64 * W) logprobs_kernel(Params p) {
  constexpr int E = Vec<DT>::E, U = Vec<DT>::U, STEP = U * W * 64, QUADS = MAX_SPLITS / 4;
  __shared__ Shared sh;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x / p.S, split = blockIdx.x - row * p.S;
  const Row<DT> r(p, row);
  const int vb = max(split * p.per, r.whole_b), ve = min((split + 1) * p.per, r.whole_e);
  const unsigned low = DT == FA_DTYPE_F32 ? 0xff800000u : DT == FA_DTYPE_F16 ? 0xfc00fc00u : 0xff80ff80u;  // -inf

  u32x4 raw[U], next[U];
  auto fetch = [&](int v0) {
    const int v1 = v0 + threadIdx.x;
    if (v0 + STEP <= ve) {
#pragma unroll
      for (int u = 0; u < U; u++) next[u] = __builtin_nontemporal_load(r.base + v1 + u * W * 64);
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) {
        next[u] = u32x4{low, low, low, low};
        if (v1 + u * W * 64 < ve) next[u] = __builtin_nontemporal_load(r.base + v1 + u * W * 64);
      }
    }
  };
  Sums a{-INFINITY, 0.f, 0.f};
  if (split == 0 && r.end(threadIdx.x) >= 0) {
    const float x = value_at<DT>(r.x, r.end(threadIdx.x));
    a = Sums{x == x ? x : -INFINITY, x > -INFINITY ? 1.f : x == x ? 0.f : x, 0.f};
    if (x == INFINITY) a.s = NAN;
  }
  if (vb < ve) fetch(vb);
  float own = -INFINITY;  // the maximum of this thread's whole vectors
  for (int v0 = vb; v0 < ve; v0 += STEP) {
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = next[u];
    if (v0 + STEP < ve) fetch(v0 + STEP);
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < E; i++) most = fmaxf(most, value<DT>(raw[u], i));
    own = fmaxf(own, most);
    const float m = fmaxf(a.m, most), ms = m == -INFINITY ? 0.f : m;
    const float down = fmaxf((a.m - ms) * p.c, LEAST), w = exp2_w(down);
    a.t = w * (a.t + down * a.s);
    a.s *= w;
    a.m = m;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < E; i++) {
        const float d = (value<DT>(raw[u], i) - ms) * p.c, e = exp2_w(d);
        a.s += e;
        a.t += fmaxf(d, LEAST) * e;
      }
  }
  a = sum_lanes(a, p.c);
  if (lane == 0) sh.sums[wave] = a;
  __syncthreads();
  a = sum_lanes(lane < W ? sh.sums[lane] : Sums{-INFINITY, 0.f, 0.f}, p.c);
  f32x4 maxima[TOP ? QUADS : 1];  // the threads' of all splits: quad i of this thread is of split 4 i + wave, threads 4 lane ..
  if (p.S > 1) {
    constexpr int one = part_floats(TOP);
    const rsrc_t parts = make_rsrc(p.part + (size_t)row * p.S * one, (uint32_t)(p.S * one * 4));
    if (threadIdx.x == 0) stb128<kCpSc1>(parts, split * one * 4, u32x4{as_u32(a.m), as_u32(a.s), as_u32(a.t), 0});
    if constexpr (TOP) __builtin_amdgcn_raw_buffer_store_b32(as_u32(own), parts, (split * one + 4 + threadIdx.x) * 4, 0, kCpSc1);
    if (!arrived_last(p.arrived + (size_t)row * p.S, p.nonce, split, p.S, &sh.flag)) return;
    const u32x4 x = ldb128<kCpSc1>(parts, lane < p.S ? lane * one * 4 : 0);
    if constexpr (TOP) {
#pragma unroll
      for (int i = 0; i < QUADS; i++) {
        maxima[i] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (4 * i + wave < p.S) maxima[i] = as_f32x4(ldb128<kCpSc1>(parts, ((4 * i + wave) * one + 4 + 4 * lane) * 4));
      }
    }
    a = sum_lanes(lane < p.S ? Sums{as_f32(x[0]), as_f32(x[1]), as_f32(x[2])} : Sums{-INFINITY, 0.f, 0.f}, p.c);
  }
  const bool nothing = a.m == -INFINITY && a.s == 0.f;
  const float logs = nothing ? 0.f : logf(a.s), m = nothing ? 0.f : a.m;
  if (threadIdx.x == 0) {
    const int64_t token = p.wide ? static_cast<const int64_t*>(p.tokens)[row] : static_cast<const int*>(p.tokens)[row];
    float z = -INFINITY;
    if (token >= 0 && token < p.V) z = value_at<DT>(r.x, (int)token);
    p.logprob[row] = (z - m) * p.scale - logs;
    p.entropy[row] = nothing ? 0.f : logs - a.t / a.s * LN2;
  }
  if constexpr (TOP) alternatives<DT>(p, r, row, sh, m, logs, own, maxima);
}

// Workgroups of a row: about 1024 for all rows, each with a batch of every thread or more. Up to 32: the pass of one row becomes no shorter
// with more, and the join reads more maxima (262144 values, 16, 32 and 64 workgroups, us: bf16, 8 alternatives, 1 row 11.1, 10.4, 10.6, 2 rows
// 11.8, 10.8, 10.8, 16 rows 12.3, 12.6, 15.6; without alternatives 7.0, 6.2, 6.2; fp32, 1 alternative 10.1, 9.8, 10.3). `per`: vectors of each.
int splits_for(int rows, int V, int dtype, int* per = nullptr) {
  const int e = dtype == FA_DTYPE_F32 ? 4 : 8, nv = V / e + 2, batch = 64 * W * 16 / e;
  const int most = std::max(1, std::min({MAX_SPLITS, (nv + batch - 1) / batch, 1024 / std::min(rows, 1024)}));
  const int each = (nv + most - 1) / most;
  if (per) *per = each;
  return (nv + each - 1) / each;
}
size_t arrived_bytes(int rows, int S) { return ((size_t)rows * S * sizeof(uint64_t) + 255) / 256 * 256; }
size_t workspace(int rows, int S, int top) {
  return S == 1 ? 0 : arrived_bytes(rows, S) + (size_t)rows * S * part_floats(top > 0) * sizeof(float);
}

template <int DT>
void launch(const Params& p, hipStream_t s) {
  const dim3 grid((unsigned)p.rows * p.S);
  if (p.top) hipLaunchKernelGGL((logprobs_kernel<DT, true>), grid, dim3(64 * W), 0, s, p);
  else hipLaunchKernelGGL((logprobs_kernel<DT, false>), grid, dim3(64 * W), 0, s, p);
}

}  // namespace tokens
}  // namespace fa

extern "C" size_t fa_token_logprobs_workspace_bytes(int dtype, int rows, int vocabulary, int top) {
  if (rows < 1 || vocabulary < 1 || top < 0 || top > FA_TOKENS_MAX_TOP) return 0;
  return fa::tokens::workspace(rows, fa::tokens::splits_for(rows, vocabulary, dtype), top);
}

extern "C" int fa_token_logprobs(const fa_token_logprobs_args* a, fa_stream_t stream) {
  using namespace fa;
  const char* who = "fa_token_logprobs";
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->dtype != FA_DTYPE_BF16 && a->dtype != FA_DTYPE_F16 && a->dtype != FA_DTYPE_F32)
    return host::fail(FA_ERR_INVALID_ARG, "%s: dtype %d: logits are bf16, fp16 or fp32", who, a->dtype);
  if (a->rows < 0 || a->rows > (1 << 20) || a->vocabulary < 1 || a->vocabulary > (1 << 30))
    return host::fail(FA_ERR_INVALID_ARG, "%s: rows=%d outside [0, 2^20] or vocabulary=%d outside [1, 2^30]", who, a->rows, a->vocabulary);
  if (a->top < 0 || a->top > FA_TOKENS_MAX_TOP || a->top > a->vocabulary)
    return host::fail(FA_ERR_INVALID_ARG, "%s: top=%d outside [0, %d] or more than the vocabulary of %d", who, a->top, FA_TOKENS_MAX_TOP,
                      a->vocabulary);
  if (!(a->scale > 0.f) || !(a->scale * tokens::LOG2E < INFINITY))
    return host::fail(FA_ERR_INVALID_ARG, "%s: scale=%g must be positive and finite", who, a->scale);
  if (a->rows == 0) return FA_OK;
  const unsigned xb = a->dtype == FA_DTYPE_F32 ? 4 : 2, tb = a->wide_tokens ? 8 : 4;
  const struct {
    const void* p;
    const char* name;
    unsigned align;
    bool need;
  } ptrs[] = {{a->logits, "logits", xb, true}, {a->tokens, "tokens", tb, true}, {a->logprob, "logprob", 4, true},
              {a->entropy, "entropy", 4, true}, {a->top_tokens, "top_tokens", 4, a->top > 0},
              {a->top_logprobs, "top_logprobs", 4, a->top > 0}};
  for (const auto& t : ptrs) {
    if (t.need && !t.p) return host::fail(FA_ERR_INVALID_ARG, "%s: %s is NULL", who, t.name);
    if (reinterpret_cast<uintptr_t>(t.p) % t.align) return host::fail(FA_ERR_INVALID_ARG, "%s: %s is not %u-byte aligned", who, t.name, t.align);
  }
  int per = 0;
  const int S = tokens::splits_for(a->rows, a->vocabulary, a->dtype, &per);
  const size_t need = tokens::workspace(a->rows, S, a->top);
  if (need && (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return host::fail(FA_ERR_INVALID_ARG, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, need,
                      a->workspace ? a->workspace_bytes : (size_t)0);
  const int rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  tokens::Params p{};
  p.x = static_cast<const unsigned char*>(a->logits), p.xs = a->stride, p.tokens = a->tokens, p.wide = a->wide_tokens;
  p.scale = a->scale, p.c = a->scale * tokens::LOG2E, p.rows = a->rows, p.V = a->vocabulary, p.top = a->top, p.S = S, p.per = per;
  p.logprob = a->logprob, p.entropy = a->entropy, p.top_tokens = a->top_tokens, p.top_logprobs = a->top_logprobs;
  if (S > 1) {
    p.arrived = static_cast<uint64_t*>(a->workspace), p.nonce = host::launch_nonce();
    p.part = reinterpret_cast<float*>(static_cast<unsigned char*>(a->workspace) + tokens::arrived_bytes(a->rows, S));
  }
  if (a->dtype == FA_DTYPE_F32) tokens::launch<FA_DTYPE_F32>(p, (hipStream_t)stream);
  else if (a->dtype == FA_DTYPE_F16) tokens::launch<FA_DTYPE_F16>(p, (hipStream_t)stream);
  else tokens::launch<FA_DTYPE_BF16>(p, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return host::fail(FA_ERR_LAUNCH, "%s: %s", who, hipGetErrorString(e));
  return FA_OK;
}
