// Log probabilities of given tokens, with entropy and the best alternatives (fa_token_logprobs), out of logits read once.
//
//   z = scale x;  m = max z, s = sum e^(z - m), t = sum (z - m) e^(z - m):
//   log p_i = z_i - m - log s,  entropy = log s - t / s,  alternatives by (x descending, index ascending).
//
// Bound by reading the logits. A workgroup takes a part of a row, 16 values a thread at a time; every lane keeps its own running
// maximum (of x, exact) and sums. The alternatives are a sorted list in the lanes of each wave, lane i the i-th best. Against it
// each batch costs one comparison of the lane's maximum, which the running maximum needs anyway; only where that passes the list's
// last are the single values looked at, and those that pass are inserted one by one. A wave's first batch is filtered by
// a bound under which k values lie: the k-th largest of the lanes' maxima, by bisection of their upper 16 bits. Behind it a
// batch of n values after N has k n / N that pass.
// Few rows are split over up to 64 workgroups, whose sums and lists the last one to arrive joins.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"

namespace fa {
namespace tokens {

constexpr int W = 4;  // waves of a workgroup
constexpr int MAX_SPLITS = 64;
constexpr int NONE = 0x7fffffff;  // index of an alternative that is not there
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LEAST = -1e30f;  // for -inf where it is multiplied by a weight of 0

struct Params {
  const unsigned char* x;
  int64_t xs;  // row stride, elements
  const void* tokens;
  int wide;  // tokens are 64-bit
  float scale, c;  // c: scale log2(e)
  int rows, V, top, S;
  float *logprob, *entropy;
  int* top_tokens;
  float* top_logprobs;
  float* part;  // [row][split] {m, s, t, 0, {x, index}[top]}
  uint64_t *arrived, nonce;  // [row][split]
};
__host__ __device__ constexpr int part_floats(int top) { return 4 + 2 * top; }

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

// A wave's best alternatives: lane i < k holds the i-th.
struct Best {
  float v;
  int i;
  float last_v;  // the k-th
  int last_i, k;

  __device__ __forceinline__ void clear(int top) { v = last_v = -INFINITY, i = last_i = NONE, k = top; }
  __device__ __forceinline__ bool passes(float x, int at) const { return x > last_v || (x == last_v && at < last_i); }
  __device__ __forceinline__ void insert(float x, int at) {
    const bool before = v > x || (v == x && i < at);  // a prefix of the lanes
    const int place = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before)), lane = threadIdx.x & 63;
    const float up_v = __shfl_up(v, 1);
    const int up_i = __shfl_up(i, 1);
    v = lane < place ? v : lane == place ? x : up_v;
    i = lane < place ? i : lane == place ? at : up_i;
    last_v = as_f32(__builtin_amdgcn_readlane(as_u32(v), k - 1));
    last_i = __builtin_amdgcn_readlane(i, k - 1);
  }
  // Each lane offers one value; whether any passed.
  __device__ __forceinline__ bool offer(float x, int at, bool there) {
    uint64_t todo = __builtin_amdgcn_ballot_w64(there && passes(x, at));
    if (!todo) return false;
    do {
      const int l = __builtin_ctzll(todo);
      insert(as_f32(__builtin_amdgcn_readlane(as_u32(x), l)), __builtin_amdgcn_readlane(at, l));
      todo &= todo - 1;
      todo &= __builtin_amdgcn_ballot_w64(passes(x, at));
    } while (todo);
    return true;
  }
};

// A bound that at least k of the lanes' values x reach: their k-th largest, its lower 16 bits cleared downwards.
__device__ __forceinline__ float kth_bound(float x, int k) {
  const unsigned u = as_u32(x), key = (u >> 31 ? ~u : u | 0x80000000u) >> 16;  // ordered as the values are
  unsigned p = 0;
#pragma unroll
  for (int bit = 15; bit >= 0; bit--) {
    const unsigned next = p | 1u << bit;
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= next)) >= k) p = next;
  }
  if (p <= 0x007fu) return -INFINITY;  // the key of -inf
  const unsigned b = p << 16;
  return as_f32(b >> 31 ? b & 0x7fffffffu : ~b);
}

struct Sums {
  float m, s, t;
};
// The lanes' sums as one, in every lane.
__device__ __forceinline__ Sums sum_lanes(Sums x, float c) {
  Sums y;
  y.m = wave_max(x.m);
  const float d = fmaxf((x.m - (y.m == -INFINITY ? 0.f : y.m)) * c, LEAST), a = exp2_w(d);
  y.s = wave_sum(a * x.s);
  y.t = wave_sum(a * (x.t + d * x.s));
  return y;
}

template <int DT, bool TOP>
__global__ void __launch_bounds__(64 * W) logprobs_kernel(Params p) {
  constexpr int E = Vec<DT>::E, U = Vec<DT>::U, BYTES = Vec<DT>::BYTES;
  __shared__ Sums sums[W];
  __shared__ float list_v[W][FA_TOKENS_MAX_TOP];
  __shared__ int list_i[W][FA_TOKENS_MAX_TOP], flag;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x / p.S, split = blockIdx.x - row * p.S;
  const unsigned char* x = p.x + (int64_t)row * p.xs * BYTES;
  // vectors of 16 aligned bytes; the first may begin before the row and the last end behind it
  const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15) / BYTES;
  const int nv = (int)(((int64_t)off + p.V + E - 1) / E);
  const int vb = (int)((int64_t)nv * split / p.S), ve = (int)((int64_t)nv * (split + 1) / p.S);
  const int whole_b = off ? 1 : 0, whole_e = (int)(((int64_t)off + p.V) / E);  // vectors that lie in the row
  const u32x4* base = reinterpret_cast<const u32x4*>(x - off * BYTES);
  const unsigned low = DT == FA_DTYPE_F32 ? 0xff800000u : DT == FA_DTYPE_F16 ? 0xfc00fc00u : 0xff80ff80u;  // -inf

  Sums a{-INFINITY, 0.f, 0.f};
  Best best;
  if constexpr (TOP) best.clear(p.top);
  bool fresh = true;
  for (int v0 = vb; v0 < ve; v0 += U * W * 64) {
    u32x4 raw[U];
    if (v0 >= whole_b && v0 + U * W * 64 <= min(ve, whole_e)) {
#pragma unroll
      for (int u = 0; u < U; u++) raw[u] = __builtin_nontemporal_load(base + v0 + (u * W + wave) * 64 + lane);
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int v = v0 + (u * W + wave) * 64 + lane;
        raw[u] = u32x4{low, low, low, low};
        if (v >= ve) continue;
        if (v >= whole_b && v < whole_e) {
          raw[u] = __builtin_nontemporal_load(base + v);
        } else {
#pragma unroll
          for (int i = 0; i < E; i++) {
            const int64_t at = (int64_t)v * E - off + i;
            if (at < 0 || at >= p.V) continue;
            if constexpr (DT == FA_DTYPE_F32) {
              raw[u][i] = reinterpret_cast<const unsigned*>(x)[at];
            } else {
              const unsigned w = reinterpret_cast<const unsigned short*>(x)[at];
              raw[u][i >> 1] = i & 1 ? (raw[u][i >> 1] & 0xffffu) | w << 16 : (raw[u][i >> 1] & 0xffff0000u) | w;
            }
          }
        }
      }
    }
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < E; i++) most = fmaxf(most, value<DT>(raw[u], i));
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
    if constexpr (TOP) {
      float bound = best.last_v;
      if (fresh) bound = kth_bound(most, p.top);
      fresh = false;
      if (__builtin_amdgcn_ballot_w64(most >= bound)) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int i = 0; i < E; i++) {
            const int64_t at = ((int64_t)v0 + (u * W + wave) * 64 + lane) * E - off + i;
            const float y = value<DT>(raw[u], i);
            best.offer(y, (int)at, y >= bound && at >= 0 && at < p.V && v0 + (u * W + wave) * 64 + lane < ve);
          }
      }
    }
  }
  a = sum_lanes(a, p.c);
  if (lane == 0) sums[wave] = a;
  if constexpr (TOP) {
    if (lane < p.top) list_v[wave][lane] = best.v, list_i[wave][lane] = best.i;
  }
  __syncthreads();
  if (wave == 0) {
    a = sum_lanes(lane < W ? sums[lane] : Sums{-INFINITY, 0.f, 0.f}, p.c);
    if constexpr (TOP) {
      constexpr int PER = 64 / FA_TOKENS_MAX_TOP;  // lists side by side
#pragma unroll
      for (int w0 = 1; w0 < W; w0 += PER) {  // the other waves'
        const int w = w0 + lane / FA_TOKENS_MAX_TOP, j = lane % FA_TOKENS_MAX_TOP;
        best.offer(list_v[min(w, W - 1)][j], list_i[min(w, W - 1)][j], w < W && j < p.top);
      }
    }
  }
  if (p.S > 1) {
    const int one = part_floats(TOP ? p.top : 0);
    const rsrc_t parts = make_rsrc(p.part + (size_t)row * p.S * one, (uint32_t)(p.S * one * 4));
    if (wave == 0) {
      if (lane == 0)
        stb128<kCpSc1>(parts, split * one * 4, u32x4{as_u32(a.m), as_u32(a.s), as_u32(a.t), 0});
      if constexpr (TOP)
        if (lane < p.top) stb64<kCpSc1>(parts, (split * one + 4 + 2 * lane) * 4, u32x2{as_u32(best.v), (unsigned)best.i});
    }
    if (!arrived_last(p.arrived + (size_t)row * p.S, p.nonce, split, p.S, &flag)) return;
    if (wave == 0) {
      const u32x4 s = lane < p.S ? ldb128<kCpSc1>(parts, lane * one * 4) : u32x4{as_u32(-INFINITY), 0, 0, 0};
      a = sum_lanes(Sums{as_f32(s[0]), as_f32(s[1]), as_f32(s[2])}, p.c);
      if constexpr (TOP) {
        best.clear(p.top);
        for (int j = 0; j < p.top; j++) {  // the lists are sorted: once no split's j-th passes, none does
          const u32x2 e = lane < p.S ? ldb64<kCpSc1>(parts, (lane * one + 4 + 2 * j) * 4) : u32x2{as_u32(-INFINITY), (unsigned)NONE};
          if (!best.offer(as_f32(e[0]), (int)e[1], lane < p.S)) break;
        }
      }
    }
  }
  if (wave != 0) return;
  const bool nothing = a.m == -INFINITY && a.s == 0.f;
  const float logs = nothing ? 0.f : logf(a.s), m = nothing ? 0.f : a.m;
  if (lane == 0) {
    const int64_t token = p.wide ? static_cast<const int64_t*>(p.tokens)[row] : static_cast<const int*>(p.tokens)[row];
    float z = -INFINITY;
    if (token >= 0 && token < p.V) z = value_at<DT>(x, (int)token);
    p.logprob[row] = (z - m) * p.scale - logs;
    p.entropy[row] = nothing ? 0.f : logs - a.t / a.s * LN2;
  }
  if constexpr (TOP) {
    if (lane < p.top) {
      p.top_tokens[(size_t)row * p.top + lane] = best.i == NONE ? -1 : best.i;
      p.top_logprobs[(size_t)row * p.top + lane] = (best.v - m) * p.scale - logs;
    }
  }
}

// Workgroups of a row: the chip full, each with a batch of every thread or more.
int splits_for(int rows, int V, int dtype) {
  const int batches = (int)(((int64_t)V + 64 * W * 16 - 1) / (64 * W * 16));
  return std::max(1, std::min({MAX_SPLITS, batches, 1024 / std::min(rows, 1024)}));
}
size_t arrived_bytes(int rows, int S) { return ((size_t)rows * S * sizeof(uint64_t) + 255) / 256 * 256; }
size_t workspace(int rows, int S, int top) {
  return S == 1 ? 0 : arrived_bytes(rows, S) + (size_t)rows * S * part_floats(top) * sizeof(float);
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
  if (a->rows < 0 || a->rows > (1 << 24) || a->vocabulary < 1 || a->vocabulary > (1 << 30))
    return host::fail(FA_ERR_INVALID_ARG, "%s: rows=%d outside [0, 2^24] or vocabulary=%d outside [1, 2^30]", who, a->rows, a->vocabulary);
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
  const int S = tokens::splits_for(a->rows, a->vocabulary, a->dtype);
  const size_t need = tokens::workspace(a->rows, S, a->top);
  if (need && (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return host::fail(FA_ERR_INVALID_ARG, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, need,
                      a->workspace ? a->workspace_bytes : (size_t)0);
  const int rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  tokens::Params p{};
  p.x = static_cast<const unsigned char*>(a->logits), p.xs = a->stride, p.tokens = a->tokens, p.wide = a->wide_tokens;
  p.scale = a->scale, p.c = a->scale * tokens::LOG2E, p.rows = a->rows, p.V = a->vocabulary, p.top = a->top, p.S = S;
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
