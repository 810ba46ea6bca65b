// Low-rank adapters of many requests beside a shared projection (fa_lora_add): row m of x has the adapter a = index[m], or none.
//
//   out[m] = y[m] + s_a B_a (A_a x[m]);   gate: out'[m][f] = gelu_tanh(out[m][2f]) out[m][2f + 1]
//
// Two launches: h[m] = A_a x[m] (`rank` values a row), whose K is split over waves and workgroups, and the way back to N. Bound by
// bytes: x, y and out once, each adapter in use once (from HBM; row tiles that share one meet it in the L2). Both products
// run on the 16x16x32 MFMA in tiles of 16 rows: of each adapter that a tile's rows name, the product is taken of the whole tile and kept
// for its own rows. So a prompt's tile costs one product, a tile of sixteen requests up to sixteen, and nothing of one
// request's adapter, NaN included, reaches another one's rows.
//
// Layout (laid out once): a[adapter][K / 8][rank][8] and b[adapter][rank / 8][N][8], so that the lanes of an MFMA operand find
// their 8 inner elements side by side, 16 rank rows or 4 outputs in one run of memory.
//
// h stays fp32: for the second product it is split into two values of the weights' type, h = hi + lo (2^-17 lost in bf16, 2^-22 in
// fp16, where a power of two per row keeps both in its range); the inner dimension holds hi, then lo, so rank 16 takes one MFMA.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"

namespace fa {
namespace lora {

constexpr int W = 4;          // waves of a workgroup
constexpr int MAX_RANK = 128;
constexpr int MAX_SPLITS = 16;

struct Params {
  const unsigned short* x;
  int64_t xs;  // row stride of x, elements
  const unsigned short *a, *b;
  const float* scale;
  const int* index;
  const void* y;
  void* out;
  float* h;  // [split][M][rank]
  int M, N, K, rank, adapters, splits, share;  // share: workgroups that deal a tile's adapters among them
};

template <bool F16>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  return F16 ? mfma16h(a, b, c) : mfma16(a, b, c);
}

// The adapters that a tile of ROWS rows names, one after the other: each(adapter, lanes), bit i of lanes: row i is its own.
template <int ROWS, class F>
__device__ __forceinline__ void for_adapters(const Params& p, int m0, int first, int step, F&& each) {
  const int i = threadIdx.x & 63;
  int mine = -1;
  if (i < ROWS && m0 + i < p.M) mine = p.index[m0 + i];
  const bool has = (unsigned)mine < (unsigned)p.adapters;
  uint64_t todo = __builtin_amdgcn_ballot_w64(has);
  for (int n = 0; todo; n++) {
    const int ad = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    const uint64_t own = __builtin_amdgcn_ballot_w64(has && mine == ad);
    todo &= ~own;
    if (n % step == first) each(ad, own);
  }
}

// h of MB tiles of 16 rows. RT: tiles of 16 rank rows. D[j][m] += A[j][k] x[m][k]; lane r + 16 q holds k = 64 c + 16 q + 8 s .. + 7 of
// chunk c (s = 0, 1: a row's 128 bytes of a chunk are read by four lanes).
template <bool F16, int RT, int MB>
__global__ void __launch_bounds__(64 * W) shrink_kernel(Params p) {
  constexpr int PITCH = RT * 16 + 4;
  __shared__ float sums[W][MB * 16][PITCH];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  const int m0 = blockIdx.x * (16 * MB), split = blockIdx.y, K8 = p.K >> 3, nch = (p.K + 63) >> 6;
  const int part = split * W + wave, parts = p.splits * W;
  const int cb = (int)((int64_t)nch * part / parts), ce = (int)((int64_t)nch * (part + 1) / parts);
  const unsigned short* xr[MB];
#pragma unroll
  for (int b = 0; b < MB; b++) xr[b] = p.x + (int64_t)min(m0 + b * 16 + r, p.M - 1) * p.xs;
  for_adapters<16 * MB>(p, m0, blockIdx.z, p.share, [&](int ad, uint64_t own) {
    const unsigned short* a = p.a + (size_t)ad * K8 * p.rank * 8;
    f32x4 acc[RT][MB];
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int b = 0; b < MB; b++) acc[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto step = [&](int c, bool whole) {
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const int k8 = 8 * c + 2 * q + s, at = whole ? k8 : min(k8, K8 - 1);
        u32x4 x[MB];
#pragma unroll
        for (int b = 0; b < MB; b++) {
          x[b] = *reinterpret_cast<const u32x4*>(xr[b] + at * 8);
          if (!whole && k8 >= K8) x[b] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int t = 0; t < RT; t++) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(a + ((size_t)at * p.rank + min(t * 16 + r, p.rank - 1)) * 8);
#pragma unroll
          for (int b = 0; b < MB; b++) acc[t][b] = mma<F16>(w, x[b], acc[t][b]);
        }
      }
    };
    const int whole = min(ce, p.K >> 6);
    int c = cb;
    for (; c + 4 <= whole; c += 4)
#pragma unroll
      for (int u = 0; u < 4; u++) step(c + u, true);
    for (; c < whole; c++) step(c, true);
    if (c < ce) step(c, false);
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int b = 0; b < MB; b++) *reinterpret_cast<f32x4*>(&sums[wave][b * 16 + r][t * 16 + 4 * q]) = acc[t][b];
    __syncthreads();
    for (int e = threadIdx.x; e < MB * 16 * p.rank; e += 64 * W) {
      const int m = e / p.rank, j = e - m * p.rank;
      if (!(own >> m & 1)) continue;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < W; w++) v += sums[w][m][j];
      p.h[((size_t)split * p.M + m0 + m) * p.rank + j] = v;
    }
    __syncthreads();
  });
}

template <int DT>
__device__ __forceinline__ float elem(const void* p, size_t i) {
  if constexpr (DT == FA_DTYPE_F32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == FA_DTYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
  else return as_f32((unsigned)static_cast<const unsigned short*>(p)[i] << 16);
}
template <int DT>
__device__ __forceinline__ void put(void* p, size_t i, float v) {
  if constexpr (DT == FA_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if constexpr (DT == FA_DTYPE_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
  else static_cast<unsigned short*>(p)[i] = bf16_bits(v);
}
// Four neighbours, aligned.
template <int DT>
__device__ __forceinline__ f32x4 elem4(const void* p, size_t i) {
  if constexpr (DT == FA_DTYPE_F32) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
  const u32x2 v = *reinterpret_cast<const u32x2*>(static_cast<const unsigned short*>(p) + i);
  if constexpr (DT == FA_DTYPE_F16) return f32x4{h_lo(v[0]), h_hi(v[0]), h_lo(v[1]), h_hi(v[1])};
  else return f32x4{bf_lo(v[0]), bf_hi(v[0]), bf_lo(v[1]), bf_hi(v[1])};
}
template <int DT>
__device__ __forceinline__ void put4(void* p, size_t i, f32x4 v) {
  if constexpr (DT == FA_DTYPE_F32) *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = v;
  else if constexpr (DT == FA_DTYPE_F16)
    *reinterpret_cast<u32x2*>(static_cast<unsigned short*>(p) + i) = u32x2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
  else
    *reinterpret_cast<u32x2*>(static_cast<unsigned short*>(p) + i) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

// The way back: a wave takes 16 MB rows x 64 outputs. D[m][n] += h[m][k] B[n][k]; column r of MFMA t is output n0 + 4 r + t, so a
// lane ends with four neighbouring outputs of rows 4 q .. 4 q + 3. CH: chunks of 32 inner slots: groups of 8, the R8 = rank / 8
// of hi, then those of lo. QUADS: rows of y and out keep four neighbours aligned.
template <bool F16, int CH, int MB, int YT, bool GATE, bool QUADS>
__global__ void __launch_bounds__(64 * W) expand_kernel(Params p) {
  extern __shared__ float hs[];  // [16 MB][rank + 4]: the pad spreads the rows over the banks
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  const int m0 = blockIdx.y * (16 * MB), n0 = (blockIdx.x * W + wave) * 64, R8 = p.rank >> 3, pitch = p.rank + 4;
  const int rows = min(16 * MB, p.M - m0);
  for (int e = threadIdx.x; e < rows * p.rank; e += 64 * W) {
    const int m = e / p.rank, ad = p.index[m0 + m];
    if ((unsigned)ad >= (unsigned)p.adapters) continue;
    float v = 0.f;
    for (int s = 0; s < p.splits; s++) v += p.h[((size_t)s * p.M + m0) * p.rank + e];
    hs[m * pitch + e - m * p.rank] = v * p.scale[ad];
  }
  __syncthreads();
  if (n0 >= p.N) return;
  // hi and lo of this lane's row and slots
  u32x4 hf[MB][CH];
  float up[MB];  // the power of two that h was divided by
#pragma unroll
  for (int b = 0; b < MB; b++) {
    const float* row = hs + min(b * 16 + r, rows - 1) * pitch;
    up[b] = 1.f;
    if constexpr (F16) {
      float most = 0.f;
      for (int j = q; j < p.rank; j += 4) most = fmaxf(most, fabsf(row[j]));
      most = cols_max(most);
      // the largest into [2^13, 2^14): lo is held to 2^-38 of it
      if (most > 0.f && most < INFINITY) up[b] = ldexpf(1.f, max(-126, min(126, ilogbf(most) - 13)));
    }
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const int g = 4 * c + q, k = (g < R8 ? g : g - R8) * 8;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        hf[b][c][i] = 0;
        if (g < 2 * R8) {
          const float v0 = row[k + 2 * i] / up[b], v1 = row[k + 2 * i + 1] / up[b];
          const unsigned hi = F16 ? pack_f16x2(v0, v1) : pack_bf16x2(v0, v1);
          const float l0 = v0 - (F16 ? h_lo(hi) : bf_lo(hi)), l1 = v1 - (F16 ? h_hi(hi) : bf_hi(hi));
          hf[b][c][i] = g < R8 ? hi : F16 ? pack_f16x2(l0, l1) : pack_bf16x2(l0, l1);
        }
      }
    }
  }
  f32x4 acc[MB][4];  // [t]: rows 4 q + i, output n0 + 4 r + t
#pragma unroll
  for (int b = 0; b < MB; b++)
#pragma unroll
    for (int t = 0; t < 4; t++) acc[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for_adapters<16 * MB>(p, m0, 0, 1, [&](int ad, uint64_t own) {
    const unsigned short* w = p.b + (size_t)ad * R8 * p.N * 8;
    f32x4 one[MB][4];
#pragma unroll
    for (int b = 0; b < MB; b++)
#pragma unroll
      for (int t = 0; t < 4; t++) one[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const int g = min(4 * c + q, 2 * R8 - 1), k8 = g < R8 ? g : g - R8;
#pragma unroll
      for (int t = 0; t < 4; t++) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(w + ((size_t)k8 * p.N + min(n0 + 4 * r + t, p.N - 1)) * 8);
#pragma unroll
        for (int b = 0; b < MB; b++) one[b][t] = mma<F16>(hf[b][c], v, one[b][t]);
      }
    }
#pragma unroll
    for (int b = 0; b < MB; b++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (own >> (b * 16 + 4 * q + i) & 1)
#pragma unroll
          for (int t = 0; t < 4; t++) acc[b][t][i] = one[b][t][i];
  });
  float factor[MB][4];  // of rows 4 q + i: their lanes must still be there
#pragma unroll
  for (int b = 0; b < MB; b++)
#pragma unroll
    for (int i = 0; i < 4; i++) factor[b][i] = F16 ? __shfl(up[b], 4 * q + i) : 1.f;
  const int n = n0 + 4 * r;
  if (n >= p.N) return;
#pragma unroll
  for (int b = 0; b < MB; b++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int m = b * 16 + 4 * q + i;
      const float f = factor[b][i];
      if (m >= rows) continue;
      const size_t at = (size_t)(m0 + m) * p.N + n;
      f32x4 v = f32x4{acc[b][0][i] * f, acc[b][1][i] * f, acc[b][2][i] * f, acc[b][3][i] * f};
      if constexpr (QUADS) {
        v += elem4<YT>(p.y, at);
        if constexpr (GATE)
          reinterpret_cast<unsigned*>(p.out)[at >> 2] = F16 ? pack_f16x2(gelu_tanh(v[0]) * v[1], gelu_tanh(v[2]) * v[3])
                                                            : pack_bf16x2(gelu_tanh(v[0]) * v[1], gelu_tanh(v[2]) * v[3]);
        else put4<YT>(p.out, at, v);
      } else {
#pragma unroll
        for (int t = 0; t < 4; t++)
          if (n + t < p.N) v[t] += elem<YT>(p.y, at + t);
#pragma unroll
        for (int t = 0; t < 4; t += GATE ? 2 : 1) {
          if (n + t >= p.N) continue;
          if constexpr (GATE) put<F16 ? FA_DTYPE_F16 : FA_DTYPE_BF16>(p.out, (at + t) >> 1, gelu_tanh(v[t]) * v[t + 1]);
          else put<YT>(p.out, at + t, v[t]);
        }
      }
    }
}

// Splits of K across workgroups.
int splits_for(int M, int K, int rank) {
  const int tiles = (M + 15) / 16, nch = (K + 63) / 64;
  return std::max(1, std::min({512 / tiles, nch / (2 * W), MAX_SPLITS}));
}

template <bool F16, int RT>
void launch_shrink(const Params& p, hipStream_t s) {
  if (p.M > 256)
    hipLaunchKernelGGL((shrink_kernel<F16, RT, 2>), dim3((p.M + 31) / 32, p.splits, p.share), dim3(64 * W), 0, s, p);
  else
    hipLaunchKernelGGL((shrink_kernel<F16, RT, 1>), dim3((p.M + 15) / 16, p.splits, p.share), dim3(64 * W), 0, s, p);
}

template <bool F16, int CH, int YT, bool GATE>
void launch_expand(const Params& p, bool quads, hipStream_t s) {
  const int blocks = (p.N + 64 * W - 1) / (64 * W);
  if (p.M > 256) {
    const dim3 grid(blocks, (p.M + 31) / 32);
    const unsigned lds = 32 * (p.rank + 4) * sizeof(float);
    if (quads) hipLaunchKernelGGL((expand_kernel<F16, CH, 2, YT, GATE, true>), grid, dim3(64 * W), lds, s, p);
    else hipLaunchKernelGGL((expand_kernel<F16, CH, 2, YT, GATE, false>), grid, dim3(64 * W), lds, s, p);
  } else {
    const dim3 grid(blocks, (p.M + 15) / 16);
    const unsigned lds = 16 * (p.rank + 4) * sizeof(float);
    if (quads) hipLaunchKernelGGL((expand_kernel<F16, CH, 1, YT, GATE, true>), grid, dim3(64 * W), lds, s, p);
    else hipLaunchKernelGGL((expand_kernel<F16, CH, 1, YT, GATE, false>), grid, dim3(64 * W), lds, s, p);
  }
}

template <bool F16, int CH>
void launch_expand(const Params& p, int yt, bool gate, bool quads, hipStream_t s) {
  constexpr int XT = F16 ? FA_DTYPE_F16 : FA_DTYPE_BF16;
  if (yt == FA_DTYPE_F32) {
    if (gate) launch_expand<F16, CH, FA_DTYPE_F32, true>(p, quads, s);
    else launch_expand<F16, CH, FA_DTYPE_F32, false>(p, quads, s);
  } else {
    if (gate) launch_expand<F16, CH, XT, true>(p, quads, s);
    else launch_expand<F16, CH, XT, false>(p, quads, s);
  }
}

template <bool F16>
void launch(const Params& p, int yt, bool gate, bool quads, hipStream_t s) {
  if (p.rank <= 16) launch_shrink<F16, 1>(p, s), launch_expand<F16, 1>(p, yt, gate, quads, s);
  else if (p.rank <= 32) launch_shrink<F16, 2>(p, s), launch_expand<F16, 2>(p, yt, gate, quads, s);
  else if (p.rank <= 64) launch_shrink<F16, 4>(p, s), launch_expand<F16, 4>(p, yt, gate, quads, s);
  else launch_shrink<F16, 8>(p, s), launch_expand<F16, 8>(p, yt, gate, quads, s);
}

}  // namespace lora
}  // namespace fa

extern "C" size_t fa_lora_workspace_bytes(int rows, int k, int rank) {
  if (rows < 1 || k < 8 || rank < 8 || rank > fa::lora::MAX_RANK || k > (1 << 24)) return 0;
  return (size_t)fa::lora::splits_for(rows, k, rank) * rows * rank * sizeof(float);
}

extern "C" int fa_lora_add(const fa_lora_args* a, fa_stream_t stream) {
  using namespace fa;
  const char* who = "fa_lora_add";
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->dtype != FA_DTYPE_BF16 && a->dtype != FA_DTYPE_F16)
    return host::fail(FA_ERR_INVALID_ARG, "%s: dtype %d: x and the adapters are bf16 or fp16", who, a->dtype);
  if (a->y_dtype != FA_DTYPE_F32 && a->y_dtype != a->dtype)
    return host::fail(FA_ERR_INVALID_ARG, "%s: y_dtype %d: y is fp32 or of x's type", who, a->y_dtype);
  if (a->rows < 0 || a->rows > (1 << 24)) return host::fail(FA_ERR_INVALID_ARG, "%s: rows=%d outside [0, 2^24]", who, a->rows);
  if (a->n < 1 || a->k < 8 || a->k % 8 || a->n > (1 << 24) || a->k > (1 << 24))
    return host::fail(FA_ERR_INVALID_ARG, "%s: need 1 <= n, k <= 2^24 and k a multiple of 8, got n=%d k=%d", who, a->n, a->k);
  if (a->rank < 8 || a->rank > lora::MAX_RANK || a->rank % 8)
    return host::fail(FA_ERR_INVALID_ARG, "%s: rank=%d is no multiple of 8 up to %d", who, a->rank, lora::MAX_RANK);
  if (a->adapters < 1 || a->adapters > (1 << 20)) return host::fail(FA_ERR_INVALID_ARG, "%s: adapters=%d", who, a->adapters);
  if (a->gate && a->n % 2) return host::fail(FA_ERR_INVALID_ARG, "%s: the gated form needs an even n, got %d", who, a->n);
  if (a->rows == 0) return FA_OK;
  const unsigned yb = a->y_dtype == FA_DTYPE_F32 ? 4 : 2, ob = a->gate ? 2 : yb;
  const struct {
    const void* p;
    const char* name;
    unsigned align;
  } ptrs[] = {{a->x, "x", 16}, {a->a, "a", 16}, {a->b, "b", 16}, {a->scale, "scale", 4}, {a->index, "index", 4}, {a->y, "y", yb},
              {a->out, "out", ob}};
  for (const auto& t : ptrs) {
    if (!t.p) return host::fail(FA_ERR_INVALID_ARG, "%s: %s is NULL", who, t.name);
    if (reinterpret_cast<uintptr_t>(t.p) % t.align) return host::fail(FA_ERR_INVALID_ARG, "%s: %s is not %u-byte aligned", who, t.name, t.align);
  }
  if (a->rows > 1 && (a->x_stride < a->k || a->x_stride % 8))
    return host::fail(FA_ERR_INVALID_ARG, "%s: x_stride=%lld must be a multiple of 8 and >= k=%d", who, (long long)a->x_stride, a->k);
  const size_t need = fa_lora_workspace_bytes(a->rows, a->k, a->rank);
  if (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16)
    return host::fail(FA_ERR_INVALID_ARG, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, need,
                      a->workspace ? a->workspace_bytes : (size_t)0);
  int rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  lora::Params p{static_cast<const unsigned short*>(a->x), a->x_stride, static_cast<const unsigned short*>(a->a),
                 static_cast<const unsigned short*>(a->b), a->scale, a->index, a->y, a->out, static_cast<float*>(a->workspace),
                 a->rows, a->n, a->k, a->rank, a->adapters, lora::splits_for(a->rows, a->k, a->rank),
                 a->rows > 64 ? 1 : std::min({16, a->rows, a->adapters})};
  const bool quads = a->n % 4 == 0 && reinterpret_cast<uintptr_t>(a->y) % (4 * yb) == 0 &&
                     reinterpret_cast<uintptr_t>(a->out) % (a->gate ? 4 : 4 * ob) == 0;
  if (a->dtype == FA_DTYPE_F16) lora::launch<true>(p, a->y_dtype, a->gate, quads, (hipStream_t)stream);
  else lora::launch<false>(p, a->y_dtype, a->gate, quads, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return host::fail(FA_ERR_LAUNCH, "%s: %s", who, hipGetErrorString(e));
  return FA_OK;
}
