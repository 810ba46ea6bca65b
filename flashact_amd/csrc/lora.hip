// Low-rank adapters of many requests beside a shared projection (fa_lora_add): row m of x has the adapter a = index[m], or none.
//
//   out[m] = y[m] + s_a B_a (A_a x[m]);   gate: out'[m][f] = gelu_tanh(out[m][2f]) out[m][2f + 1]
//
// Two launches: h[m] = A_a x[m] (`rank` values a row), whose K is split over waves and workgroups, and the way back to N. Bound by
// bytes: x, y and out once, each adapter in use once (from HBM; row tiles that share one meet it in the L2). Both products
// run on the 16x16x32 MFMA in tiles of 16 rows: of each adapter that a tile's rows name, the product is taken of the whole tile and kept
// for its own rows (up to rank 16, two of them with one reading of x). So a prompt's tile costs one product, a tile of sixteen requests
// up to sixteen, and nothing of one request's adapter, NaN included, reaches another one's rows.
//
// Layout (laid out once): a[adapter][K / 8][rank][8] and b[adapter][rank / 8][N][8], so that the lanes of an MFMA operand find
// their 8 inner elements side by side, 16 rank rows or 4 outputs in one run of memory.
//
// h stays fp32: for the second product it is split into two values of the weights' type, h = hi + lo (2^-17 lost in bf16, 2^-22 in
// fp16, where a power of two per row keeps both in its range), or three where bf16 weights meet an fp32 result (2^-25); the inner
// dimension holds one part behind the other, so that rank 16 in two parts takes one MFMA.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"

namespace fa {
namespace lora {

constexpr int W = 4;  // waves of a workgroup on the way back
constexpr int MAX_RANK = 128;
constexpr int MAX_SPLITS = 4;
// Waves of a workgroup on the way to h, which deal K among them, at most; chunks of 64 columns that a wave asks for at once: by registers
// and LDS.
constexpr int shrink_waves(int rt) { return rt <= 2 ? 16 : 8; }
constexpr int shrink_ahead(int rt) { return rt <= 4 ? 4 : 2; }
// LDS bytes of a wave: its stage of x, later its sums.
constexpr int shrink_bytes(int rt) { return std::max(shrink_ahead(rt) * 2048, 16 * (rt * 16 + 4) * 4); }

struct Params {
  const unsigned short* x;
  int64_t xs;  // row stride of x, elements
  const unsigned short *a, *b;
  const float* scale;
  const int* index;
  const void* y;
  void* out;
  float* h;  // [split][M][rank]
  int M, N, K, rank, adapters, splits, waves;
  bool runs;  // neighbouring tiles on one XCD
  int share;  // workgroups that deal a tile's adapters among them
};

template <bool F16>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  return F16 ? mfma16h(a, b, c) : mfma16(a, b, c);
}

// The adapters that a tile of ROWS rows names, one after the other: each(adapter, lanes), bit i of lanes: row i is its own. Returns the
// rows that have none.
template <int ROWS, class F>
__device__ __forceinline__ uint64_t for_adapters(const Params& p, int m0, int first, int step, F&& each) {
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
  return __builtin_amdgcn_ballot_w64(i < ROWS && m0 + i < p.M && !has);
}

// h of a tile of 16 rows. RT: tiles of 16 rank rows. D[j][m] += A[j][k] x[m][k]; lane r + 16 q holds k = 64 c + 32 s + 8 q .. + 7 of
// chunk c in product s. x comes through LDS, private to the wave, four lanes to the 64 bytes of a row (lanes in MFMA order are taken
// one by one by the address unit: with the way back, 1993 rows of 16384 columns 38.8 us so and 34.8 in copies); the adapter's operand is
// one run of 1 KB at rank 16 as it lies.
template <bool F16, int RT>
__global__ void __launch_bounds__(64 * shrink_waves(RT)) shrink_kernel(Params p) {
  constexpr int PITCH = RT * 16 + 4, AHEAD = shrink_ahead(RT), BYTES = shrink_bytes(RT);
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int waves = blockDim.x >> 6;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  const int K8 = p.K >> 3, nch = (p.K + 63) >> 6;
  // Neighbouring tiles, which mostly name the same adapter, on one XCD, where each has eight or more (1993 rows, K 16384, seven adapters: 41.4
  // us with the way back, 37.5 so; five tiles of 70 rows 37.9 and 43.3).
  const int tiles = (p.M + 15) >> 4, per = (tiles + 7) >> 3, at = blockIdx.x >> 3;
  int split, tile;
  if (p.runs) split = at / per, tile = (blockIdx.x & 7) * per + at - split * per;
  else split = blockIdx.x / tiles, tile = blockIdx.x - split * tiles;
  if (tile >= tiles) return;
  const int m0 = tile * 16;
  // Runs of AHEAD chunks are dealt to the waves one by one, and each tile begins elsewhere: rows are often a power of two apart, and
  // tiles that walk through K side by side meet in the same memory channels.
  const int part = split * waves + wave, parts = p.splits * waves, turns = (nch + parts * AHEAD - 1) / (parts * AHEAD);
  unsigned char* stage = lds + wave * BYTES;
  const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)stage);
  const unsigned short* row = p.x + (int64_t)min(m0 + copy_row(lane), p.M - 1) * p.xs;
  // Of one adapter, or of two with one reading of x (a prompt's end inside a tile would else take its workgroup twice as long as the others).
  auto product = [&](auto two, int ad0, uint64_t own0, int ad1, uint64_t own1) {
    constexpr int N = decltype(two)::value ? 2 : 1;
    const unsigned short* a[2] = {p.a + (size_t)ad0 * K8 * p.rank * 8, p.a + (size_t)ad1 * K8 * p.rank * 8};
    f32x4 acc[N][RT];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int t = 0; t < RT; t++) acc[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    int turn = tile % turns;
    for (int i = 0; i < turns; i++) {
      const int c = (turn * parts + part) * AHEAD;
      turn = turn + 1 == turns ? 0 : turn + 1;
      if (c >= nch) continue;
      u32x4 w[AHEAD][2][N][RT];
#pragma unroll
      for (int u = 0; u < AHEAD; u++)
#pragma unroll
        for (int s = 0; s < 2; s++) {
          const int k8 = 8 * (c + u) + 4 * s;  // behind the end of K the last group, which meets zeros
          copy_to_lds(row + min(k8 + copy_chunk(lane), K8 - 1) * 8, to + (u * 2 + s) * 1024);
#pragma unroll
          for (int n = 0; n < N; n++)
#pragma unroll
            for (int t = 0; t < RT; t++)
              w[u][s][n][t] = *reinterpret_cast<const u32x4*>(a[n] + ((size_t)min(k8 + q, K8 - 1) * p.rank + min(t * 16 + r, p.rank - 1)) * 8);
        }
      __builtin_amdgcn_s_waitcnt(0xf70);  // vmcnt(0)
      asm volatile("" ::: "memory");
#pragma unroll
      for (int u = 0; u < AHEAD; u++)
#pragma unroll
        for (int s = 0; s < 2; s++) {
          u32x4 x = *reinterpret_cast<const u32x4*>(stage + (u * 2 + s) * 1024 + frag_slot(r, q));
          if (8 * (c + u) + 4 * s + q >= K8) x = u32x4{0, 0, 0, 0};
#pragma unroll
          for (int n = 0; n < N; n++)
#pragma unroll
            for (int t = 0; t < RT; t++) acc[n][t] = mma<F16>(w[u][s][n][t], x, acc[n][t]);
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next copies
    }
    float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int n = 0; n < N; n++) {
      const uint64_t own = n ? own1 : own0;
      __syncthreads();
#pragma unroll
      for (int t = 0; t < RT; t++)
        *reinterpret_cast<f32x4*>(sums + wave * (BYTES / 4) + r * PITCH + t * 16 + 4 * q) = acc[n][t];
      __syncthreads();
      for (int e = threadIdx.x; e < 16 * p.rank; e += blockDim.x) {
        const int m = e / p.rank, j = e - m * p.rank;
        if (!(own >> m & 1)) continue;
        float v = 0.f;
#pragma unroll 4
        for (int w = 0; w < waves; w++) v += sums[w * (BYTES / 4) + m * PITCH + j];
        p.h[((size_t)split * p.M + m0 + m) * p.rank + j] = v;
      }
    }
    __syncthreads();
  };
  int first = -1;
  uint64_t first_own = 0;
  for_adapters<16>(p, m0, blockIdx.y, p.share, [&](int ad, uint64_t own) {
    if constexpr (RT == 1) {  // by registers
      if (first < 0) {
        first = ad, first_own = own;
        return;
      }
      product(std::true_type{}, first, first_own, ad, own);
      first = -1;
    } else {
      product(std::false_type{}, ad, own, ad, own);
    }
  });
  if constexpr (RT == 1)
    if (first >= 0) product(std::false_type{}, first, first_own, first, first_own);
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
// lane ends with four neighbouring outputs of rows 4 q .. 4 q + 3. The inner slots are groups of 8: the R8 = rank / 8 of h's first part,
// of its second, and so on; RANK8: the most that R8 may be. All that a wave reads depends on its rows' adapters alone and is asked for
// at once. QUADS: rows of y and out keep four neighbours aligned.
template <bool F16, int PARTS, int RANK8, int MB, int YT, bool GATE, bool QUADS>
__global__ void __launch_bounds__(64 * W) expand_kernel(Params p) {
  constexpr int CH = (PARTS * RANK8 + 3) / 4;  // chunks of 32 slots
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  const int m0 = blockIdx.y * (16 * MB), n0 = (blockIdx.x * W + wave) * 64, R8 = p.rank >> 3, rows = min(16 * MB, p.M - m0);
  if (n0 >= p.N) return;
  const int n = n0 + 4 * r;
  // y of the rows of `own`, and y plus their product -> out
  auto load = [&](uint64_t own, f32x4 (*y)[4]) {
    if constexpr (QUADS)
#pragma unroll
      for (int b = 0; b < MB; b++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (n < p.N && (own >> (b * 16 + 4 * q + i) & 1)) y[b][i] = elem4<YT>(p.y, (size_t)(m0 + b * 16 + 4 * q + i) * p.N + n);
  };
  auto finish = [&](uint64_t own, const f32x4 (*y)[4], const f32x4 (*acc)[4], const float* up) {
    float factor[MB][4];  // of rows 4 q + i
#pragma unroll
    for (int b = 0; b < MB; b++)
#pragma unroll
      for (int i = 0; i < 4; i++) factor[b][i] = acc && F16 ? __shfl(up[b], 4 * q + i) : 1.f;
#pragma unroll
    for (int b = 0; b < MB; b++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int m = b * 16 + 4 * q + i;
        if (n >= p.N || !(own >> m & 1)) continue;
        const size_t at = (size_t)(m0 + m) * p.N + n;
        const float f = factor[b][i];
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
        if (acc) v = f32x4{acc[b][0][i] * f, acc[b][1][i] * f, acc[b][2][i] * f, acc[b][3][i] * f};
        if constexpr (QUADS) {
          v += y[b][i];
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
  };
  // What does not depend on the adapters is asked for before they are known: h, but of large ranks by registers, and y where one workgroup
  // has all of the tile's.
  constexpr bool HELD = CH <= 3;
  const bool together = p.share == 1;
  auto group = [&](int b, int k8, float* v) {  // of a row's h, eight values
    const float* from = p.h + ((size_t)m0 + min(b * 16 + r, rows - 1)) * p.rank + 8 * k8;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = 0.f;
#pragma unroll 2
    for (int s = 0; s < p.splits; s++, from += (size_t)p.M * p.rank) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(from), hi = *reinterpret_cast<const f32x4*>(from + 4);
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] += lo[j], v[4 + j] += hi[j];
    }
  };
  auto slot = [&](int c, int& part) {  // this lane's group of chunk c; behind the last part, group 0
    const int g = 4 * c + q;
    part = g / R8;
    return part < PARTS ? g - part * R8 : 0;
  };
  f32x4 y[MB][4];
  float held[MB][HELD ? CH : 1][8];
  if (together) load(~0ull >> (64 - rows), y);
  if constexpr (HELD)
#pragma unroll
    for (int b = 0; b < MB; b++)
#pragma unroll
      for (int c = 0; c < CH; c++) {
        int part;
        if (4 * c < PARTS * R8) group(b, slot(c, part), held[b][c]);
      }
  const uint64_t bare = for_adapters<16 * MB>(p, m0, blockIdx.z, p.share, [&](int ad, uint64_t own) {
    if (!together) load(own, y);
    const unsigned short* w = p.b + (size_t)ad * R8 * p.N * 8;
    const float scale = p.scale[ad];
    float up[MB], down[MB];  // the power of two that h is divided by, and its inverse
    f32x4 acc[MB][4];        // [t]: rows 4 q + i, output n0 + 4 r + t
#pragma unroll
    for (int b = 0; b < MB; b++) {
      up[b] = down[b] = 1.f;
      if constexpr (F16) {
        // the largest into [2^13, 2^14): the second part is held to 2^-38 of it
        float most = 0.f;
        if constexpr (HELD) {
#pragma unroll
          for (int c = 0; c < CH; c++)
#pragma unroll
            for (int j = 0; j < 8; j++)
              if (4 * c < PARTS * R8) most = fmaxf(most, fabsf(held[b][c][j]));
        } else {
          for (int k8 = q; k8 < R8; k8 += 4) {
            float v[8];
            group(b, k8, v);
#pragma unroll
            for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(v[j]));
          }
        }
        most *= fabsf(scale);
        most = cols_max(most);
        if (most > 0.f && most < INFINITY) {
          const int e = max(-126, min(126, ilogbf(most) - 13));
          up[b] = ldexpf(1.f, e), down[b] = ldexpf(1.f, -e);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; t++) acc[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    constexpr int AHEAD = CH <= 3 ? CH : 1;  // of large ranks one chunk after the other, by registers
#pragma unroll AHEAD
    for (int c = 0; c < CH; c++) {
      if (4 * c >= PARTS * R8) break;
      int part;
      const int k8 = slot(c, part);
      u32x4 bf[4];
#pragma unroll
      for (int t = 0; t < 4; t++)
        bf[t] = *reinterpret_cast<const u32x4*>(w + ((size_t)k8 * p.N + min(n0 + 4 * r + t, p.N - 1)) * 8);
#pragma unroll
      for (int b = 0; b < MB; b++) {
        float v[8];
        if constexpr (!HELD) group(b, k8, v);
        u32x4 hf;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float a0 = HELD ? held[b][HELD ? c : 0][2 * i] : v[2 * i], a1 = HELD ? held[b][HELD ? c : 0][2 * i + 1] : v[2 * i + 1];
          a0 = a0 * scale * down[b], a1 = a1 * scale * down[b];
          unsigned one = F16 ? pack_f16x2(a0, a1) : pack_bf16x2(a0, a1);
#pragma unroll
          for (int u = 1; u <= PARTS; u++)
            if (part >= u) {  // what the part before left
              a0 -= F16 ? h_lo(one) : bf_lo(one), a1 -= F16 ? h_hi(one) : bf_hi(one);
              one = u == PARTS ? 0 : F16 ? pack_f16x2(a0, a1) : pack_bf16x2(a0, a1);
            }
          hf[i] = one;
        }
#pragma unroll
        for (int t = 0; t < 4; t++) acc[b][t] = mma<F16>(hf, bf[t], acc[b][t]);
      }
    }
    finish(own, y, acc, up);
  });
  if (blockIdx.z == 0 && bare && (GATE || p.out != p.y)) {
    if (!together) load(bare, y);
    finish(bare, y, nullptr, nullptr);
  }
}

// Splits of K across workgroups and waves of each. A wave that asks for all of its chunks at once is best for few rows; splits, whose sums
// every workgroup on the way back reads, only for a long K and until there is a workgroup a CU (16 rows, K 2048, gated N 32768, five adapters:
// 13.5 us in one split of eight waves, 14.4 in two of four, 18 in four of four; 1993 rows, K 16384: 44 in one split, 34.8 in two, 37 in four).
struct Cut {
  int splits, waves;
};
Cut cut(int M, int K, int rank) {
  const int rt = rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8, most = shrink_waves(rt), tiles = (M + 15) / 16;
  const int runs = ((K + 63) / 64 + shrink_ahead(rt) - 1) / shrink_ahead(rt);
  Cut c;
  c.splits = std::max(1, std::min({MAX_SPLITS, runs / (2 * most), 256 / std::min(tiles, 256)}));
  c.waves = std::min(most, (runs + c.splits - 1) / c.splits);
  return c;
}

// Workgroups that deal a tile's adapters among them, where all tiles have `workgroups`. Up to 64 rows are tokens of as many requests, or a
// prompt: as many as leave no more than 1024 in all, those without an adapter among them (gated, N 32768, K 2048, rank 32, a bank of 16, us with
// up to 1024 and with one for each: 64 rows of one adapter 12.5 and 31.2, of 16 19.2 and 37.4; 16 rows of one 9.9 and 12.4, of 16 17.3 and 21.0;
// up to 256 takes 8.6 to 19.9 there, and for 5 rows of 5 11.9 instead of 10.8). More may be those or prompts, of whose tiles most name one
// adapter: no more than 256. (N and K 2048, rank 16, rows of
// three neighbours an adapter: 70 rows 18.7 us with one, 8.9 so; 300 30.7 and 17.0; 1000 35.5 and 30.8; prompts of 70, 300 and 1000 rows 8.4, 10.2
// and 13.3 both ways, 8.5, 12.4 and 19.1 with up to 512. Gated, 300 rows to N 32768, 20.5; 50 with more than one there.)
int share_of(const Params& p, int64_t workgroups) {
  return (int)std::min<int64_t>({16, p.M, p.adapters, std::max<int64_t>(1, (p.M <= 64 ? 1024 : 256) / workgroups)});
}

template <bool F16, int RT>
int launch_shrink(Params p, hipStream_t s) {
  p.share = share_of(p, (int64_t)((p.M + 15) / 16) * p.splits);
  const int rc = host::allow_lds(reinterpret_cast<const void*>(&shrink_kernel<F16, RT>), shrink_waves(RT) * shrink_bytes(RT), "fa_lora_add");
  if (rc != FA_OK) return rc;
  hipLaunchKernelGGL((shrink_kernel<F16, RT>), dim3((p.runs ? (p.M + 127) / 128 * 8 : (p.M + 15) / 16) * p.splits, p.share), dim3(64 * p.waves), p.waves * shrink_bytes(RT), s,
                     p);
  return FA_OK;
}

template <bool F16, int PARTS, int RANK8, int YT, bool GATE>
void launch_expand(Params p, bool quads, hipStream_t s) {
  const int blocks = (p.N + 64 * W - 1) / (64 * W);
  p.share = share_of(p, (int64_t)blocks * (p.M > 256 ? (p.M + 31) / 32 : (p.M + 15) / 16));
  if (p.M > 256) {
    const dim3 grid(blocks, (p.M + 31) / 32, p.share);
    if (quads) hipLaunchKernelGGL((expand_kernel<F16, PARTS, RANK8, 2, YT, GATE, true>), grid, dim3(64 * W), 0, s, p);
    else hipLaunchKernelGGL((expand_kernel<F16, PARTS, RANK8, 2, YT, GATE, false>), grid, dim3(64 * W), 0, s, p);
  } else {
    const dim3 grid(blocks, (p.M + 15) / 16, p.share);
    if (quads) hipLaunchKernelGGL((expand_kernel<F16, PARTS, RANK8, 1, YT, GATE, true>), grid, dim3(64 * W), 0, s, p);
    else hipLaunchKernelGGL((expand_kernel<F16, PARTS, RANK8, 1, YT, GATE, false>), grid, dim3(64 * W), 0, s, p);
  }
}

template <bool F16, int RANK8>
void launch_expand(Params p, int yt, bool gate, bool quads, hipStream_t s) {
  constexpr int XT = F16 ? FA_DTYPE_F16 : FA_DTYPE_BF16;
  if (yt == FA_DTYPE_F32) {
    if (gate) launch_expand<F16, 2, RANK8, FA_DTYPE_F32, true>(p, quads, s);
    else launch_expand<F16, F16 ? 2 : 3, RANK8, FA_DTYPE_F32, false>(p, quads, s);
  } else {
    if (gate) launch_expand<F16, 2, RANK8, XT, true>(p, quads, s);
    else launch_expand<F16, 2, RANK8, XT, false>(p, quads, s);
  }
}

template <bool F16, int RANK8>
int launch(const Params& p, int yt, bool gate, bool quads, hipStream_t s) {
  const int rc = launch_shrink<F16, RANK8 / 2>(p, s);
  if (rc == FA_OK) launch_expand<F16, RANK8>(p, yt, gate, quads, s);
  return rc;
}
template <bool F16>
int launch(const Params& p, int yt, bool gate, bool quads, hipStream_t s) {
  if (p.rank <= 16) return launch<F16, 2>(p, yt, gate, quads, s);
  if (p.rank <= 32) return launch<F16, 4>(p, yt, gate, quads, s);
  if (p.rank <= 64) return launch<F16, 8>(p, yt, gate, quads, s);
  return launch<F16, 16>(p, yt, gate, quads, s);
}

}  // namespace lora
}  // namespace fa

extern "C" size_t fa_lora_workspace_bytes(int rows, int k, int rank) {
  if (rows < 1 || k < 8 || rank < 8 || rank > fa::lora::MAX_RANK || k > (1 << 24)) return 0;
  return (size_t)fa::lora::cut(rows, k, rank).splits * rows * rank * sizeof(float);
}

extern "C" int fa_lora_add(const fa_lora_args* a, fa_stream_t stream) {
  using namespace fa;
  const char* who = "fa_lora_add";
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->dtype != FA_DTYPE_BF16 && a->dtype != FA_DTYPE_F16)
    return host::fail(FA_ERR_INVALID_ARG, "%s: dtype %d: x and the adapters are bf16 or fp16", who, a->dtype);
  if (a->y_dtype != FA_DTYPE_F32 && a->y_dtype != a->dtype)
    return host::fail(FA_ERR_INVALID_ARG, "%s: y_dtype %d: y is fp32 or of x's type", who, a->y_dtype);
  if (a->rows < 0 || a->rows > (1 << 20)) return host::fail(FA_ERR_INVALID_ARG, "%s: rows=%d outside [0, 2^20]", who, a->rows);
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
  const lora::Cut cut = lora::cut(a->rows, a->k, a->rank);
  lora::Params p{static_cast<const unsigned short*>(a->x), a->x_stride, static_cast<const unsigned short*>(a->a),
                 static_cast<const unsigned short*>(a->b), a->scale, a->index, a->y, a->out, static_cast<float*>(a->workspace),
                 a->rows, a->n, a->k, a->rank, a->adapters, cut.splits, cut.waves, (a->rows + 15) / 16 >= 64, 1};
  const bool quads = a->n % 4 == 0 && reinterpret_cast<uintptr_t>(a->y) % (4 * yb) == 0 &&
                     reinterpret_cast<uintptr_t>(a->out) % (a->gate ? 4 : 4 * ob) == 0;
  rc = a->dtype == FA_DTYPE_F16 ? lora::launch<true>(p, a->y_dtype, a->gate, quads, (hipStream_t)stream)
                                : lora::launch<false>(p, a->y_dtype, a->gate, quads, (hipStream_t)stream);
  if (rc != FA_OK) return rc;
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return host::fail(FA_ERR_LAUNCH, "%s: %s", who, hipGetErrorString(e));
  return FA_OK;
}
