// Products of a few rows of activations with 4-bit weights (fa_w4_linear): y = x W^T, 1 to 64 rows.
//
//   W[n][k] = e2m1(code[n][k]) * scale[n][k / group],  y[m][n] = sum_k x[m][k] W[n][k]
//   then  y += bias[n];  gate: y'[m][f] = gelu_tanh(y[m][2f]) y[m][2f + 1];  y += residual[m][n].
//
// Per output the sum over one group is taken on the MFMA from exact operands (a code is exact in bf16 and
// fp16), and the group's scale multiplies that fp32 sum: nothing is rounded below 32 bits before the store.
//
// Layout (laid out once, w4.pack): tiles of 16 weight rows x 128 columns, 1 KB each, whose 16 bytes at
// [q][r] are the A operands of four MFMAs 16x16x32 for lane r + 16 q: byte j holds columns 32 (j / 4) + 8 q +
// 2 (j % 4) and the next (lower nibble first). One wave load of 16 bytes a lane is one tile, contiguous. The
// groups' scales are [tile][group][16 rows].
//
// A workgroup owns NT tiles of 16 rows and its waves split K into contiguous ranges; their fp32 sums are added
// in LDS in wave order, so results do not depend on timing. Work per weight byte is small (the bound is
// HBM): per 1 KB tile a wave converts 32 codes a lane (v_cvt_scalef32_pk_*_fp4, two a time) and issues four
// MFMAs. The activations of a run of chunks go through LDS, private to the wave: lanes in MFMA order would
// fetch 16 bytes each from 16 rows, which the address unit takes lane by lane.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"

namespace fa {
namespace w4 {

struct Params {
  const unsigned short* x;
  int64_t xs;  // row stride of x, elements
  const unsigned char* codes;
  const unsigned short* scales;
  const float* bias;
  const float* residual;
  void* out;
  float* part;  // [workgroup's tiles][split][pair of outputs][2] where K is split across workgroups
  uint64_t *arrived, nonce;  // [workgroup's tiles][WORDS]: a word a split, and the claim
  int M, N, K, nch, out_dtype, gate;
};

template <bool F16>
__device__ __forceinline__ u32x4 dequant8(unsigned c) {  // eight codes, lower nibble first -> eight bf16 / fp16
  if constexpr (F16) {
    return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 0)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 1)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 2)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 3))};
  } else {
    return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 0)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 1)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 2)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 3))};
  }
}

// value of lane g of the own row of 16 lanes (DPP row_newbcast); g is a constant once the loops are unrolled
template <int G = 0>
__device__ __forceinline__ u32x2 row_bcast(u32x2 v, int g) {
  if (g == G)
    return u32x2{(unsigned)__builtin_amdgcn_update_dpp(0, (int)v[0], 0x150 + G, 0xF, 0xF, false),
                 (unsigned)__builtin_amdgcn_update_dpp(0, (int)v[1], 0x150 + G, 0xF, 0xF, false)};
  if constexpr (G < 15) return row_bcast<G + 1>(v, g);
  return v;
}

__device__ __forceinline__ void store_out(const Params& p, size_t at, float v) {
  if (p.out_dtype == FA_DTYPE_F32) static_cast<float*>(p.out)[at] = v;
  else if (p.out_dtype == FA_DTYPE_F16) static_cast<_Float16*>(p.out)[at] = (_Float16)v;
  else static_cast<unsigned short*>(p.out)[at] = bf16_bits(v);
}

// What follows the product, for weight rows n and n + 1 (n even) of row m of x.
__device__ __forceinline__ void finish(const Params& p, int m, int n, float y0, float y1) {
  const bool two = n + 1 < p.N;
  if (p.bias) {
    y0 += p.bias[n];
    if (two) y1 += p.bias[n + 1];
  }
  if (p.gate) {
    const size_t at = (size_t)m * (p.N >> 1) + (n >> 1);
    float y = gelu_tanh(y0) * y1;
    if (p.residual) y += p.residual[at];
    store_out(p, at, y);
  } else {
    const size_t at = (size_t)m * p.N + n;
    if (p.residual) {
      y0 += p.residual[at];
      if (two) y1 += p.residual[at + 1];
    }
    store_out(p, at, y0);
    if (two) store_out(p, at + 1, y1);
  }
}

constexpr int MAX_SPLITS = 16, WORDS = MAX_SPLITS + 1;
constexpr int max_waves(int MR, int NT) { return MR <= 16 && NT == 1 ? 16 : 8; }  // of a workgroup at most, by registers and LDS

// MR: rows of x the LDS stage holds (1, 4, 16, 32 or 64); XC: chunks a stage; NT: weight tiles a workgroup; RUN:
// chunks whose codes are in flight while the run before is used.
template <int GROUP, int MR, int XC, int NT, int RUN>
struct Shape {
  static constexpr int MB = (MR + 15) / 16;           // column blocks of 16 rows of x
  static constexpr int GC = 128 / GROUP;              // groups a chunk
  static constexpr int XROW = XC * 256 + 16;          // LDS bytes of a row: the pad spreads 16 rows over the banks
  static constexpr int STAGE = MR * XROW, SUMS = MB * NT * 1024;
  static constexpr int XBYTES = STAGE > SUMS ? STAGE : SUMS;  // of a wave: its stage, later its sums
  static_assert(max_waves(MR, NT) * XBYTES <= 160 * 1024, "LDS");
  static_assert(RUN % XC == 0 && RUN * GC <= 16, "a run is whole stages, its scales one row of lanes");
};

// SPLIT: K is split across workgroups (blockIdx.y). A kernel of its own: with the join behind it, the unsplit one of four tiles a
// workgroup, whose loop has all registers, ran 32768 x 2048 in 11.4 us instead of 9.6.
template <bool F16, int GROUP, int MR, int XC, int NT, int RUN, bool SPLIT>
__global__ void __launch_bounds__(64 * max_waves(MR, NT)) w4_kernel(Params p) {
  using S = Shape<GROUP, MR, XC, NT, RUN>;
  constexpr int MB = S::MB, GC = S::GC;
  extern __shared__ unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int ntile = (p.N + 15) >> 4;
  const int t0 = blockIdx.x * NT;
  unsigned char* xl = lds + wave * S::XBYTES;
  const int part = SPLIT ? blockIdx.y * W + wave : wave, parts = SPLIT ? gridDim.y * W : W;  // of K: contiguous ranges of chunks
  const int cb = (int)((int64_t)p.nch * part / parts), ce = (int)((int64_t)p.nch * (part + 1) / parts);

  f32x4 acc[NT][MB];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int b = 0; b < MB; b++) acc[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};

  u32x4 code[NT][RUN], cnext[NT][RUN];
  u32x2 sc[NT], snext[NT];
  // codes of chunks [c, c + RUN) and their scales: lane (r, q) loads the four rows 4q .. 4q + 3 of group r of
  // the run (RUN * GC <= 16 groups), which row_bcast hands to its row of lanes
  auto fetch = [&](int c) {
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const size_t tile = min(t0 + t, ntile - 1);  // a tile behind the last one repeats it and is not stored
#pragma unroll
      for (int j = 0; j < RUN; j++)
        if (c + j < ce) cnext[t][j] = ld_stream128(p.codes + (tile * p.nch + c + j) * 1024 + lane * 16);
      if (c < ce)
        snext[t] = *reinterpret_cast<const u32x2*>(p.scales + ((tile * p.nch + c) * GC + min(r, (ce - c) * GC - 1)) * 16 +
                                                   4 * q);
    }
  };
  // a stage's activations: pieces of 16 bytes, the XC * 16 pieces of a row in neighbouring lanes
  constexpr int PR = XC * 16, PIECES = (MR * PR + 63) / 64;
  u32x4 xv[PIECES];
  auto load_x = [&](int c) {
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
      const int pc = i * 64 + lane, row = pc / PR, k = c * 128 + (pc % PR) * 8;
      xv[i] = u32x4{0, 0, 0, 0};
      if (row < p.M && k < p.K) xv[i] = *reinterpret_cast<const u32x4*>(p.x + row * p.xs + k);
    }
  };
  load_x(cb);
  fetch(cb);
  for (int c = cb; c < ce; c += RUN) {
#pragma unroll
    for (int t = 0; t < NT; t++) {
      sc[t] = snext[t];
#pragma unroll
      for (int j = 0; j < RUN; j++) code[t][j] = cnext[t][j];
    }
    if (c + RUN < ce) fetch(c + RUN);
#pragma unroll
    for (int j0 = 0; j0 < RUN; j0 += XC) {
      if (c + j0 < ce) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
          const int pc = i * 64 + lane, row = pc / PR;
          if (MR * PR % 64 == 0 || row < MR) *reinterpret_cast<u32x4*>(xl + row * S::XROW + (pc % PR) * 16) = xv[i];
        }
        if (c + j0 + XC < ce) load_x(c + j0 + XC);
        wave_fence();
#pragma unroll
        for (int jj = 0; jj < XC; jj++) {
          const int j = j0 + jj;
          if (c + j < ce) {
            u32x4 b[MB][4];
#pragma unroll
            for (int m = 0; m < MB; m++)
#pragma unroll
              for (int i = 0; i < 4; i++)
                b[m][i] = *reinterpret_cast<const u32x4*>(xl + (MR < 16 ? min(r, MR - 1) : m * 16 + r) * S::XROW +
                                                          jj * 256 + i * 64 + q * 16);
#pragma unroll
            for (int t = 0; t < NT; t++) {
              f32x4 part[MB];
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const u32x4 a = dequant8<F16>(code[t][j][i]);
                const bool first = (i * 32) % GROUP == 0;
#pragma unroll
                for (int m = 0; m < MB; m++) {
                  const f32x4 from = first ? f32x4{0.f, 0.f, 0.f, 0.f} : part[m];
                  part[m] = F16 ? mfma16h(a, b[m][i], from) : mfma16(a, b[m][i], from);
                }
                if ((i * 32 + 32) % GROUP == 0) {
                  const u32x2 s = row_bcast(sc[t], j * GC + i * 32 / GROUP);
#pragma unroll
                  for (int m = 0; m < MB; m++) {
                    acc[t][m][0] += bf_lo(s[0]) * part[m][0];
                    acc[t][m][1] += bf_hi(s[0]) * part[m][1];
                    acc[t][m][2] += bf_lo(s[1]) * part[m][2];
                    acc[t][m][3] += bf_hi(s[1]) * part[m][3];
                  }
                }
              }
            }
          }
        }
        wave_fence();
      }
    }
  }

  // sums of the waves, in wave order: [wave][tile][block][lane] 16 bytes over the stages
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int b = 0; b < MB; b++)
      *reinterpret_cast<f32x4*>(lds + (((wave * NT + t) * MB + b) * 64 + lane) * 16) = acc[t][b];
  __syncthreads();
  // one thread per output pair (rows 2f, 2f + 1 of the tile) and row of x
  constexpr int PAIRS = NT * MB * 128;
  auto pairs = [&](auto&& each) {
    for (int e = threadIdx.x; e < PAIRS; e += blockDim.x) {
      const int tb = e >> 7, pr = e & 7, col = (e >> 3) & 15;  // tile and block, pair, row of x within the block
      const int m = (tb % MB) * 16 + col, n = (t0 + tb / MB) * 16 + 2 * pr;
      if (m < p.M && n < p.N) each(e, tb, pr, col, m, n);
    }
  };
  auto sum = [&](int tb, int pr, int col) {
    const float* s = reinterpret_cast<const float*>(lds) + (tb * 64 + (pr >> 1) * 16 + col) * 4 + (pr & 1) * 2;
    f32x2 y = f32x2{0.f, 0.f};
    for (int w = 0; w < W; w++) {
      y[0] += s[w * NT * MB * 256];
      y[1] += s[w * NT * MB * 256 + 1];
    }
    return y;
  };
  if constexpr (!SPLIT) {
    pairs([&](int, int tb, int pr, int col, int m, int n) {
      const f32x2 y = sum(tb, pr, col);
      finish(p, m, n, y[0], y[1]);
    });
  } else {
    // The last of the splits' workgroups adds them in their order and finishes: once, as the result may lie over the residual.
    uint64_t* words = p.arrived + (size_t)blockIdx.x * WORDS;
    if (blockIdx.y == 0 && threadIdx.x == 0)
      __hip_atomic_store(words + MAX_SPLITS, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const rsrc_t sums = make_rsrc(p.part + (size_t)blockIdx.x * gridDim.y * PAIRS * 2, 0xffffffffu);
    pairs([&](int e, int tb, int pr, int col, int, int) {
      stb64<kCpSc1>(sums, (blockIdx.y * PAIRS + e) * 8, __builtin_bit_cast(u32x2, sum(tb, pr, col)));
    });
    if (!arrived_last(words, p.nonce, blockIdx.y, gridDim.y, reinterpret_cast<int*>(lds), words + MAX_SPLITS)) return;
    pairs([&](int e, int, int, int, int m, int n) {
      float y0 = 0.f, y1 = 0.f;
#pragma unroll 8
      for (unsigned s = 0; s < gridDim.y; s++) {
        const f32x2 v = __builtin_bit_cast(f32x2, ldb64<kCpSc1>(sums, (s * PAIRS + e) * 8));
        y0 += v[0];
        y1 += v[1];
      }
      finish(p, m, n, y0, y1);
    });
  }
}

// How a product is cut: tiles a workgroup, splits of K across workgroups, waves a workgroup. Times in us of both sides, in
// turn, group 32, at N x K and rows M.
struct Cut {
  int nt, splits, waves;
};
Cut cut(int M, int N, int K) {
  const int tiles = (N + 15) / 16, nch = (K + 127) / 128;
  Cut c{1, 1, 1};
  // Four tiles a workgroup share its activations and keep four tiles' codes in flight. Tiles x chunks of 128 columns: us with
  // one tile, with four. 5 to 16 rows: from 1024 tiles on (2048 x 16: 13.2, 10.4 at 5 rows and 14.7, 11.3 at 16; at worst 1250 x 32: 15.0,
  // 17.1), and from 32 tiles of 112 chunks on, where K is split (32 x 112: 10.0, 9.4 and 12.0, 10.0; 128 x 128: 11.9, 9.8 and 13.3, 10.4;
  // 300 x 128: 23.1, 15.1; below it 16 x 112: 8.9, 9.3; 32 x 104: 9.8, 10.3) but for 201 to 256 tiles of fewer than 160 chunks, whose workgroups
  // are one too many for a CU each (200 x 128: 12.4, 12.4; 208 x 128: 12.5, 13.6; 208 x 160: 14.8, 14.7). 1 to 4 rows: only from 2048
  // tiles of up to 8 chunks on, whose waves have next to nothing to do (4096 x 8, 1 row: 11.2, 10.4; 1500 x 8: 6.3, 6.8;
  // 3125 x 16: 13.6, 21.1). More than 16 rows leave registers and LDS for two tiles, more than 32 for one.
  if (M > 32) c.nt = 1;
  else if (M > 16) c.nt = 2;
  else if (M > 4) c.nt = tiles >= 1024 || (tiles >= 32 && nch >= 112 && (tiles <= 200 || tiles > 256 || nch >= 160)) ? 4 : 1;
  else c.nt = tiles >= 2048 && nch <= 8 ? 4 : 1;
  const int blocks = (tiles + c.nt - 1) / c.nt, most = M <= 16 && c.nt == 1 ? 16 : 8;
  // Splits cost the join of the last workgroup, about 2 us. With one tile and few rows 16 waves share K already, and only a handful of
  // workgroups needs more (64 x 16384: 5.4 instead of 7.7, but 2048 x 8192 in two 7.0 instead of 5.9); else K is split until there is a
  // workgroup a CU (2048 x 16384: 9.4 instead of 24.2 at M = 5, 14.2 instead of 24.1 at 32, 20.8 instead of 28.8 at 48), in
  // parts of 2048 columns or more (2048 x 2048 in two at M = 32: 8.2 instead of 6.2).
  c.splits = std::max(1, std::min({(most == 16 ? 32 : 256) / blocks, nch / 16, MAX_SPLITS}));
  const int mine = (nch + c.splits - 1) / c.splits;
  // Waves: 4096 in all, with two tiles 2048 (16384 x 2048 at M = 32: 10.9 instead of 12.7), of two chunks each or more
  // (2560 x 2048: 4.2 instead of 4.5 at M = 5, 3.7 instead of 3.9 at 1), and no fewer than four (32768 x 2048 with four
  // instead of eight: 11.6 instead of 10.6).
  c.waves = std::max(1, std::min({most, std::max(4, (c.nt == 2 ? 2048 : 4096) / (blocks * c.splits)), mine, std::max(4, mine / 2)}));
  return c;
}

template <bool F16, int GROUP, int MR, int XC, int NT, int RUN, bool SPLIT = false>
int launch_shape(const Params& p, const Cut& c, hipStream_t stream) {
  if constexpr (!SPLIT && !(MR <= 4 && NT == 4))  // these have workgroups enough
    if (c.splits > 1) return launch_shape<F16, GROUP, MR, XC, NT, RUN, true>(p, c, stream);
  using S = Shape<GROUP, MR, XC, NT, RUN>;
  const int blocks = ((p.N + 15) / 16 + NT - 1) / NT;
  const unsigned lds = (unsigned)(c.waves * S::XBYTES);
  const void* k = reinterpret_cast<const void*>(&w4_kernel<F16, GROUP, MR, XC, NT, RUN, SPLIT>);
  int rc = host::allow_lds(k, max_waves(MR, NT) * S::XBYTES, "fa_w4_linear");
  if (rc != FA_OK) return rc;
  hipLaunchKernelGGL((w4_kernel<F16, GROUP, MR, XC, NT, RUN, SPLIT>), dim3(blocks, c.splits), dim3(64 * c.waves), lds, stream,
                     p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return host::fail(FA_ERR_LAUNCH, "fa_w4_linear: %s", hipGetErrorString(e));
  return FA_OK;
}

template <bool F16, int GROUP>
int launch_rows(const Params& p, const Cut& c, hipStream_t s) {
  if (p.M == 1)
    return c.nt == 4 ? launch_shape<F16, GROUP, 1, 1, 4, 1>(p, c, s) : launch_shape<F16, GROUP, 1, 4, 1, 4>(p, c, s);
  if (p.M <= 4)
    return c.nt == 4 ? launch_shape<F16, GROUP, 4, 1, 4, 1>(p, c, s) : launch_shape<F16, GROUP, 4, 4, 1, 4>(p, c, s);
  if (p.M <= 16)
    return c.nt == 4 ? launch_shape<F16, GROUP, 16, 1, 4, 1>(p, c, s) : launch_shape<F16, GROUP, 16, 2, 1, 4>(p, c, s);
  if (p.M <= 32) return launch_shape<F16, GROUP, 32, 1, 2, 2>(p, c, s);
  return launch_shape<F16, GROUP, 64, 1, 1, 2>(p, c, s);
}

template <bool F16>
int launch_group(const Params& p, const Cut& c, int group, hipStream_t s) {
  if (group == 32) return launch_rows<F16, 32>(p, c, s);
  if (group == 64) return launch_rows<F16, 64>(p, c, s);
  return launch_rows<F16, 128>(p, c, s);
}

size_t blocks_of(const Cut& c, int N) { return ((N + 15) / 16 + c.nt - 1) / c.nt; }
size_t arrived_bytes(const Cut& c, int N) { return (blocks_of(c, N) * WORDS * sizeof(uint64_t) + 255) / 256 * 256; }
size_t part_bytes(const Cut& c, int M, int N) {
  if (c.splits == 1) return 0;
  const int rows = M <= 16 ? 16 : M <= 32 ? 32 : 64;
  return arrived_bytes(c, N) + blocks_of(c, N) * c.splits * c.nt * rows * 16 * sizeof(float);
}

}  // namespace w4
}  // namespace fa

extern "C" int fa_w4_linear(const fa_w4_args* a, fa_stream_t stream) {
  using namespace fa;
  const char* who = "fa_w4_linear";
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->dtype != FA_DTYPE_BF16 && a->dtype != FA_DTYPE_F16)
    return host::fail(FA_ERR_INVALID_ARG, "%s: dtype %d: x is bf16 or fp16", who, a->dtype);
  if (a->out_dtype != FA_DTYPE_BF16 && a->out_dtype != FA_DTYPE_F16 && a->out_dtype != FA_DTYPE_F32)
    return host::fail(FA_ERR_INVALID_ARG, "%s: out_dtype %d", who, a->out_dtype);
  if (a->rows < 0 || a->rows > FA_W4_MAX_ROWS)
    return host::fail(FA_ERR_INVALID_ARG, "%s: rows=%d outside [0, %d]", who, a->rows, FA_W4_MAX_ROWS);
  if (a->n < 1 || a->k < 1 || a->k % 8 || a->n > (1 << 24) || a->k > (1 << 24))
    return host::fail(FA_ERR_INVALID_ARG, "%s: need 1 <= n, k <= 2^24 and k a multiple of 8, got n=%d k=%d", who, a->n,
                      a->k);
  if (a->group != 32 && a->group != 64 && a->group != 128)
    return host::fail(FA_ERR_INVALID_ARG, "%s: group=%d is none of 32, 64, 128", who, a->group);
  if (a->gate && a->n % 2) return host::fail(FA_ERR_INVALID_ARG, "%s: the gated form needs an even n, got %d", who, a->n);
  if (a->rows == 0) return FA_OK;
  const struct {
    const void* p;
    const char* name;
    unsigned align;
    bool need;
  } ptrs[] = {{a->x, "x", 16, true},       {a->codes, "codes", 16, true},         {a->scales, "scales", 8, true},
              {a->out, "out", 4, true},    {a->bias, "bias", 4, false},           {a->residual, "residual", 4, false}};
  for (const auto& t : ptrs) {
    if (t.need && !t.p) return host::fail(FA_ERR_INVALID_ARG, "%s: %s is NULL", who, t.name);
    const unsigned align = t.p == a->out && a->out_dtype != FA_DTYPE_F32 ? 2 : t.align;
    if (reinterpret_cast<uintptr_t>(t.p) % align)
      return host::fail(FA_ERR_INVALID_ARG, "%s: %s is not %u-byte aligned", who, t.name, align);
  }
  if (a->rows > 1 && (a->x_stride < a->k || a->x_stride % 8))
    return host::fail(FA_ERR_INVALID_ARG, "%s: x_stride=%lld must be a multiple of 8 and >= k=%d", who,
                      (long long)a->x_stride, a->k);
  const w4::Cut c = w4::cut(a->rows, a->n, a->k);
  const size_t need = w4::part_bytes(c, a->rows, a->n);
  if (need && (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return host::fail(FA_ERR_INVALID_ARG, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, need,
                      a->workspace ? a->workspace_bytes : (size_t)0);
  int rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  w4::Params p{static_cast<const unsigned short*>(a->x),
               a->x_stride,
               static_cast<const unsigned char*>(a->codes),
               static_cast<const unsigned short*>(a->scales),
               a->bias,
               a->residual,
               a->out,
               need ? reinterpret_cast<float*>(static_cast<unsigned char*>(a->workspace) + w4::arrived_bytes(c, a->n)) : nullptr,
               static_cast<uint64_t*>(a->workspace),
               need ? host::launch_nonce() : 0,
               a->rows,
               a->n,
               a->k,
               (a->k + 127) / 128,
               a->out_dtype,
               a->gate};
  return a->dtype == FA_DTYPE_F16 ? w4::launch_group<true>(p, c, a->group, (hipStream_t)stream)
                                  : w4::launch_group<false>(p, c, a->group, (hipStream_t)stream);
}

extern "C" size_t fa_w4_workspace_bytes(int rows, int n, int k) {
  if (rows < 1 || rows > FA_W4_MAX_ROWS || n < 1 || k < 1 || n > (1 << 24) || k > (1 << 24)) return 0;
  return fa::w4::part_bytes(fa::w4::cut(rows, n, k), rows, n);
}
