// The 8-bit K/V cache: rows of keys and values into e4m3 codes with one power of two for each block of 32 tokens
// and head (fa_kv8_store), codes back to rows (fa_kv8_load), and attention over it (fa_kv8_attention).
//
// Layout, contiguous, per sample and K/V head: k[block][hd / 16][32 tokens][16 dims] and v[block][hd][32 tokens]
// bytes, ks / vs[block] fp32. They are the operand orders of the attention below: a wave's 16-byte loads of keys
// are runs of whole lines, and a lane finds the eight keys of a value's MFMA operand side by side.
//
// scale = the smallest power of two s with max|x| <= 448 s, code = x / s rounded to nearest even. A power of two costs
// a floating code no precision (only its range moves), and makes every step exact but that one rounding: x / s, the
// recoding of earlier rows when a later row needs a larger s (exact unless a code turns subnormal), and code * s.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/flashact_mi355x.h"
#include "fa_device.h"
#include "fa_host.h"

namespace fa {
namespace kv8 {

constexpr int BT = 32;  // tokens of a block

// ---------------------------------------------------------------- rows <-> codes
struct Rows {
  unsigned char* p;
  int64_t sb, st, sh, sd;  // strides of sample, token, head, dim in elements
};

struct CacheArgs {
  unsigned char *k, *v;
  float *ks, *vs;
  Rows kr, vr;
  const int *start, *count;  // store: [B], count may be NULL; load: count = rows held per sample
  int B, T, H, hd, nblk, zero;
};

template <int DT>
__device__ __forceinline__ float elem(const unsigned char* p, int64_t i) {
  if constexpr (DT == FA_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (DT == FA_DTYPE_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
  else return as_f32((unsigned)reinterpret_cast<const unsigned short*>(p)[i] << 16);
}
template <int DT>
__device__ __forceinline__ void put(unsigned char* p, int64_t i, float v) {
  if constexpr (DT == FA_DTYPE_F32) reinterpret_cast<float*>(p)[i] = v;
  else if constexpr (DT == FA_DTYPE_F16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
  else reinterpret_cast<unsigned short*>(p)[i] = bf16_bits(v);
}

// Eight neighbouring dims of a row; VEC: contiguous and 16-byte aligned.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const Rows& r, int64_t at, float (&x)[8]) {
  if constexpr (VEC && DT == FA_DTYPE_F32) {
    const f32x4* q = reinterpret_cast<const f32x4*>(r.p + at * 4);
    const f32x4 a = q[0], b = q[1];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = a[i], x[4 + i] = b[i];
  } else if constexpr (VEC) {
    const u32x4 a = *reinterpret_cast<const u32x4*>(r.p + at * 2);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = DT == FA_DTYPE_F16 ? h_lo(a[i]) : bf_lo(a[i]);
      x[2 * i + 1] = DT == FA_DTYPE_F16 ? h_hi(a[i]) : bf_hi(a[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = elem<DT>(r.p, at + i * r.sd);
  }
}
template <int DT, bool VEC>
__device__ __forceinline__ void store8(const Rows& r, int64_t at, const float (&x)[8]) {
  if constexpr (VEC && DT == FA_DTYPE_F32) {
    f32x4* q = reinterpret_cast<f32x4*>(r.p + at * 4);
    q[0] = f32x4{x[0], x[1], x[2], x[3]};
    q[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else if constexpr (VEC) {
    u32x4 a;
#pragma unroll
    for (int i = 0; i < 4; i++)
      a[i] = DT == FA_DTYPE_F16 ? pack_f16x2(x[2 * i], x[2 * i + 1]) : pack_bf16x2(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<u32x4*>(r.p + at * 2) = a;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) put<DT>(r.p, at + i * r.sd, x[i]);
  }
}

// 2^e for the smallest e with amax <= 448 * 2^e, within [2^-100, 2^120]: 448 = 1.75 * 2^8, so e is the exponent less 8,
// one more if the mantissa passes 1.75.
__device__ __forceinline__ float scale_for(float amax) {
  const unsigned u = as_u32(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = amax > 0.f ? max(-100, min(120, e)) : -100;
  return as_f32((unsigned)(e + 127) << 23);
}

// Four values, already divided by the scale -> four codes, rounded to nearest even. What is not finite becomes a NaN
// code (e4m3 has no infinity, and the instruction does not saturate).
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
__device__ __forceinline__ void values4(unsigned c, float (&x)[4]) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
}
__device__ __forceinline__ unsigned recode4(unsigned c, float ratio) {
  float x[4];
  values4(c, x);
  return codes4(x[0] * ratio, x[1] * ratio, x[2] * ratio, x[3] * ratio);
}

// LDS slot of the word that holds tokens 4 rg .. 4 rg + 3 of dim d of a value block: lanes that hold neighbouring
// groups of eight dims would all meet in one bank.
__device__ __forceinline__ int vslot(int d, int rg) { return d * 8 + (rg ^ ((d >> 3) & 7)); }

// One workgroup: one block of one (sample, head), of the keys or of the values. Thread (c8, rg) = dims 8 c8 .. + 7 of tokens
// 4 rg .. 4 rg + 3. Rows of the block that came before `start` keep their values; if the new rows need a larger
// scale they are recoded. Rows behind the new ones keep their codes.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) store_kernel(CacheArgs a) {
  __shared__ unsigned words[256 * 8];
  __shared__ float wmax[4];
  const int per = (a.T + 30) / BT + 1;  // blocks that T rows can touch
  int i = blockIdx.x;
  const int w = i % per;
  i /= per;
  const bool val = i & 1;
  i >>= 1;
  const int h = i % a.H, b = i / a.H;
  const int start = a.start[b];
  const int64_t room = (int64_t)a.nblk * BT - start;
  int n = a.count ? min(a.count[b], a.T) : a.T;
  n = start < 0 || room <= 0 ? 0 : (int)min((int64_t)n, room);
  const int blk = start / BT + w;
  const int lo = max(start - blk * BT, 0), hi = min(start + n - blk * BT, BT);  // the block's new tokens
  if (n <= 0 || lo >= hi) return;

  const Rows& r = val ? a.vr : a.kr;
  const size_t unit = ((size_t)b * a.H + h) * a.nblk + blk;
  unsigned char* code = (val ? a.v : a.k) + unit * BT * a.hd;
  float* scale = (val ? a.vs : a.ks) + unit;
  const int c8 = threadIdx.x % (a.hd / 8), rg = threadIdx.x / (a.hd / 8);
  const bool mine = rg < 8;
  const float old = lo > 0 ? *scale : 0.f;

  // what the block holds and keeps is asked for together with the new rows: two words a token of keys, one a dim of values
  unsigned held[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (mine && val && (4 * rg < lo || 4 * rg + 4 > hi)) {
#pragma unroll
    for (int d = 0; d < 8; d++) held[d] = *reinterpret_cast<const unsigned*>(code + (8 * c8 + d) * BT + 4 * rg);
  } else if (mine && !val) {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (4 * rg + j < lo) {
        const u32x2 c = *reinterpret_cast<const u32x2*>(code + ((c8 >> 1) * BT + 4 * rg + j) * 16 + (c8 & 1) * 8);
        held[2 * j] = c[0], held[2 * j + 1] = c[1];
      }
  }
  float x[4][8], amax = 0.f;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int row = 4 * rg + j;
#pragma unroll
    for (int d = 0; d < 8; d++) x[j][d] = 0.f;
    if (mine && row >= lo && row < hi)
      load8<DT, VEC>(r, b * r.sb + (int64_t)(blk * BT + row - start) * r.st + h * r.sh + 8 * c8 * r.sd, x[j]);
#pragma unroll
    for (int d = 0; d < 8; d++) {
      const float m = fabsf(x[j][d]);
      amax = m <= 3.4028234663852886e38f ? fmaxf(amax, m) : amax;  // neither infinities nor NaN set a scale
    }
  }
  amax = wave_max(amax);
  if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
  const float to = lo > 0 ? fmaxf(scale_for(amax), old) : scale_for(amax);
  const float inv = 1.f / to, ratio = old * inv;  // powers of two: exact
  if (threadIdx.x == 0) *scale = to;

  if (!val) {
    if (!mine) return;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int row = 4 * rg + j;
      u32x2* p = reinterpret_cast<u32x2*>(code + ((c8 >> 1) * BT + row) * 16 + (c8 & 1) * 8);
      if (row >= lo && row < hi) {
        const float(&y)[8] = x[j];
        *p = u32x2{codes4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv),
                   codes4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv)};
      } else if (row < lo && to != old) {
        *p = u32x2{recode4(held[2 * j], ratio), recode4(held[2 * j + 1], ratio)};
      }
    }
    return;
  }
  if (mine) {
#pragma unroll
    for (int d = 0; d < 8; d++) {
      unsigned c = codes4(x[0][d] * inv, x[1][d] * inv, x[2][d] * inv, x[3][d] * inv);
      if (4 * rg < lo || 4 * rg + 4 > hi) {  // tokens of the word that are not new
        const unsigned was = held[d], again = to != old ? recode4(was, ratio) : was;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const unsigned m = 0xffu << (8 * j);
          if (4 * rg + j < lo) c = (c & ~m) | (again & m);
          else if (4 * rg + j >= hi) c = (c & ~m) | (was & m);
        }
      }
      words[vslot(8 * c8 + d, rg)] = c;
    }
  }
  __syncthreads();
  for (int p = threadIdx.x; p < a.hd * 2; p += 256) {
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = words[vslot(p >> 1, (p & 1) * 4 + j)];
    *reinterpret_cast<u32x4*>(code + p * 16) = o;
  }
}

// The same blocks back to rows [0, count[b]) of k and v; zero: rows [count[b], T) become zeros.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) load_kernel(CacheArgs a) {
  __shared__ unsigned words[256 * 8];
  const int per = (a.T + BT - 1) / BT;
  int i = blockIdx.x;
  const int blk = i % per;
  i /= per;
  const bool val = i & 1;
  i >>= 1;
  const int h = i % a.H, b = i / a.H;
  const int held = max(0, min(a.count[b], a.nblk * BT)) - blk * BT, rows = min(BT, a.T - blk * BT);
  if (held <= 0 && !a.zero) return;
  const Rows& r = val ? a.vr : a.kr;
  const size_t unit = ((size_t)b * a.H + h) * a.nblk + blk;
  const unsigned char* code = (val ? a.v : a.k) + unit * BT * a.hd;
  const float s = held > 0 ? (val ? a.vs : a.ks)[unit] : 0.f;
  const int c8 = threadIdx.x % (a.hd / 8), rg = threadIdx.x / (a.hd / 8);
  if (val && held > 0) {
    for (int p = threadIdx.x; p < a.hd * 2; p += 256) {
      const u32x4 o = *reinterpret_cast<const u32x4*>(code + p * 16);
#pragma unroll
      for (int j = 0; j < 4; j++) words[vslot(p >> 1, (p & 1) * 4 + j)] = o[j];
    }
    __syncthreads();
  }
  if (rg >= 8) return;
  unsigned c[8];
  if (val && held > 0) {
#pragma unroll
    for (int d = 0; d < 8; d++) c[d] = words[vslot(8 * c8 + d, rg)];
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int row = 4 * rg + j;
    if (row >= rows || (row >= held && !a.zero)) continue;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row < held) {
      u32x2 w;
      if (val) {
        const unsigned sh = 8 * j;
        w[0] = ((c[0] >> sh) & 0xffu) | (((c[1] >> sh) & 0xffu) << 8) | (((c[2] >> sh) & 0xffu) << 16) | ((c[3] >> sh) << 24);
        w[1] = ((c[4] >> sh) & 0xffu) | (((c[5] >> sh) & 0xffu) << 8) | (((c[6] >> sh) & 0xffu) << 16) | ((c[7] >> sh) << 24);
      } else {
        w = *reinterpret_cast<const u32x2*>(code + ((c8 >> 1) * BT + row) * 16 + (c8 & 1) * 8);
      }
      float y[4];
      values4(w[0], y);
#pragma unroll
      for (int d = 0; d < 4; d++) x[d] = y[d] * s;
      values4(w[1], y);
#pragma unroll
      for (int d = 0; d < 4; d++) x[4 + d] = y[d] * s;
    }
    store8<DT, VEC>(r, b * r.sb + (int64_t)(blk * BT + row) * r.st + h * r.sh + 8 * c8 * r.sd, x);
  }
}

int check_cache(const void* k, const void* v, const void* ks, const void* vs, int batch, int heads, int hd, int blocks,
                const char* who) {
  if (batch < 1 || heads < 1 || blocks < 1 || batch > (1 << 20) || heads > (1 << 16) || blocks >= (1 << 26))
    return host::fail(FA_ERR_INVALID_ARG, "%s: batch=%d, kv_heads=%d, blocks=%d", who, batch, heads, blocks);
  if (hd != 64 && hd != 96 && hd != 128 && hd != 256)
    return host::fail(FA_ERR_INVALID_ARG, "%s: head_dim=%d is none of 64, 96, 128, 256", who, hd);
  const struct {
    const void* p;
    const char* name;
    unsigned align;
  } ptrs[] = {{k, "k", 16}, {v, "v", 16}, {ks, "ks", 4}, {vs, "vs", 4}};
  for (const auto& t : ptrs) {
    if (!t.p) return host::fail(FA_ERR_INVALID_ARG, "%s: cache %s is NULL", who, t.name);
    if (reinterpret_cast<uintptr_t>(t.p) % t.align)
      return host::fail(FA_ERR_INVALID_ARG, "%s: cache %s is not %u-byte aligned", who, t.name, t.align);
  }
  return FA_OK;
}

int rows_args(const fa_kv8_rows_args* a, bool store, CacheArgs& c, bool& vec, const char* who) {
  if (!a) return host::fail(FA_ERR_INVALID_ARG, "%s: args is NULL", who);
  int rc = check_cache(a->cache_k, a->cache_v, a->cache_ks, a->cache_vs, a->batch, a->kv_heads, a->head_dim, a->blocks, who);
  if (rc != FA_OK) return rc;
  if (a->dtype != FA_DTYPE_BF16 && a->dtype != FA_DTYPE_F16 && a->dtype != FA_DTYPE_F32)
    return host::fail(FA_ERR_INVALID_ARG, "%s: dtype %d: rows are bf16, fp16 or fp32", who, a->dtype);
  if (a->tokens < 0 || a->tokens > (1 << 30))
    return host::fail(FA_ERR_INVALID_ARG, "%s: tokens=%d", who, a->tokens);
  const int size = a->dtype == FA_DTYPE_F32 ? 4 : 2;
  if (a->tokens > 0 && (!a->k || !a->v)) return host::fail(FA_ERR_INVALID_ARG, "%s: k or v is NULL", who);
  if (reinterpret_cast<uintptr_t>(a->k) % size || reinterpret_cast<uintptr_t>(a->v) % size)
    return host::fail(FA_ERR_INVALID_ARG, "%s: k or v is not aligned to its elements", who);
  if (store ? !a->start : !a->count)
    return host::fail(FA_ERR_INVALID_ARG, "%s: %s is NULL", who, store ? "start" : "count");
  if (reinterpret_cast<uintptr_t>(a->start) % 4 || reinterpret_cast<uintptr_t>(a->count) % 4)
    return host::fail(FA_ERR_INVALID_ARG, "%s: start or count is not 4-byte aligned", who);
  vec = a->k_stride[3] == 1 && a->v_stride[3] == 1 && reinterpret_cast<uintptr_t>(a->k) % 16 == 0 &&
        reinterpret_cast<uintptr_t>(a->v) % 16 == 0;
  for (int i = 0; i < 3; i++) vec = vec && a->k_stride[i] * size % 16 == 0 && a->v_stride[i] * size % 16 == 0;
  auto rows = [](const void* p, const long long* s) {
    return Rows{static_cast<unsigned char*>(const_cast<void*>(p)), s[0], s[1], s[2], s[3]};
  };
  c = CacheArgs{static_cast<unsigned char*>(a->cache_k),
                static_cast<unsigned char*>(a->cache_v),
                a->cache_ks,
                a->cache_vs,
                rows(a->k, a->k_stride),
                rows(a->v, a->v_stride),
                a->start,
                a->count,
                a->batch,
                a->tokens,
                a->kv_heads,
                a->head_dim,
                a->blocks,
                a->zero_rest};
  return FA_OK;
}

template <int DT>
void launch_rows(const CacheArgs& c, bool store, bool vec, unsigned grid, hipStream_t s) {
  if (store)
    if (vec) hipLaunchKernelGGL((store_kernel<DT, true>), dim3(grid), dim3(256), 0, s, c);
    else hipLaunchKernelGGL((store_kernel<DT, false>), dim3(grid), dim3(256), 0, s, c);
  else if (vec) hipLaunchKernelGGL((load_kernel<DT, true>), dim3(grid), dim3(256), 0, s, c);
  else hipLaunchKernelGGL((load_kernel<DT, false>), dim3(grid), dim3(256), 0, s, c);
}

int run_rows(const fa_kv8_rows_args* a, bool store, fa_stream_t stream) {
  const char* who = store ? "fa_kv8_store" : "fa_kv8_load";
  CacheArgs c;
  bool vec;
  int rc = rows_args(a, store, c, vec, who);
  if (rc != FA_OK) return rc;
  if (a->tokens == 0) return FA_OK;
  const int64_t per = store ? (a->tokens + 30) / BT + 1 : (a->tokens + BT - 1) / BT;
  const int64_t grid = per * 2 * a->kv_heads * a->batch;
  if (grid > 0x7fffffff) return host::fail(FA_ERR_INVALID_ARG, "%s: too many rows for one call", who);
  rc = host::check_gfx950(who);
  if (rc != FA_OK) return rc;
  if (a->dtype == FA_DTYPE_F32) launch_rows<FA_DTYPE_F32>(c, store, vec, (unsigned)grid, (hipStream_t)stream);
  else if (a->dtype == FA_DTYPE_F16) launch_rows<FA_DTYPE_F16>(c, store, vec, (unsigned)grid, (hipStream_t)stream);
  else launch_rows<FA_DTYPE_BF16>(c, store, vec, (unsigned)grid, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return host::fail(FA_ERR_LAUNCH, "%s: %s", who, hipGetErrorString(e));
  return FA_OK;
}

}  // namespace kv8
}  // namespace fa

extern "C" int fa_kv8_store(const fa_kv8_rows_args* a, fa_stream_t stream) { return fa::kv8::run_rows(a, true, stream); }
extern "C" int fa_kv8_load(const fa_kv8_rows_args* a, fa_stream_t stream) { return fa::kv8::run_rows(a, false, stream); }
