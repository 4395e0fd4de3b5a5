// What the kernels of linear, norm, route and experts share: their arguments, element types, the epilogue of a product.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "euler_hip.h"

namespace ehip {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i4u __attribute__((ext_vector_type(4), aligned(1)));   // any address: the load is still one instruction
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// ---- linear ------------------------------------------------------------------------------------------------------
// The packed weights are matrix-core operands: 16 rows x 64 bytes of K = 1 KB, lane l holding the 16 bytes of row l % 16
// from byte 16 * (l / 16) on.  [expert][tile of 16 rows][chunk of 64 bytes][lane].  Four tiles are a group of 64 output
// columns; row i of tile t in it is column 16 * (i / 4) + 4 * t + i % 4, so that a lane, which holds rows 4 g .. 4 g + 3 of
// each tile's result, has 16 columns beside each other.  Gated: tiles 0, 2 are the gates of 32 columns, 1, 3 their partners:
// row i of tiles 2 u, 2 u + 1 is column 8 * (i / 4) + 4 * u + i % 4.
struct LinearArgs {
  const char *w;          // packed
  const float *wscale;    // [expert][tile][16] in the order of the packed rows, or null
  const float *bias;      // likewise
  const char *zeros;      // 16 bytes of zeros
  const char *x;
  const float *xscale;
  char *out;
  const char *res;
  const int32_t *slots, *offsets;   // experts, or null
  long long ldx, ldo, ldr;          // bytes
  long long rows;
  int oc, kbytes;         // real columns of the output, real bytes of K
  int tiles, chunks;      // of the packed weights, per expert: a multiple of 4, a multiple of 2
  int experts, topk, in_rows, out_rows;
  int out_type, act, gated;
  float res_scale;
  int form;                 // EHIP_LINEAR_FORM, or -1
  int blocks_m, blocks_n;   // set by the launcher
  int first;                // number of the launch's first workgroup
};

hipError_t launch_linear_pack(void *packed, const void *weights, int experts, int oc, int ic, int elem, int gated, int tiles, int chunks,
                              char *zeros, hipStream_t s);
hipError_t launch_linear_constants(float *dst, const float *src, int experts, int oc, int gated, int tiles, hipStream_t s);
hipError_t launch_linear(const LinearArgs &a, int type, hipStream_t s);
const char *linear_kernel_name(const LinearArgs &a);   // for rows without gaps, at multiples of 16 bytes
// many rows: tiles of 128 x 128 (form 0; form 1: four steps in LDS) or 256 x 256 (form 2) results staged through LDS
hipError_t launch_linear_tile_bf16(const LinearArgs &a, int form, long long blocks_m, hipStream_t s);
hipError_t launch_linear_tile_f16(const LinearArgs &a, int form, long long blocks_m, hipStream_t s);
hipError_t launch_linear_tile_s8(const LinearArgs &a, int form, long long blocks_m, hipStream_t s);

struct NormArgs {
  char *out;
  float *out_scale;
  char *sum;
  const char *block, *res, *gate;
  const float *pw, *w1, *b1, *w2, *b2;
  long long ldo, lds, ldb, ldr, ldg;   // bytes
  long long rows;
  int cols, parts, post, pre, rows_per_gate;
  float block_scale, res_scale, eps1, eps2;
  long long first;   // number of the launch's first workgroup
};
hipError_t launch_norm(const NormArgs &a, int type, int out_s8, hipStream_t s);

struct RouteArgs {
  int32_t *ids;
  float *weights;
  int32_t *offsets, *slots;
  int32_t *totals, *hist;   // [experts]; [experts][blocks of kRouteBlock tokens]
  const char *logits;
  const float *bias;
  long long tokens, ld;   // ld in bytes
  int experts, topk, groups, open, best, sigmoid, renorm;
  float scale;
};
constexpr int kRouteBlock = 128;   // tokens of a workgroup
constexpr long long kRouteTokens = (1ll << 29) - kRouteBlock;   // a launch's threads are counted in 32 bits, 8 a token
hipError_t launch_route(const RouteArgs &a, int type, hipStream_t s);

// A launch's threads are counted in 32 bits: more workgroups than that go out in pieces.  launch(number of the first, count)
template <typename F>
hipError_t launch_pieces(long long blocks, int threads, F launch)
{
  const long long most = ((1ll << 32) / threads - 1) / 8 * 8;   // (a workgroup's XCD stays its number modulo 8)
  for (long long first = 0; first < blocks; first += most) {
    launch(first, (unsigned)(blocks - first < most ? blocks - first : most));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

#if defined(__HIPCC__)

__device__ __forceinline__ unsigned pack_bf16(float a, float b)
{
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  bf2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ unsigned pack_f16(float a, float b)
{
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  h2 v = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(unsigned, v);
}
// the two values of a dword
__device__ __forceinline__ void unpack(unsigned d, bool bf16, float &lo, float &hi)
{
  if (bf16) {
    lo = __builtin_bit_cast(float, d << 16);
    hi = __builtin_bit_cast(float, d & 0xffff0000u);
  } else {
    lo = (float)__builtin_bit_cast(_Float16, (uint16_t)(d & 0xffffu));
    hi = (float)__builtin_bit_cast(_Float16, (uint16_t)(d >> 16));
  }
}
// one element of type EHIP_F32 / F16 / BF16
__device__ __forceinline__ float load_one(const char *p, int type)
{
  if (type == EHIP_F32) return *reinterpret_cast<const float *>(p);
  if (type == EHIP_F16) return (float)*reinterpret_cast<const _Float16 *>(p);
  return (float)*reinterpret_cast<const __bf16 *>(p);
}
__device__ __forceinline__ void store_one(char *p, int type, float v)
{
  if (type == EHIP_F32) *reinterpret_cast<float *>(p) = v;
  else if (type == EHIP_F16) *reinterpret_cast<_Float16 *>(p) = (_Float16)v;
  else *reinterpret_cast<__bf16 *>(p) = (__bf16)v;
}

// v of the lane that DPP control CTRL names; lanes without one, or outside of ROWS, keep `old`
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int dpp(int old, int v)
{
  return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float old, float v)
{
  return __builtin_bit_cast(float, dpp<CTRL, ROWS>(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v)));
}
constexpr int kShr1 = 0x111, kShr2 = 0x112, kShr4 = 0x114, kShr8 = 0x118, kBcast15 = 0x142, kBcast31 = 0x143;

// 16 bytes at p of which the first `valid` exist; the others are zero.  ELEM: bytes of an element
template <int ELEM>
__device__ __forceinline__ i4 load_part(const char *p, int valid)
{
  if (valid >= 16) return *reinterpret_cast<const i4u *>(p);
  uint64_t half[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 16 / ELEM; ++j)
    if ((j + 1) * ELEM <= valid) {
      const uint64_t e = ELEM == 1 ? (uint64_t)reinterpret_cast<const uint8_t *>(p)[j] : (uint64_t)reinterpret_cast<const uint16_t *>(p)[j];
      half[j * ELEM / 8] |= e << (8 * (j * ELEM % 8));
    }
  return i4{(int)half[0], (int)(half[0] >> 32), (int)half[1], (int)(half[1] >> 32)};
}

// The matrix instruction on two 16-byte operands: 16 rows of weights x 16 rows of activations, 64 bytes of K.  Lane l gets
// rows 4 * (l / 16) .. + 3 of the weights for row l % 16 of the activations.
template <int TYPE> struct Product;
template <> struct Product<EHIP_BF16> {
  typedef f4 Acc;
  static constexpr int elem = 2;
  __device__ static __forceinline__ Acc mma(i4 w, i4 x, Acc c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, w), __builtin_bit_cast(bf8, x), c, 0, 0, 0);
  }
};
template <> struct Product<EHIP_F16> {
  typedef f4 Acc;
  static constexpr int elem = 2;
  __device__ static __forceinline__ Acc mma(i4 w, i4 x, Acc c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, w), __builtin_bit_cast(h8, x), c, 0, 0, 0);
  }
};
template <> struct Product<EHIP_S8> {
  typedef i4 Acc;
  static constexpr int elem = 1;
  __device__ static __forceinline__ Acc mma(i4 w, i4 x, Acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0); }
};

// The activation functions in single precision, for results of type TYPE.  Units are 2^-24 of a value.
// GELU: v * Phi(v) = max(v, 0) - |v| * Phi(-|v|) = max(v, 0) - x * erfc(sqrt(2) x), x = |v| / 2.  For v < 0 the second term is all of
// the result, and a gate's partner can make it large: it keeps its digits however small it is, down to the least exponential, whose
// place is v = -13.
//   16-bit results: x * 2^(x p(x)), p of degree 10 fitted to log2(erfc(sqrt(2) x)) / x on 0 <= x <= 6.6 (least squares of the term,
//   weighted until its largest error, against 2 units of |v| or 5e-5 of the term, is even): off by at most 3.3 units of |v|, and
//   by 8.2e-5 of the term down to v = -8, 1.3e-4 from there (f16 rounds by 4.9e-4); the exponent's roundings add 14 (1 + v^2) units
//   of the term.  One transcendental instruction and 15 others.
//   f32 results: x * exp(-2 x^2) * E(x), E = erfc(sqrt(2) x) exp(2 x^2): 1 at 0 and like 1 / x far out, so a polynomial without a
//   constant in t = 1 / (1 + 0.7 x).  Degree 9 on 0 <= x <= 7, fitted likewise: 3.2e-8.  With the roundings (of t, counted 2.3
//   times, and of the exponent, v^2 / 2 times) 16 + 2 v^2 units of the term.  Two transcendental instructions and 17 others: f16 results
//   of s8 3001 x 4104 x 5000 would take 80 us with it where they take 77, f32 results of bf16 4096 x 1024 x 4096 take 43 (41 without).
// SiLU: off by at most 8 + 2 |v| units (the exponent's roundings); the exponential of a large negative v is infinite and the
// result -0, as the limit is.
template <int ACT, int TYPE>
__device__ __forceinline__ float activate(float v)
{
  if (ACT == EHIP_ACT_RELU) return v > 0.0f ? v : v != v ? v : 0.0f;
  if (ACT == EHIP_ACT_GELU) {
    const float h = 0.5f * v;
    if (TYPE == EHIP_F32) {
      const float x = __builtin_fminf(__builtin_fabsf(h), 7.0f);
      const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(x, 0.7f, 1.0f));
      float p = __builtin_fmaf(t, -0.058291804f, 0.28794315f);
      p = __builtin_fmaf(t, p, -0.51142806f);
      p = __builtin_fmaf(t, p, 0.31834787f);
      p = __builtin_fmaf(t, p, -0.046219379f);
      p = __builtin_fmaf(t, p, 0.21101590f);
      p = __builtin_fmaf(t, p, 0.23966576f);
      p = __builtin_fmaf(t, p, 0.27972373f);
      p = __builtin_fmaf(t, p, 0.27924281f);
      const float e = __builtin_amdgcn_exp2f(x * (x * -2.8853901f));
      return __builtin_fmaf(-(x * e), p * t, h + __builtin_fabsf(h));
    }
    const float x = __builtin_fminf(__builtin_fabsf(h), 6.6f);
    float p = __builtin_fmaf(x, 1.3627697e-7f, -4.6344026e-6f);
    p = __builtin_fmaf(x, p, 6.6200366e-5f);
    p = __builtin_fmaf(x, p, -5.0509541e-4f);
    p = __builtin_fmaf(x, p, 0.0020654162f);
    p = __builtin_fmaf(x, p, -0.0026251888f);
    p = __builtin_fmaf(x, p, -0.017977515f);
    p = __builtin_fmaf(x, p, 0.12327838f);
    p = __builtin_fmaf(x, p, -0.42386577f);
    p = __builtin_fmaf(x, p, -1.8361757f);
    p = __builtin_fmaf(x, p, -2.3022454f);
    return __builtin_fmaf(-x, __builtin_amdgcn_exp2f(x * p), h + __builtin_fabsf(h));
  }
  if (ACT == EHIP_ACT_SILU) return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
  return v;
}
// f(integral constants of the activation, the output type and whether it is gated): code for each, chosen once
template <int V> struct Const {
  static constexpr int value = V;
};
template <typename F>
__device__ __forceinline__ void for_epilogue(const LinearArgs &a, F f)
{
  auto with_act = [&](auto act) {
    auto with_type = [&](auto type) {
      if (a.gated) f(act, type, Const<1>());
      else f(act, type, Const<0>());
    };
    if (a.out_type == EHIP_BF16) with_type(Const<EHIP_BF16>());
    else if (a.out_type == EHIP_F16) with_type(Const<EHIP_F16>());
    else with_type(Const<EHIP_F32>());
  };
  if (a.act == EHIP_ACT_NONE) with_act(Const<EHIP_ACT_NONE>());
  else if (a.act == EHIP_ACT_SILU) with_act(Const<EHIP_ACT_SILU>());
  else if (a.act == EHIP_ACT_GELU) with_act(Const<EHIP_ACT_GELU>());
  else with_act(Const<EHIP_ACT_RELU>());
}

// a tile's sums of one lane as f32: scaled (s8), with bias.  at: the lane's first row in the packed order
template <typename Acc>
__device__ __forceinline__ f4 finish_sums(const LinearArgs &a, Acc acc, long long at, float xs)
{
  f4 v = {(float)acc[0], (float)acc[1], (float)acc[2], (float)acc[3]};
  if (a.wscale) {
    const f4 ws = *reinterpret_cast<const f4 *>(a.wscale + at);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] *= xs * ws[r];
  }
  if (a.bias) {
    const f4 b = *reinterpret_cast<const f4 *>(a.bias + at);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += b[r];
  }
  return v;
}

// N (a multiple of 4) columns beside each other of one row at o (its residual at r, or null): residual, rounding, store.  Only
// the first n exist.
template <int TYPE, int N>
__device__ __forceinline__ void store_columns(float (&v)[N], char *o, const char *r, float res_scale, int n)
{
  constexpr int SIZE = TYPE == EHIP_F32 ? 4 : 2;
  if (n < N) {
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (q < n) store_one(o + q * SIZE, TYPE, r ? __builtin_fmaf(res_scale, load_one(r + q * SIZE, TYPE), v[q]) : v[q]);
    return;
  }
  if constexpr (TYPE == EHIP_F32) {
    typedef float fu __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (int q = 0; q < N; q += 4) {
      fu s = {v[q], v[q + 1], v[q + 2], v[q + 3]};
      if (r) {
        const fu old = *reinterpret_cast<const fu *>(r + 4 * q);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = __builtin_fmaf(res_scale, old[j], s[j]);
      }
      *reinterpret_cast<fu *>(o + 4 * q) = s;
    }
  } else {
    // 4 columns of 16 bits are 8 bytes, 8 are 16
    constexpr int STEP = N % 8 == 0 ? 8 : 4;
    typedef unsigned dw __attribute__((ext_vector_type(STEP / 2), aligned(2)));
#pragma unroll
    for (int q = 0; q < N; q += STEP) {
      if (r) {
        const dw old = *reinterpret_cast<const dw *>(r + 2 * q);
#pragma unroll
        for (int j = 0; j < STEP / 2; ++j) {
          float lo, hi;
          unpack(old[j], TYPE == EHIP_BF16, lo, hi);
          v[q + 2 * j] = __builtin_fmaf(res_scale, lo, v[q + 2 * j]);
          v[q + 2 * j + 1] = __builtin_fmaf(res_scale, hi, v[q + 2 * j + 1]);
        }
      }
      dw p;
#pragma unroll
      for (int j = 0; j < STEP / 2; ++j)
        p[j] = TYPE == EHIP_BF16 ? pack_bf16(v[q + 2 * j], v[q + 2 * j + 1]) : pack_f16(v[q + 2 * j], v[q + 2 * j + 1]);
      *reinterpret_cast<dw *>(o + 2 * q) = p;
    }
  }
}

// Rows of the activations and of the output for position `p` of the product.  there = false: a slot that is out of range,
// whose row 0 may be read in its place and which is not written
struct RowOf {
  long long in, out;
  bool there;
};
__device__ __forceinline__ RowOf row_of(const LinearArgs &a, long long p)
{
  RowOf r = {p, p, true};
  if (a.slots && (a.in_rows != EHIP_ROWS_SORTED || a.out_rows != EHIP_ROWS_SORTED)) {
    const int s = a.slots[p];
    r.there = s >= 0 && s < a.rows;
    const int c = r.there ? s : 0;
    if (a.in_rows != EHIP_ROWS_SORTED) r.in = a.in_rows == EHIP_ROWS_TOKEN ? c / a.topk : c;
    if (a.out_rows != EHIP_ROWS_SORTED) r.out = c;
  }
  return r;
}

// Which expert's positions [first, last) the index-th block of `rows` of them has, blocks counted expert after expert; past
// the last one there is no work (expert < 0).  Every lane gets the same answer.  An offset out of range counts as the nearest
// one in it.
struct Block {
  int expert;
  long long first, last;
};
__device__ __forceinline__ Block block_of(const LinearArgs &a, int index, int rows)
{
  if (!a.offsets) return {0, (long long)index * rows, a.rows};
  const int lane = threadIdx.x & 63, most = (int)a.rows;
  int before = 0;
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;
    if (e < a.experts) {
      lo = a.offsets[e];
      hi = a.offsets[e + 1];
    }
    lo = lo < 0 ? 0 : lo > most ? most : lo;
    hi = hi < lo ? lo : hi > most ? most : hi;
    const int n = (hi - lo + rows - 1) / rows;
    int sum = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int t = __shfl_up(sum, d);
      if (lane >= d) sum += t;
    }
    const int at = index - before - (sum - n);
    const unsigned long long who = __ballot(at >= 0 && at < n);
    if (who) {
      const int l = __builtin_ctzll(who);
      return {__builtin_amdgcn_readfirstlane(e0 + l), (long long)__builtin_amdgcn_readlane(lo, l) + (long long)__builtin_amdgcn_readlane(at, l) * rows,
              __builtin_amdgcn_readlane(hi, l)};
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return {-1, 0, 0};
}

#endif
}  // namespace ehip
