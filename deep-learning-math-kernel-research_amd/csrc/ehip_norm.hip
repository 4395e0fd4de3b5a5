// The norm after a block, its gate and residual scale, and the norm before the next block, on rows held in registers: every
// input is read once and every output written once, so memory bounds it: 16384 x 4096 bf16 with both norms, gate and residual
// 110 us, 4.87 TB/s of reads and writes (a large copy of as many reads as writes: 4.94).
#include "ehip_layers.hpp"

namespace ehip {
namespace {

template <int TYPE> struct Elem {
  static constexpr int size = 2;
};
template <> struct Elem<EHIP_F32> {
  static constexpr int size = 4;
};

// 8 columns from p on as f32; only the first n exist, the others are 0
template <int TYPE>
__device__ __forceinline__ void load8(const char *p, int n, float (&v)[8])
{
  if (n >= 8) {
    if constexpr (TYPE == EHIP_F32) {
      typedef float fu __attribute__((ext_vector_type(4), aligned(4)));
      const fu a = *reinterpret_cast<const fu *>(p), b = *reinterpret_cast<const fu *>(p + 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = a[j];
        v[4 + j] = b[j];
      }
    } else {
      const i4 a = *reinterpret_cast<const i4u *>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) unpack((unsigned)a[j], TYPE == EHIP_BF16, v[2 * j], v[2 * j + 1]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < n ? load_one(p + j * Elem<TYPE>::size, TYPE) : 0.0f;
}
template <int TYPE>
__device__ __forceinline__ void store8(char *p, int n, const float (&v)[8])
{
  if (n >= 8) {
    if constexpr (TYPE == EHIP_F32) {
      typedef float fu __attribute__((ext_vector_type(4), aligned(4)));
      *reinterpret_cast<fu *>(p) = fu{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<fu *>(p + 16) = fu{v[4], v[5], v[6], v[7]};
    } else {
      i4 a;
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = (int)(TYPE == EHIP_BF16 ? pack_bf16(v[2 * j], v[2 * j + 1]) : pack_f16(v[2 * j], v[2 * j + 1]));
      *reinterpret_cast<i4u *>(p) = a;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) store_one(p + j * Elem<TYPE>::size, TYPE, v[j]);
}

// over the 64 lanes, by cross-lane operands; the same bits in each of them
__device__ __forceinline__ float over_wave(float v)
{
  v += dpp<kShr1>(0.0f, v);
  v += dpp<kShr2>(0.0f, v);
  v += dpp<kShr4>(0.0f, v);
  v += dpp<kShr8>(0.0f, v);
  v += dpp<kBcast15, 0xa>(0.0f, v);
  v += dpp<kBcast31, 0xc>(0.0f, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned over_wave(unsigned v)
{
  v = larger(v, (unsigned)dpp<kShr1>(0, (int)v));
  v = larger(v, (unsigned)dpp<kShr2>(0, (int)v));
  v = larger(v, (unsigned)dpp<kShr4>(0, (int)v));
  v = larger(v, (unsigned)dpp<kShr8>(0, (int)v));
  v = larger(v, (unsigned)dpp<kBcast15, 0xa>(0, (int)v));
  v = larger(v, (unsigned)dpp<kBcast31, 0xc>(0, (int)v));
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
// Sum (or, of bit patterns without a sign, the maximum: a NaN's is above every number's, so it is kept) over the THREADS of a
// row, the same bits in each of them
template <int THREADS, typename T, typename Op>
__device__ __forceinline__ T over_row(T v, T *room, Op op)
{
  v = over_wave(v);
  if constexpr (THREADS > 64) {
    __syncthreads();   // the room's last readers
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = v;
    __syncthreads();
    v = room[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v = op(v, room[w]);
  }
  return v;
}

// THREADS threads have a row (64: four rows to a workgroup), each of them V runs of 8 columns, THREADS * 8 apart.  Two passes over the registers for the
// variance of a layer norm: a row whose mean is large against its spread loses nothing.
template <int TYPE, bool S8, int THREADS, int V>
__global__ __launch_bounds__(THREADS == 64 ? 256 : THREADS) void k_norm(NormArgs a)
{
  constexpr int ROWS = THREADS == 64 ? 4 : 1, SIZE = Elem<TYPE>::size;
  __shared__ float froom[THREADS > 64 ? THREADS / 64 : 1];
  __shared__ unsigned uroom[THREADS > 64 ? THREADS / 64 : 1];
  const long long r = (a.first + blockIdx.x) * ROWS + (ROWS > 1 ? threadIdx.x / THREADS : 0);
  if (r >= a.rows) return;   // (whole waves: rows share a workgroup only where a wave has one)
  const int t = threadIdx.x % THREADS;
  auto add = [](float x, float y) { return x + y; };
  const float inv = 1.0f / (float)a.cols;

  float v[V][8];
  if (a.parts == 1 && !a.pw) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = (i * THREADS + t) * 8;
      load8<TYPE>(a.block + r * a.ldb + (long long)col * SIZE, a.cols - col, v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    for (int p = 0; p < a.parts; ++p) {
      const float w = a.pw[r * a.parts + p];
      if (w == 0.0f) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int col = (i * THREADS + t) * 8;
        float q[8];
        load8<TYPE>(a.block + (r * a.parts + p) * a.ldb + (long long)col * SIZE, a.cols - col, q);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = __builtin_fmaf(w, q[j], v[i][j]);
      }
    }
  }

  auto norm = [&](int kind, float eps, const float *w, const float *b) {
    if (kind == EHIP_NORM_LAYER) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[i][j];
      const float mean = over_row<THREADS>(s, froom, add) * inv;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int n = a.cols - (i * THREADS + t) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = j < n ? v[i][j] - mean : 0.0f;
      }
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s = __builtin_fmaf(v[i][j], v[i][j], s);
    const float rstd = 1.0f / sqrtf(over_row<THREADS>(s, froom, add) * inv + eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = (i * THREADS + t) * 8, n = a.cols - col;
      if (n <= 0) continue;
      float wv[8], bv[8];
      if (w) load8<EHIP_F32>(reinterpret_cast<const char *>(w + col), n, wv);
      if (b) load8<EHIP_F32>(reinterpret_cast<const char *>(b + col), n, bv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] *= rstd;
        if (w) v[i][j] *= wv[j];
        if (b) v[i][j] += bv[j];
      }
    }
  };

  if (a.post != EHIP_NORM_NONE) norm(a.post, a.eps1, a.w1, a.b1);
  const char *gate = a.gate ? a.gate + (a.rows_per_gate ? r / a.rows_per_gate : 0) * a.ldg : nullptr;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int col = (i * THREADS + t) * 8, n = a.cols - col;
    if (n <= 0) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] *= a.block_scale;
    if (gate) {
      float q[8];
      load8<TYPE>(gate + (long long)col * SIZE, n, q);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= q[j];
    }
    if (a.res) {
      float q[8];
      load8<TYPE>(a.res + r * a.ldr + (long long)col * SIZE, n, q);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = __builtin_fmaf(a.res_scale, q[j], v[i][j]);
    }
    if (a.sum) store8<TYPE>(a.sum + r * a.lds + (long long)col * SIZE, n, v[i]);
  }
  if (!a.out) return;
  if (a.pre != EHIP_NORM_NONE) norm(a.pre, a.eps2, a.w2, a.b2);

  if constexpr (S8) {
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = a.cols - (i * THREADS + t) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned m = __builtin_bit_cast(unsigned, v[i][j]) & 0x7fffffffu;
        if (j < n && m > most) most = m;
      }
    }
    most = over_row<THREADS>(most, uroom, larger);
    const float amax = __builtin_bit_cast(float, most);
    // a row of zeros has codes 0 and scale 0; one with an infinity or a NaN says so in its scale
    const float lift = amax < 1e-30f ? 0x1p64f : 1.0f;   // 127 / amax stays finite
    const float to_code = amax > 0.0f ? 127.0f / (amax * lift) : 0.0f;
    if (t == 0) a.out_scale[r] = amax / 127.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = (i * THREADS + t) * 8, n = a.cols - col;
      if (n <= 0) continue;
      unsigned d[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = __builtin_amdgcn_fmed3f(__builtin_rintf(v[i][j] * lift * to_code), -127.0f, 127.0f);
        d[j / 4] |= ((unsigned)(int)f & 0xffu) << (8 * (j % 4));
      }
      char *o = a.out + r * a.ldo + col;
      if (n >= 8) {
        typedef unsigned u2 __attribute__((ext_vector_type(2), aligned(1)));
        *reinterpret_cast<u2 *>(o) = u2{d[0], d[1]};
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n) o[j] = (char)(d[j / 4] >> (8 * (j % 4)));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = (i * THREADS + t) * 8, n = a.cols - col;
      if (n > 0) store8<TYPE>(a.out + r * a.ldo + (long long)col * SIZE, n, v[i]);
    }
  }
}

template <int TYPE, bool S8, int THREADS, int V>
hipError_t run(NormArgs a, hipStream_t s)
{
  constexpr int rows = THREADS == 64 ? 4 : 1, threads = THREADS == 64 ? 256 : THREADS;
  return launch_pieces((a.rows + rows - 1) / rows, threads, [&](long long first, unsigned count) {
    a.first = first;
    hipLaunchKernelGGL((k_norm<TYPE, S8, THREADS, V>), dim3(count), dim3(threads), 0, s, a);
  });
}

// Eight columns a thread as long as a workgroup has the threads, whatever the rows: bf16, us, against four times as many columns
// a thread: 64 x 4096 3.7 (64 threads: 12.9), 16384 x 4096 113 (120 with 128, 181 with 64), 16384 x 1024 30 (64 threads: 39).
// Above 8192 columns fewer waves that each have more in flight: 4096 x 16384 134, with 1024 threads 162.
template <int TYPE, bool S8>
hipError_t run_wide(const NormArgs &a, hipStream_t s)
{
  if (a.cols <= 512) return run<TYPE, S8, 64, 1>(a, s);
  if (a.cols <= 1024) return run<TYPE, S8, 128, 1>(a, s);
  if (a.cols <= 2048) return run<TYPE, S8, 256, 1>(a, s);
  if (a.cols <= 4096) return run<TYPE, S8, 512, 1>(a, s);
  if (a.cols <= 8192) return run<TYPE, S8, 1024, 1>(a, s);
  if (a.cols <= 16384) return run<TYPE, S8, 512, 4>(a, s);
  if (a.cols <= 32768) return run<TYPE, S8, 1024, 4>(a, s);
  return run<TYPE, S8, 1024, 8>(a, s);
}

template <int TYPE>
hipError_t run_type(const NormArgs &a, int out_s8, hipStream_t s)
{
  return out_s8 ? run_wide<TYPE, true>(a, s) : run_wide<TYPE, false>(a, s);
}

}  // namespace

hipError_t launch_norm(const NormArgs &a, int type, int out_s8, hipStream_t s)
{
  switch (type) {
  case EHIP_F32: return run_type<EHIP_F32>(a, out_s8, s);
  case EHIP_F16: return run_type<EHIP_F16>(a, out_s8, s);
  default: return run_type<EHIP_BF16>(a, out_s8, s);
  }
}

}  // namespace ehip
