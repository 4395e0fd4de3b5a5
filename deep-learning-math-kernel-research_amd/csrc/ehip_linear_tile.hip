// Products of many rows of activations with a matrix, or with the matrices of the experts they are sent to: tiles of both
// operands staged through LDS for the matrix cores.
#include "ehip_layers.hpp"
#include "ehip_linear_tile.hpp"

namespace ehip {

// 64 lanes x 16 bytes from memory into LDS at lds + 16 * lane, no registers between.  The wait is the caller's.
__device__ __forceinline__ void load_to_lds(const char *src, unsigned lds)
{
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(src) : "memory", "m0");
}

// A workgroup has WN x WM waves of NTW x MTW tiles of 16 x 16 results.  A step is 128 bytes of K: while the waves multiply the
// operands of one step out of LDS, those of the next arrive in the other half.  ALIGNED: rows of activations at multiples of 16
// bytes and a whole number of 16-byte parts in K, so they go straight into LDS too; else through registers.
template <int TYPE, int NTW, int MTW, int WN, int WM, bool ALIGNED>
__global__ __launch_bounds__(WN * WM * 64) void k_linear_tile(LinearArgs a)
{
  typedef Product<TYPE> P;
  typedef typename P::Acc Acc;
  constexpr int WAVES = WN * WM, BN = NTW * WN, BM = MTW * WM, STAGE = (BN + BM) * 2048;
  constexpr int WL = BN / WAVES, XL = BM / WAVES;   // tiles of each operand that a wave loads
  static_assert(BN % WAVES == 0 && BM % WAVES == 0, "every wave loads as much");
  extern __shared__ char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;

  // blocks of an XCD are neighbours: 4 of rows x 8 of columns, so that 32 CUs share 12 panels in its L2
  const int total = a.blocks_m * a.blocks_n, per_xcd = (total + 7) / 8;
  const int index = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || index >= total) return;
  const int group = index / (4 * a.blocks_n), rest = index - group * 4 * a.blocks_n;
  const int high = a.blocks_m - group * 4 < 4 ? a.blocks_m - group * 4 : 4;
  const int bn = rest / high, bm = group * 4 + rest - bn * high;
  const Block blk = block_of(a, bm, 16 * BM);
  if (blk.expert < 0) return;

  // what the wave loads: WL tiles of weights (tiles past the last repeat it, their results are dropped) and XL of activations
  const char *wsrc[WL];
#pragma unroll
  for (int i = 0; i < WL; ++i) {
    const int tile = bn * BN + wave * WL + i;
    wsrc[i] = a.w + ((long long)blk.expert * a.tiles + (tile < a.tiles ? tile : a.tiles - 1)) * a.chunks * 1024 + lane * 16;
  }
  const char *xsrc[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const long long p = blk.first + (wave * XL + i) * 16 + c;
    xsrc[i] = a.x + row_of(a, p < blk.last ? p : blk.last - 1).in * a.ldx + g * 16;
  }
  const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
  const int steps = a.chunks >> 1;

  i4 xr[XL][2];
  auto load = [&](int step, int stage) {
    const unsigned to = base + stage * STAGE;
#pragma unroll
    for (int i = 0; i < WL; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) load_to_lds(wsrc[i] + (long long)step * 2048 + h * 1024, to + (wave * WL + i) * 2048 + h * 1024);
#pragma unroll
    for (int i = 0; i < XL; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = step * 128 + h * 64;
        if (ALIGNED) load_to_lds(at + g * 16 < a.kbytes ? xsrc[i] + at : a.zeros, to + (BN + wave * XL + i) * 2048 + h * 1024);
        else xr[i][h] = load_part<P::elem>(xsrc[i] + at, a.kbytes - at - g * 16);
      }
  };
  auto put = [&](int stage) {
    if (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < XL; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<i4 *>(lds + stage * STAGE + (BN + wave * XL + i) * 2048 + h * 1024 + lane * 16) = xr[i][h];
    }
  };

  const int wn = wave % WN, wm = wave / WN;
  Acc acc[NTW][MTW];
#pragma unroll
  for (int n = 0; n < NTW; ++n)
#pragma unroll
    for (int m = 0; m < MTW; ++m) acc[n][m] = Acc{0, 0, 0, 0};

  load(0, 0);
  put(0);
  for (int step = 0; step < steps; ++step) {
    const int stage = step & 1;
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_s_barrier();
    if (step + 1 < steps) load(step + 1, stage ^ 1);
    const char *wl = lds + stage * STAGE + wn * NTW * 2048 + lane * 16;
    const char *xl = lds + stage * STAGE + (BN + wm * MTW) * 2048 + lane * 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i4 wq[NTW], xq[MTW];
#pragma unroll
      for (int m = 0; m < MTW; ++m) xq[m] = *reinterpret_cast<const i4 *>(xl + m * 2048 + h * 1024);
#pragma unroll
      for (int n = 0; n < NTW; ++n) wq[n] = *reinterpret_cast<const i4 *>(wl + n * 2048 + h * 1024);
#pragma unroll
      for (int n = 0; n < NTW; ++n)
#pragma unroll
        for (int m = 0; m < MTW; ++m) acc[n][m] = P::mma(wq[n], xq[m], acc[n][m]);
    }
    if (step + 1 < steps) put(stage ^ 1);
  }

#pragma unroll
  for (int m = 0; m < MTW; ++m) {
    const long long p = blk.first + (wm * MTW + m) * 16 + c;
    if (p >= blk.last) continue;
    const RowOf row = row_of(a, p);
    if (!row.there) continue;
    const float xs = a.xscale ? a.xscale[row.in] : 1.0f;
    char *orow = a.out + row.out * a.ldo;
    const char *rrow = a.res ? a.res + row.out * a.ldr : nullptr;
#pragma unroll
    for (int n = 0; n < NTW; n += 4) {
      const int tile = bn * BN + wn * NTW + n;
      if (tile >= a.tiles) continue;
      const long long at = ((long long)blk.expert * a.tiles + tile) * 16 + g * 4;
      if (a.gated) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f4 gate = finish_sums(a, acc[n + 2 * u][m], at + 32 * u, xs), up = finish_sums(a, acc[n + 2 * u + 1][m], at + 32 * u + 16, xs);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[4 * u + r] = activate(gate[r], a.act) * up[r];
        }
        store_columns<8>(a, v, orow, rrow, (tile >> 2) * 32 + g * 8);
      } else {
        float v[16];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const f4 s = finish_sums(a, acc[n + t][m], at + 16 * t, xs);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[4 * t + r] = activate(s[r], a.act);
        }
        store_columns<16>(a, v, orow, rrow, (tile >> 2) * 64 + g * 16);
      }
    }
  }
}

namespace {

template <int TYPE, int NTW, int MTW, int WN, int WM>
hipError_t run(LinearArgs a, long long blocks_m, hipStream_t s)
{
  const long long n = (a.tiles + NTW * WN - 1) / (NTW * WN), all = (blocks_m * n + 7) / 8 * 8;
  if (all >= 1ll << 31) return hipErrorInvalidValue;
  a.blocks_m = (int)blocks_m;
  a.blocks_n = (int)n;
  const bool aligned = ((uintptr_t)a.x | (unsigned long long)a.ldx | (unsigned)a.kbytes) % 16 == 0;
  constexpr int lds = (NTW * WN + MTW * WM) * 2048 * 2;
  auto kernel = aligned ? k_linear_tile<TYPE, NTW, MTW, WN, WM, true> : k_linear_tile<TYPE, NTW, MTW, WN, WM, false>;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)all), dim3(WN * WM * 64), lds, s, a);
  return hipGetLastError();
}

template <int TYPE>
hipError_t run_typed(const LinearArgs &a, int form, long long blocks_m, hipStream_t s)
{
  if (form == 0) return run<TYPE, 4, 4, 2, 2>(a, blocks_m, s);
  return run<TYPE, 8, 4, 2, 4>(a, blocks_m, s);
}

}  // namespace

hipError_t launch_linear_tile(const LinearArgs &a, int type, int form, long long blocks_m, hipStream_t s)
{
  switch (type) {
  case EHIP_BF16: return run_typed<EHIP_BF16>(a, form, blocks_m, s);
  case EHIP_F16: return run_typed<EHIP_F16>(a, form, blocks_m, s);
  default: return run_typed<EHIP_S8>(a, form, blocks_m, s);
  }
}

}  // namespace ehip
