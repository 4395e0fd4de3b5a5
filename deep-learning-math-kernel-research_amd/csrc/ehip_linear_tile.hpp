// Products of many rows of activations with a matrix, or with the matrices of the experts they are sent to: tiles of both
// operands staged through LDS for the matrix cores.  The kernels of one type a file (ehip_linear_tile_*.hip): they compile side
// by side.
#pragma once
#include "ehip_layers.hpp"

namespace ehip {

// 64 lanes x 16 bytes from memory into LDS at lds + 16 * lane, no registers between.  The wait is the caller's, and so is the order:
// every wave's reads of a place end before the meeting that the loads into it follow, reads of what they bring come behind the
// next one, and meet() lets no access to memory past it.  Nothing else in these kernels uses m0 (tests/test_compiled_kernels.py).
__device__ __forceinline__ void load_to_lds(const char *src, unsigned lds)
{
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(src) : "m0");
}

// A workgroup has WN x WM waves of NTW x MTW tiles of 16 x 16 results.  A step is 128 bytes of K, in two halves.  A wave multiplies one half out of registers while it reads the next into others.  The workgroup meets once a step,
// between the halves: by then every wave has read the whole step, and the next one has arrived; another one is loaded into the
// place that came free.  LDS holds STAGES steps.
// Measured: bf16 gated 4096 x 4096 x 8192 382 - 411 us (1338 - 1439 TFLOP/s; by card and clock: other boxes took up to 453), of which
// the results are 40 us and loads that miss L2 another 40; s8 4096 x 4096 x 4096 58 us (2370 TOPS).
// ALIGNED: rows of activations at multiples of 16 bytes and a whole number of 16-byte parts in K, so they go straight into LDS
// like the weights; else through registers.
template <int TYPE, int NTW, int MTW, int WN, int WM, int STAGES, bool ALIGNED>
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
  const int total = a.blocks_m * a.blocks_n, per_xcd = (total + 7) / 8, number = a.first + (int)blockIdx.x;
  const int index = (number & 7) * per_xcd + (number >> 3);
  if (number >> 3 >= per_xcd || index >= total) return;
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
  // 8 lanes have the 128 bytes of a row, so that a load is whole lines; the 16-byte parts of row r change places by r % 8, so that
  // the 8 rows that are read at a time lie in different banks
  const int part = (lane & 7) ^ (lane >> 3);
  const char *xsrc[2 * XL];
#pragma unroll
  for (int i = 0; i < 2 * XL; ++i) {
    const long long p = blk.first + (wave * XL * 2 + i) * 8 + (lane >> 3);
    xsrc[i] = a.x + row_of(a, p < blk.last ? p : blk.last - 1).in * a.ldx + part * 16;
  }
  const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
  const int steps = a.chunks >> 1;
  const int wn = wave % WN, wm = wave / WN;
  const char *wlds = lds + wn * NTW * 2048 + lane * 16, *xlds = lds + (BN + wm * MTW) * 2048 + c * 128;
  const int xpart = (g ^ (c & 7)) * 16;   // (of the second half: the same, 64 bytes away)

  // the j-th of the wave's loads of a step
  constexpr int LOADS = ALIGNED ? 2 * (WL + XL) : 2 * WL;
  auto load = [&](int j, int step, int stage) {
    const int i = j >> 1, h = j & 1;
    const unsigned to = base + stage * STAGE + h * 1024;
    if (i < WL) {
      load_to_lds(wsrc[i < WL ? i : 0] + (long long)step * 2048 + h * 1024, to + (wave * WL + i) * 2048);
    } else {
      const int x = j - 2 * WL, at = step * 128;
      load_to_lds(at + part * 16 < a.kbytes ? xsrc[x < 2 * XL ? x : 0] + at : a.zeros, base + stage * STAGE + (BN + wave * XL) * 2048 + x * 1024);
    }
  };
  i4 xr[2 * XL];
  auto fetch = [&](int step) {
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < 2 * XL; ++i) xr[i] = load_part<P::elem>(xsrc[i] + step * 128, a.kbytes - step * 128 - part * 16);
    }
  };
  auto put = [&](int stage) {
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < 2 * XL; ++i) *reinterpret_cast<i4 *>(lds + stage * STAGE + (BN + wave * XL) * 2048 + i * 1024 + lane * 16) = xr[i];
    }
  };

  Acc acc[NTW][MTW];
#pragma unroll
  for (int n = 0; n < NTW; ++n)
#pragma unroll
    for (int m = 0; m < MTW; ++m) acc[n][m] = Acc{0, 0, 0, 0};
  i4 wq[2][NTW], xq[2][MTW];   // the operands of the two halves

  auto read = [&](int j, int stage, int h) {   // the j-th of a half's operands
    if (j < MTW) xq[h][j < MTW ? j : 0] = *reinterpret_cast<const i4 *>(xlds + stage * STAGE + j * 2048 + (xpart ^ (h * 64)));
    else if (j < MTW + NTW) wq[h][j - MTW < NTW ? j - MTW : 0] = *reinterpret_cast<const i4 *>(wlds + stage * STAGE + (j - MTW) * 2048 + h * 1024);
  };
  // the products of half h, between them the reads of the other half (of step `from`) and, behind the meeting, loads
  auto half = [&](int h, int from, int step, bool loads) {
    constexpr int PER = (LOADS + NTW - 1) / NTW;
#pragma unroll
    for (int n = 0; n < NTW; ++n) {
      if (loads) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (n * PER + j < LOADS) load(n * PER + j, step, step % STAGES);
      }
      read(2 * n, from % STAGES, h ^ 1);
      read(2 * n + 1, from % STAGES, h ^ 1);
#pragma unroll
      for (int m = 0; m < MTW; ++m) acc[n][m] = P::mma(wq[h][n], xq[h][m], acc[n][m]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // every wave is done with what came before, and all of its loads but the youngest `flying` have arrived
  auto meet = [&](auto flying) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(flying.value) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
  };

  static_assert(ALIGNED || STAGES == 2, "through registers, a step is a stage ahead");
#pragma unroll
  for (int st = 0; st < STAGES; ++st)
    if (st < steps) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) load(j, st, st);
      fetch(st);
      put(st);
    }
  if (steps >= STAGES) meet(Const<(STAGES - 1) * LOADS * ALIGNED>());
  else meet(Const<0>());
#pragma unroll
  for (int j = 0; j < MTW + NTW; ++j) read(j, 0, 0);
  int step = 0;
  for (; step + STAGES < steps; ++step) {
    fetch(step + STAGES);
    half(0, step, 0, false);
    meet(Const<(STAGES - 2) * LOADS>());
    put(step % STAGES);
    half(1, step + 1, step + STAGES, true);
  }
  for (; step < steps; ++step) {
    half(0, step, 0, false);
    meet(Const<0>());
    half(1, step + 1, 0, false);
  }

  // The results go through LDS, 16 rows of every wave at a time, and come back as runs of 8 columns a thread: a wave then has
  // whole rows of results beside each other in memory.
  constexpr int ROW = BN * 64 + 16, THREADS = WAVES * 64;   // bytes of a row: its last 16 keep rows off each other's banks
  static_assert(WM * 16 * ROW <= STAGES * STAGE, "16 rows of every wave fit");
  for_epilogue(a, [&](auto act, auto type, auto gated) {
    constexpr bool GATED = gated.value;
    constexpr int SIZE = type.value == EHIP_F32 ? 4 : 2;
    constexpr int UNITS = GATED ? BN : 2 * BN, HIGH = THREADS / UNITS;   // runs of 8 results in a row; rows at a time
    static_assert(HIGH % 16 == 0 && WM * 16 % HIGH == 0, "a thread's rows are a multiple of 16 apart");
    const int unit = threadIdx.x % UNITS, row0 = threadIdx.x / UNITS;
    // packed rows of the run: those of its first 4 columns and of the next 4 (gated: of the gates; the partners are 16 behind)
    const int tile = bn * BN + (GATED ? unit / 4 : unit / 8) * 4;
    const int col = GATED ? (tile >> 2) * 32 + unit % 4 * 8 : (tile >> 2) * 64 + unit % 8 * 8;
    const bool live = tile < a.tiles && col < a.oc;
    const long long at = ((long long)blk.expert * a.tiles + (live ? tile : 0)) * 16 + (GATED ? unit % 4 * 4 : unit % 2 * 32 + unit % 8 / 2 * 4);
    f4 ws[2][1 + GATED], bias[2][1 + GATED];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int t = 0; t <= GATED; ++t) {
        if (a.wscale) ws[q][t] = *reinterpret_cast<const f4 *>(a.wscale + at + q * (GATED ? 32 : 16) + t * 16);
        if (a.bias) bias[q][t] = *reinterpret_cast<const f4 *>(a.bias + at + q * (GATED ? 32 : 16) + t * 16);
      }
    // (a run's columns are 32 bytes of f32 in LDS; gated: the 32 gates of a group of 64 come before their partners)
    const char *from = lds + row0 * ROW + (GATED ? unit / 4 * 256 + unit % 4 * 32 : unit * 32);
    char *to = lds + (wm * 16 + c) * ROW + (GATED ? g * 32 : g * 64);
    auto write = [&](auto mc) {
#pragma unroll
      for (int n = 0; n < NTW; ++n) {
        const int t = wn * NTW + n;
        *reinterpret_cast<Acc *>(to + t / 4 * 256 + (GATED ? t % 2 * 128 + t % 4 / 2 * 16 : t % 4 * 16)) = acc[n][mc.value];
      }
    };
    constexpr int RUNS = WM * 16 / HIGH;   // rows of a thread in a pass
    auto row_at = [&](int k, int m) {
      const long long p = blk.first + ((row0 / 16 + k * (HIGH / 16)) * MTW + m) * 16 + row0 % 16;
      return live && p < blk.last ? row_of(a, p) : RowOf{0, 0, false};
    };
    // whole runs of the residual are on their way while the results before them cross LDS
    typedef unsigned Old __attribute__((ext_vector_type(2 * SIZE), aligned(2)));
    Old old[RUNS];
    const bool early = a.res && a.oc - col >= 8;
    auto fetch_old = [&](int m) {
      if (!early) return;
#pragma unroll
      for (int k = 0; k < RUNS; ++k) {
        const RowOf row = row_at(k, m);
        if (row.there) old[k] = *reinterpret_cast<const Old *>(a.res + row.out * a.ldr + (long long)col * SIZE);
      }
    };
    auto read = [&](int m) {
#pragma unroll
      for (int k = 0; k < RUNS; ++k) {
        const RowOf row = row_at(k, m);
        if (!row.there) continue;
        const float xs = a.xscale ? a.xscale[row.in] : 1.0f;
        float v[1 + GATED][8];
#pragma unroll
        for (int t = 0; t <= GATED; ++t)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const Acc s = *reinterpret_cast<const Acc *>(from + k * HIGH * ROW + t * 128 + q * 16);
            f4 f = {(float)s[0], (float)s[1], (float)s[2], (float)s[3]};
            if (a.wscale) f *= xs * ws[q][t];
            if (a.bias) f += bias[q][t];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[t][4 * q + j] = f[j];
          }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[0][j] = activate<act.value, type.value>(v[0][j]);
          if (GATED) v[0][j] *= v[GATED][j];
        }
        if (early) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            float lo, hi;
            if (SIZE == 4) {
              const unsigned a0 = old[k][j], a1 = old[k][j + 1];
              lo = __builtin_bit_cast(float, a0);
              hi = __builtin_bit_cast(float, a1);
            } else {
              unpack(old[k][j / 2], type.value == EHIP_BF16, lo, hi);
            }
            v[0][j] = __builtin_fmaf(a.res_scale, lo, v[0][j]);
            v[0][j + 1] = __builtin_fmaf(a.res_scale, hi, v[0][j + 1]);
          }
        }
        store_columns<type.value, 8>(v[0], a.out + row.out * a.ldo + (long long)col * SIZE,
                                     a.res && !early ? a.res + row.out * a.ldr + (long long)col * SIZE : nullptr, a.res_scale, a.oc - col);
      }
    };
    auto pass = [&](auto mc) {
      __syncthreads();
      write(mc);
      __syncthreads();
      read(mc.value);
      if (mc.value + 1 < MTW) fetch_old(mc.value + 1);
    };
    static_assert(MTW == 4, "four passes");
    fetch_old(0);
    pass(Const<0>());
    pass(Const<1>());
    pass(Const<2>());
    pass(Const<3>());
  });
}

namespace {

template <int TYPE, int NTW, int MTW, int WN, int WM, int STAGES>
hipError_t run(LinearArgs a, long long blocks_m, hipStream_t s)
{
  const long long n = (a.tiles + NTW * WN - 1) / (NTW * WN), all = (blocks_m * n + 7) / 8 * 8;
  if (all >= 1ll << 31) return hipErrorInvalidValue;
  a.blocks_m = (int)blocks_m;
  a.blocks_n = (int)n;
  const bool aligned = ((uintptr_t)a.x | (unsigned long long)a.ldx | (unsigned)a.kbytes) % 16 == 0;
  const int lds = (NTW * WN + MTW * WM) * 2048 * (aligned ? STAGES : 2);
  auto kernel = aligned ? k_linear_tile<TYPE, NTW, MTW, WN, WM, STAGES, true> : k_linear_tile<TYPE, NTW, MTW, WN, WM, 2, false>;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  return launch_pieces(all, WN * WM * 64, [&](long long first, unsigned count) {
    a.first = (int)first;
    hipLaunchKernelGGL(kernel, dim3(count), dim3(WN * WM * 64), lds, s, a);
  });
}

}  // namespace

template <int TYPE>
hipError_t run_linear_tile(const LinearArgs &a, int form, long long blocks_m, hipStream_t s)
{
  if (form == 0) return run<TYPE, 4, 4, 2, 2, 2>(a, blocks_m, s);
  if (form == 1) return run<TYPE, 4, 4, 2, 2, 4>(a, blocks_m, s);
  return run<TYPE, 8, 4, 2, 4, 2>(a, blocks_m, s);
}

}  // namespace ehip
