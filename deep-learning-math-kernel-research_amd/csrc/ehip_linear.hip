// Products of rows of activations with a matrix (or with the matrices of the experts they are sent to), few rows: the K
// axis shared out among the waves of a workgroup, operands straight from memory to registers.  Also the packing of the
// weights, and the choice between this kernel and the one that stages tiles in LDS (ehip_linear_tile.hpp).
#include "ehip_layers.hpp"

namespace ehip {

// ---- packing -----------------------------------------------------------------------------------------------------
// source row of row i of a tile: see LinearArgs
__device__ __forceinline__ int packed_source(int tile, int i, int oc, int gated, bool *real)
{
  const int t = tile & 3, group = tile >> 2;
  const int col = gated ? group * 32 + 8 * (i >> 2) + 4 * (t >> 1) + (i & 3) : group * 64 + 16 * (i >> 2) + 4 * t + (i & 3);
  *real = col < oc;
  return gated && (t & 1) ? oc + col : col;
}

template <int ELEM>
__global__ void k_linear_pack(char *packed, const char *w, int oc, int ic, int gated, int tiles, int chunks, long long units,
                              char *zeros, long long first)
{
  const long long u = (first + blockIdx.x) * blockDim.x + threadIdx.x;
  if (u < 16) reinterpret_cast<i4 *>(zeros)[u] = i4{0, 0, 0, 0};
  if (u >= units) return;
  const int lane = (int)(u & 63);
  const long long block = u >> 6, row_block = block / chunks;
  const int chunk = (int)(block % chunks), tile = (int)(row_block % tiles);
  const long long expert = row_block / tiles;
  bool real;
  const int src = packed_source(tile, lane & 15, oc, gated, &real);
  const int at = chunk * 64 + (lane >> 4) * 16, valid = real ? ic * ELEM - at : 0;
  const long long row = expert * (gated ? 2 * oc : oc) + (real ? src : 0);
  *reinterpret_cast<i4 *>(packed + u * 16) = load_part<ELEM>(w + row * ic * ELEM + at, valid);
}

__global__ void k_linear_constants(float *dst, const float *src, int oc, int gated, int tiles, long long count)
{
  const long long u = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (u >= count) return;
  const long long row_block = u >> 4;
  bool real;
  const int at = packed_source((int)(row_block % tiles), (int)(u & 15), oc, gated, &real);
  dst[u] = real ? src[row_block / tiles * (gated ? 2 * oc : oc) + at] : 0.0f;
}

hipError_t launch_linear_pack(void *packed, const void *weights, int experts, int oc, int ic, int elem, int gated, int tiles, int chunks,
                              char *zeros, hipStream_t s)
{
  const long long units = (long long)experts * tiles * chunks * 64;
  auto kernel = elem == 1 ? k_linear_pack<1> : k_linear_pack<2>;
  return launch_pieces((units + 255) / 256, 256, [&](long long first, unsigned count) {
    hipLaunchKernelGGL(kernel, dim3(count), dim3(256), 0, s, static_cast<char *>(packed), static_cast<const char *>(weights), oc, ic, gated,
                       tiles, chunks, units, zeros, first);
  });
}

hipError_t launch_linear_constants(float *dst, const float *src, int experts, int oc, int gated, int tiles, hipStream_t s)
{
  const long long count = (long long)experts * tiles * 16;
  hipLaunchKernelGGL(k_linear_constants, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, s, dst, src, oc, gated, tiles, count);
  return hipGetLastError();
}

// ---- few rows ----------------------------------------------------------------------------------------------------
// A workgroup has NT tiles of 16 weights rows x MT tiles of 16 activations rows; its waves share K out in runs of steps of 128
// bytes, so a workgroup reads no weight twice and they stream past as runs of KBs, straight into registers, P steps ahead.  Activations
// come by whole lines, 8 lanes a row, and change lanes through a corner of LDS that is the wave's own (a load that gave every
// lane the 16 bytes that its matrix operand has would be 64 accesses instead of 16, and the loads bound these kernels).  The
// waves' sums meet in LDS, in the order of the waves.
// Measured, weights out of memory (out of the memory-side cache): bf16 1 x 4096 x 4096 8.4 us, 4.0 TB/s of weights (5.2 us); s8 gated
// 16 x 4096 x 8192 15.4 us, 4.4 TB/s (12.3); 64 slots of 32 experts of 2048 x 2816 57 us, 5.7 TB/s (51); f16 64 x 2048 x 1000 (4.0).
// Weights' bytes bound it up to some 16 rows, then the loads:
// 64 x 64 results of 64 steps take a CU 11 us, twice what their products do.
template <int TYPE, int NT, int MT, int P>
__global__ __launch_bounds__(512) void k_linear_split(LinearArgs a)
{
  typedef Product<TYPE> Pr;
  typedef typename Pr::Acc Acc;
  constexpr int WAVES = 8;
  constexpr int ROOM = MT * 2048 > NT * MT * 1024 ? MT * 2048 : NT * MT * 1024;   // bytes of LDS a wave
  __shared__ i4 lds[WAVES * ROOM / 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;

  // blocks of the same weights beside each other on one XCD: its L2 holds them for all
  const int per_xcd = (a.blocks_m * a.blocks_n + 7) / 8, number = a.first + (int)blockIdx.x;
  const int index = (number & 7) * per_xcd + (number >> 3);
  if (number >> 3 >= per_xcd || index >= a.blocks_m * a.blocks_n) return;
  const int bn = index / a.blocks_m;
  const Block blk = block_of(a, index - bn * a.blocks_m, 16 * MT);
  if (blk.expert < 0) return;

  // the 16-byte part of row r that a lane loads changes places by r % 8: the 8 rows that are read at a time lie in different banks
  const int part = (lane & 7) ^ (lane >> 3);
  const char *xp[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    const long long p = blk.first + i * 8 + (lane >> 3);
    xp[i] = a.x + row_of(a, p < blk.last ? p : blk.last - 1).in * a.ldx + part * 16;
  }
  const int tile0 = bn * NT;
  const long long tile_bytes = (long long)a.chunks * 1024;
  const char *wp = a.w + ((long long)blk.expert * a.tiles + tile0) * tile_bytes;
  const unsigned wl = lane * 16;
  i4 *own = lds + wave * (ROOM / 16);
  const int xread = c * 8 + (g ^ (c & 7));   // (of the second half: the same, 4 parts away)

  const int full = a.kbytes >> 7, per = (full + WAVES - 1) / WAVES;
  const int k0 = wave * per, k1 = k0 + per < full ? k0 + per : full;

  Acc acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = Acc{0, 0, 0, 0};

  i4 wr[P][2 * NT], xr[P][2 * MT];
  auto load = [&](int slot, int k) {
#pragma unroll
    for (int n = 0; n < 2 * NT; ++n)
      wr[slot][n] = *reinterpret_cast<const i4 *>(wp + (n >> 1) * tile_bytes + (long long)k * 2048 + (n & 1) * 1024 + wl);
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) xr[slot][i] = *reinterpret_cast<const i4u *>(xp[i] + (long long)k * 128);
    __builtin_amdgcn_sched_barrier(0);   // (loads stay behind the products that free their registers)
  };
  auto multiply = [&](const i4 (&w)[2 * NT], const i4 (&x)[2 * MT]) {
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) own[i * 64 + lane] = x[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i4 xq[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) xq[m] = own[m * 128 + (xread ^ (h * 4))];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[n][m] = Pr::mma(w[2 * n + h], xq[m], acc[n][m]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_sched_barrier(0);
  };
  if (k0 < k1) {
    // steps past the wave's last repeat it (they come from cache, and nobody waits for them)
#pragma unroll
    for (int s = 0; s < P; ++s) load(s, k0 + s < k1 ? k0 + s : k1 - 1);
    int k = k0;
    for (; k + P < k1; k += P)
#pragma unroll
      for (int s = 0; s < P; ++s) {
        multiply(wr[s], xr[s]);
        load(s, k + s + P < k1 ? k + s + P : k1 - 1);
      }
#pragma unroll
    for (int s = 0; s < P; ++s)
      if (k + s < k1) multiply(wr[s], xr[s]);
  }
  if (wave == WAVES - 1 && (a.kbytes & 127)) {   // the last step, of which a part exists
    i4 w[2 * NT], x[2 * MT];
#pragma unroll
    for (int n = 0; n < 2 * NT; ++n)
      w[n] = *reinterpret_cast<const i4 *>(wp + (n >> 1) * tile_bytes + (long long)full * 2048 + (n & 1) * 1024 + wl);
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) x[i] = load_part<Pr::elem>(xp[i] + (long long)full * 128, (a.kbytes & 127) - part * 16);
    multiply(w, x);
  }

  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) own[(n * MT + m) * 64 + lane] = __builtin_bit_cast(i4, acc[n][m]);
  __syncthreads();

  auto total = [&](int n, int m) {
    Acc s = __builtin_bit_cast(Acc, lds[(n * MT + m) * 64 + lane]);
#pragma unroll
    for (int v = 1; v < WAVES; ++v) s += __builtin_bit_cast(Acc, lds[v * (ROOM / 16) + (n * MT + m) * 64 + lane]);
    return s;
  };
  constexpr int PAIRS = NT > 1 ? NT / 2 : 1;
  for_epilogue(a, [&](auto act, auto type, auto gated) {
    constexpr int UNITS = (gated.value ? PAIRS : NT) * MT, SIZE = type.value == EHIP_F32 ? 4 : 2;
    for (int i = wave; i < UNITS; i += WAVES) {
      const int m = i % MT, n = i / MT;
      const long long p = blk.first + m * 16 + c;
      if (p >= blk.last) continue;
      const RowOf row = row_of(a, p);
      if (!row.there) continue;
      const float xs = a.xscale ? a.xscale[row.in] : 1.0f;
      float v[4];
      int col;
      if constexpr (gated.value) {
        const int tile = tile0 + 2 * n;
        const long long at = ((long long)blk.expert * a.tiles + tile) * 16 + g * 4;
        const f4 gate = finish_sums(a, total(2 * n, m), at, xs);
        const f4 up = finish_sums(a, total(NT > 1 ? 2 * n + 1 : 0, m), at + 16, xs);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = activate<act.value, type.value>(gate[r]) * up[r];
        col = (tile >> 2) * 32 + g * 8 + ((tile & 3) >> 1) * 4;
      } else {
        const int tile = tile0 + n;
        const f4 t = finish_sums(a, total(n, m), ((long long)blk.expert * a.tiles + tile) * 16 + g * 4, xs);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = activate<act.value, type.value>(t[r]);
        col = (tile >> 2) * 64 + g * 16 + (tile & 3) * 4;
      }
      store_columns<type.value, 4>(v, a.out + row.out * a.ldo + (long long)col * SIZE,
                                   a.res ? a.res + row.out * a.ldr + (long long)col * SIZE : nullptr, a.res_scale, a.oc - col);
    }
  });
}

namespace {

// blocks of `rows` positions: the experts' last blocks are partly empty, at most one each
long long blocks_of(const LinearArgs &a, int rows)
{
  if (!a.offsets) return (a.rows + rows - 1) / rows;
  return a.rows / rows + (a.rows < a.experts ? a.rows : a.experts);
}

template <int TYPE, int NT, int MT, int P>
hipError_t run_split(LinearArgs a, hipStream_t s)
{
  const long long m = blocks_of(a, 16 * MT), n = a.tiles / NT, all = (m * n + 7) / 8 * 8;
  if (all >= 1ll << 31) return hipErrorInvalidValue;
  a.blocks_m = (int)m;
  a.blocks_n = (int)n;
  return launch_pieces(all, 512, [&](long long first, unsigned count) {
    a.first = (int)first;
    hipLaunchKernelGGL((k_linear_split<TYPE, NT, MT, P>), dim3(count), dim3(512), 0, s, a);
  });
}

enum Form { SPLIT_1X1, SPLIT_2X1, SPLIT_4X1, SPLIT_2X2, SPLIT_4X2, SPLIT_4X4, TILE_128, TILE_128_DEEP, TILE_256, FORMS };

// What a form takes, in us, from what it measured on an idle card (bf16, f16 and s8 alike: a step is 128 bytes of K, and so are
// its loads and its matrix instructions).  All forms: no faster than the bytes at 5.2 TB/s; what is hidden behind those is
// not hidden whole.  Sweeps of 1 - 4096 rows, K 512 - 8192 bytes, 1024 - 8192 columns, and of experts with 1 - 770 rows each: the
// form with the least sum is the fastest one or within 15 % of it, in the worst case found 27 % (256 rows, bf16 512 -> 1024: 5.2 us
// for 4.1).  What it does not know: that each block of rows reads the weights again (32 rows, bf16 4096 x 4096: 9.7 for
// 7.8), and that rows at addresses that are no multiple of 16 bytes are slower to load (s8 1024 x 4097 x 2000: 39 for 31).
struct FormCost {
  int nt, mt;          // tiles of a workgroup's results
  int resident;        // workgroups of a CU
  double start, round, step;   // once; for each time that the workgroups fill the card; for a step of one workgroup of a CU
};
constexpr FormCost kForms[FORMS] = {
    // few rows: 0.019 us a tile of operands and step, which is what its loads take a CU (16 cycles a KB)
    {1, 1, 2, 1.5, 1.2, 0.038}, {2, 1, 2, 1.5, 1.7, 0.057}, {4, 1, 1, 1.5, 2.1, 0.095}, {2, 2, 1, 1.5, 2.1, 0.076},
    {4, 2, 1, 1.5, 2.4, 0.114}, {4, 4, 1, 1.5, 3.9, 0.17},
    // 128 x 128: two workgroups of a CU with two steps in LDS (64 steps of 512 workgroups 64 us, of 256 42), or one with four (35)
    {8, 8, 2, 0.0, 5.0, 0.47}, {8, 8, 1, 0.0, 5.0, 0.47},
    // 256 x 256: 64 steps of 256 workgroups 101 us, of 128 76 (the clock is higher)
    {16, 16, 1, 0.0, 10.0, 1.42}};

double cost(const LinearArgs &a, Form form)
{
  const FormCost &f = kForms[form];
  const double rows = (double)a.rows, high = 16.0 * f.mt, n = (a.tiles + f.nt - 1) / f.nt, steps = (a.kbytes + 127) / 128;
  double m = (double)((a.rows + 16 * f.mt - 1) / (16 * f.mt)), matrices = 1;
  if (a.offsets) {   // each expert's last block is half empty
    matrices = rows < a.experts ? rows : a.experts;
    const double each = rows / matrices / high + 0.5;
    m = matrices * (each > 1 ? each : 1);
  }
  const double groups = m * n, fill = 256.0 * f.resident;
  const double bytes = matrices * a.tiles * 16.0 * a.kbytes + rows * (a.kbytes + a.oc * (a.out_type == EHIP_F32 ? 4.0 : 2.0) * (a.res ? 2 : 1));
  const double memory = bytes / 5.2e6;
  double work;
  if (form < TILE_128) {
    work = (double)(long long)((groups + 255) / 256) * steps * f.step;
    return f.start + (double)(long long)((groups + fill - 1) / fill) * f.round + (work > memory ? work + 0.3 * memory : memory + 0.3 * work);
  }
  const double whole = (double)(long long)(groups / fill), left = groups - whole * fill;
  if (form == TILE_256) work = whole * (f.round + f.step * steps) + (left > 0 ? f.round + (1.0 + 0.42 * left / fill) * steps : 0);
  else if (form == TILE_128) work = whole * (f.round + 2 * f.step * steps) + (left > 0 ? f.round + (left > 256 ? 2 * f.step : 0.58) * steps : 0);
  else work = (whole + (left > 0)) * (f.round + f.step * steps);
  return work > 1.2 * memory + f.round ? work : 1.2 * memory + f.round;
}

Form choose(const LinearArgs &a)
{
  const bool odd = a.gated;   // a gate and its partner are two tiles
  if (a.form >= 0 && a.form < FORMS && !(odd && a.form == SPLIT_1X1)) return (Form)a.form;
  int best = odd ? SPLIT_2X1 : SPLIT_1X1;
  double least = cost(a, (Form)best);
  for (int f = best + 1; f < FORMS; ++f) {
    const double c = cost(a, (Form)f);
    if (c < least) {
      least = c;
      best = f;
    }
  }
  return (Form)best;
}

template <int TYPE>
hipError_t launch_typed(const LinearArgs &a, hipStream_t s)
{
  auto tile = TYPE == EHIP_BF16 ? launch_linear_tile_bf16 : TYPE == EHIP_F16 ? launch_linear_tile_f16 : launch_linear_tile_s8;
  switch (choose(a)) {
  case SPLIT_1X1: return run_split<TYPE, 1, 1, 4>(a, s);
  case SPLIT_2X1: return run_split<TYPE, 2, 1, 4>(a, s);
  case SPLIT_4X1: return run_split<TYPE, 4, 1, 3>(a, s);
  case SPLIT_2X2: return run_split<TYPE, 2, 2, 3>(a, s);
  case SPLIT_4X2: return run_split<TYPE, 4, 2, 2>(a, s);
  case SPLIT_4X4: return run_split<TYPE, 4, 4, 2>(a, s);
  case TILE_128: return tile(a, 0, blocks_of(a, 128), s);
  case TILE_128_DEEP: return tile(a, 1, blocks_of(a, 128), s);
  default: return tile(a, 2, blocks_of(a, 256), s);
  }
}

}  // namespace

hipError_t launch_linear(const LinearArgs &a, int type, hipStream_t s)
{
  switch (type) {
  case EHIP_BF16: return launch_typed<EHIP_BF16>(a, s);
  case EHIP_F16: return launch_typed<EHIP_F16>(a, s);
  default: return launch_typed<EHIP_S8>(a, s);
  }
}

const char *linear_kernel_name(const LinearArgs &a)
{
  static const char *const names[FORMS] = {"k_linear_split<1x1>", "k_linear_split<2x1>", "k_linear_split<4x1>", "k_linear_split<2x2>",
                                           "k_linear_split<4x2>", "k_linear_split<4x4>", "k_linear_tile<128x128>",
                                           "k_linear_tile<128x128, deep>", "k_linear_tile<256x256>"};
  const Form form = choose(a);
  // rows that end at other bytes pass through registers, and there both 128 x 128 forms are one kernel
  return names[form == TILE_128_DEEP && a.kbytes % 16 ? TILE_128 : form];
}

}  // namespace ehip
