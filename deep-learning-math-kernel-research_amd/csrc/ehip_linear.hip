// Products of rows of activations with a matrix (or with the matrices of the experts they are sent to), few rows: the K
// axis shared out among the waves of a workgroup, operands straight from memory to registers.  Also the packing of the
// weights, and the choice between this kernel and the one that stages tiles in LDS (ehip_linear_tile.hip).
#include "ehip_layers.hpp"
#include "ehip_linear_tile.hpp"

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
                              char *zeros)
{
  const long long u = (long long)blockIdx.x * blockDim.x + threadIdx.x;
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
  hipLaunchKernelGGL(kernel, dim3((unsigned)((units + 255) / 256)), dim3(256), 0, s, static_cast<char *>(packed),
                     static_cast<const char *>(weights), oc, ic, gated, tiles, chunks, units, zeros);
  return hipGetLastError();
}

hipError_t launch_linear_constants(float *dst, const float *src, int experts, int oc, int gated, int tiles, hipStream_t s)
{
  const long long count = (long long)experts * tiles * 16;
  hipLaunchKernelGGL(k_linear_constants, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, s, dst, src, oc, gated, tiles, count);
  return hipGetLastError();
}

// ---- few rows ----------------------------------------------------------------------------------------------------
// A workgroup has NT tiles of 16 weights rows x MT tiles of 16 activations rows; its waves share K out in runs of chunks, so
// no operand is read twice and the weights stream past as runs of KBs.  U chunks are in flight while U are multiplied.  The
// waves' sums meet in LDS, in the order of the waves.
template <int TYPE, int NT, int MT, int WAVES, int U>
__global__ __launch_bounds__(WAVES * 64) void k_linear_split(LinearArgs a)
{
  typedef Product<TYPE> P;
  typedef typename P::Acc Acc;
  __shared__ Acc red[WAVES][NT * MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;

  // blocks of the same weights beside each other on one XCD: its L2 holds them for all
  const int per_xcd = (a.blocks_m * a.blocks_n + 7) / 8;
  const int index = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
  if (index >= a.blocks_m * a.blocks_n) return;
  const int bn = index / a.blocks_m;
  const Block blk = block_of(a, index - bn * a.blocks_m, 16 * MT);
  if (blk.expert < 0) return;

  const char *xp[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const long long p = blk.first + m * 16 + c;
    xp[m] = a.x + row_of(a, p < blk.last ? p : blk.last - 1).in * a.ldx + g * 16;
  }
  const int tile0 = bn * NT;
  const long long tile_bytes = (long long)a.chunks * 1024;
  const char *wp = a.w + ((long long)blk.expert * a.tiles + tile0) * tile_bytes;
  const unsigned wl = lane * 16;

  const int full = a.kbytes >> 6;
  const int per = (full + WAVES - 1) / WAVES, c0 = wave * per, c1 = c0 + per < full ? c0 + per : full;

  Acc acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = Acc{0, 0, 0, 0};

  auto load = [&](i4 (&wq)[U][NT], i4 (&xq)[U][MT], int at) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = at + u < c1 ? at + u : c1 - 1;
#pragma unroll
      for (int n = 0; n < NT; ++n) wq[u][n] = *reinterpret_cast<const i4 *>(wp + n * tile_bytes + (long long)k * 1024 + wl);
#pragma unroll
      for (int m = 0; m < MT; ++m) xq[u][m] = *reinterpret_cast<const i4u *>(xp[m] + (long long)k * 64);
    }
  };
  auto multiply = [&](i4 (&wq)[U][NT], i4 (&xq)[U][MT], int count) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < count) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[n][m] = P::mma(wq[u][n], xq[u][m], acc[n][m]);
      }
  };
  i4 w0[U][NT], x0[U][MT], w1[U][NT], x1[U][MT];
  if (c0 < c1) load(w0, x0, c0);
  if (wave == WAVES - 1 && (a.kbytes & 63)) {   // the last chunk, of which a part exists
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const i4 w = *reinterpret_cast<const i4 *>(wp + n * tile_bytes + (long long)full * 1024 + wl);
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[n][m] = P::mma(w, load_part<P::elem>(xp[m] + (long long)full * 64, (a.kbytes & 63) - g * 16), acc[n][m]);
    }
  }
  for (int k = c0; k < c1; k += 2 * U) {
    if (k + U < c1) load(w1, x1, k + U);
    multiply(w0, x0, c1 - k);
    if (k + U < c1) {
      if (k + 2 * U < c1) load(w0, x0, k + 2 * U);
      multiply(w1, x1, c1 - k - U);
    }
  }

#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) red[wave][n * MT + m][lane] = acc[n][m];
  __syncthreads();

  auto total = [&](int n, int m) {
    Acc s = red[0][n * MT + m][lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) s += red[v][n * MT + m][lane];
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
        for (int r = 0; r < 4; ++r) v[r] = activate<act.value>(gate[r]) * up[r];
        col = (tile >> 2) * 32 + g * 8 + ((tile & 3) >> 1) * 4;
      } else {
        const int tile = tile0 + n;
        const f4 t = finish_sums(a, total(n, m), ((long long)blk.expert * a.tiles + tile) * 16 + g * 4, xs);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = activate<act.value>(t[r]);
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

template <int TYPE, int NT, int MT, int WAVES, int U>
hipError_t run_split(LinearArgs a, hipStream_t s)
{
  const long long m = blocks_of(a, 16 * MT), n = a.tiles / NT, all = (m * n + 7) / 8 * 8;
  if (all >= 1ll << 31) return hipErrorInvalidValue;
  a.blocks_m = (int)m;
  a.blocks_n = (int)n;
  hipLaunchKernelGGL((k_linear_split<TYPE, NT, MT, WAVES, U>), dim3((unsigned)all), dim3(WAVES * 64), 0, s, a);
  return hipGetLastError();
}

enum Form { SPLIT_1X1, SPLIT_2X1, SPLIT_2X2, SPLIT_4X4, TILE_128, TILE_256 };

Form choose(const LinearArgs &a)
{
  const double rows = a.offsets ? (double)a.rows / a.experts : (double)a.rows;   // of one matrix
  if (rows > 192) return TILE_256;
  if (rows > 32) return SPLIT_4X4;
  if (rows > 16) return SPLIT_2X2;
  return a.gated ? SPLIT_2X1 : SPLIT_1X1;
}

template <int TYPE>
hipError_t launch_typed(const LinearArgs &a, hipStream_t s)
{
  switch (choose(a)) {
  case SPLIT_1X1: return run_split<TYPE, 1, 1, 8, 8>(a, s);
  case SPLIT_2X1: return run_split<TYPE, 2, 1, 8, 6>(a, s);
  case SPLIT_2X2: return run_split<TYPE, 2, 2, 8, 4>(a, s);
  case SPLIT_4X4: return run_split<TYPE, 4, 4, 8, 2>(a, s);
  case TILE_128: return launch_linear_tile(a, TYPE, 0, blocks_of(a, 128), s);
  default: return launch_linear_tile(a, TYPE, 1, blocks_of(a, 256), s);
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

const char *linear_kernel_name(const LinearArgs &a, int)
{
  static const char *const names[] = {"k_linear_split<1x1>", "k_linear_split<2x1>", "k_linear_split<2x2>", "k_linear_split<4x4>",
                                      "k_linear_tile<128x128>", "k_linear_tile<256x256>"};
  return names[choose(a)];
}

}  // namespace ehip
