// The experts of each token, and the order of their work.
//
// A wave has a token, its lanes the experts in runs of PER.  Every score is the definition's single-precision value: exp, the
// sum over the experts in 64 bits (so that its order cannot show), one division.  A lane sorts its keys once; a choice is the
// largest of the lanes' first ones, by the lowest lane that has it, which goes on to its next.  Reductions over the lanes are
// cross-lane operands of vector instructions: through LDS each of their steps would cost its latency, 99 us where this takes
// 42 (32768 tokens, 256 experts in 8 groups, 8 choices), bounded by 590 vector instructions a token.
// The slots of an expert keep the order of the tokens: workgroups count theirs, a kernel sums the counts over the workgroups
// before each, a third places the slots.  A few tokens take one workgroup and one launch.
#include <type_traits>

#include "ehip_layers.hpp"

namespace ehip {
namespace {

constexpr float kClosed = -__builtin_inff();

// Keys are compared as integers of the same order (a zero has no sign): one instruction each, where a maximum of floats takes
// three to keep a signalling NaN quiet.
__device__ __forceinline__ int ordered(float v)
{
  const int b = __builtin_bit_cast(int, v + 0.0f);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int k) { return __builtin_bit_cast(float, k ^ ((k >> 31) & 0x7fffffff)); }
constexpr int kClosedKey = (int)0x807fffff;   // ordered(-inf)
__device__ __forceinline__ int imax(int a, int b) { return a > b ? a : b; }
__device__ __forceinline__ int imin(int a, int b) { return a < b ? a : b; }

// the maximum over the wave, in every lane (a scalar)
__device__ __forceinline__ int max_over_wave(int v)
{
  constexpr int least = (int)0x80000000;   // (with it the step is one instruction)
  v = imax(v, dpp<kShr1>(least, v));
  v = imax(v, dpp<kShr2>(least, v));
  v = imax(v, dpp<kShr4>(least, v));
  v = imax(v, dpp<kShr8>(least, v));
  v = imax(v, dpp<kBcast15, 0xa>(least, v));
  v = imax(v, dpp<kBcast31, 0xc>(least, v));
  return __builtin_amdgcn_readlane(v, 63);
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double plus(double v)
{
  const long long b = __builtin_bit_cast(long long, v);
  const int lo = dpp<CTRL, ROWS>(0, (int)b), hi = dpp<CTRL, ROWS>(0, (int)(b >> 32));
  return v + __builtin_bit_cast(double, (long long)(unsigned)lo | ((long long)hi << 32));
}
__device__ __forceinline__ double sum_over_wave(double v)
{
  v = plus<kShr1>(v);
  v = plus<kShr2>(v);
  v = plus<kShr4>(v);
  v = plus<kShr8>(v);
  v = plus<kBcast15, 0xa>(v);
  v = plus<kBcast31, 0xc>(v);
  const long long b = __builtin_bit_cast(long long, v);
  const int lo = __builtin_amdgcn_readlane((int)b, 63), hi = __builtin_amdgcn_readlane((int)(b >> 32), 63);
  return __builtin_bit_cast(double, (long long)(unsigned)lo | ((long long)hi << 32));
}

template <int TYPE, int PER>
__device__ __forceinline__ void load_logits(const RouteArgs &a, long long token, float (&x)[PER])
{
  constexpr int size = TYPE == EHIP_F32 ? 4 : 2;
  const int first = (threadIdx.x & 63) * PER;
  const char *row = a.logits + token * a.ld + (long long)first * size;
  if (first + PER <= a.experts) {
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = load_one(row + j * size, TYPE);
    return;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) x[j] = first + j < a.experts ? load_one(row + j * size, TYPE) : kClosed;
}

// What is the same for every token: the bias of the lane's experts (0 where there is none), and how the groups lie over a wave: 64 / (groups rounded up to a power of two) lanes look through one
template <int PER> struct Fixed {
  float bias[PER];
  int size, lanes, mine;
  bool own;             // each lane's keys are of the group that it looks through
  unsigned char at[PER];   // lane that speaks for the group of each of the lane's experts
};
template <int PER>
__device__ __forceinline__ Fixed<PER> fixed_of(const RouteArgs &a)
{
  Fixed<PER> g;
  const int lane = threadIdx.x & 63;
  g.size = a.experts / a.groups;
  g.lanes = 64;
  while (g.lanes * a.groups > 64) g.lanes >>= 1;
  g.mine = lane / g.lanes;
  g.own = g.lanes * PER == g.size;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane * PER + j;
    g.bias[j] = a.bias && e < a.experts ? a.bias[e] : 0.0f;
    g.at[j] = (unsigned char)(e < a.experts ? e / g.size * g.lanes : 0);
  }
  return g;
}

// the two largest of two pairs
__device__ __forceinline__ void join(int &b1, int &b2, int o1, int o2)
{
  b2 = imax(imin(b1, o1), imax(b2, o2));
  b1 = imax(b1, o1);
}

// One token from its logits: lane j < topk returns its j-th choice (-1: none) and that choice's weight.  room: of the wave
template <int PER>
__device__ __forceinline__ void choose(const RouteArgs &a, const Fixed<PER> &g, float (&x)[PER], float *room, int *id_out, float *weight_out)
{
  const int lane = threadIdx.x & 63, first = lane * PER;
  float score[PER];
  int key[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    x[j] = x[j] > kClosed ? +x[j] : kClosed;   // a NaN is closed, too
    x[j] = x[j] < 3.402823466e38f ? +x[j] : 3.402823466e38f;
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] = 1.0f / (1.0f + expf(-x[j]));
  } else {
    int most = ordered(x[0]);
#pragma unroll
    for (int j = 1; j < PER; ++j) most = imax(most, ordered(x[j]));
    const float top = unordered(max_over_wave(most));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      score[j] = x[j] > kClosed ? expf(x[j] - top) : 0.0f;
      sum += (double)score[j];
    }
    const float all = (float)sum_over_wave(sum);
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] /= all;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const float k = score[j] + g.bias[j];
    key[j] = x[j] > kClosed && k == k ? ordered(k) : kClosedKey;
  }

  if (a.open < a.groups) {
    // the best one or two keys of each group
    int b1, b2 = kClosedKey;
    if (g.own) {
      b1 = key[0];
#pragma unroll
      for (int j = 1; j < PER; ++j) join(b1, b2, key[j], kClosedKey);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) room[first + j] = __builtin_bit_cast(float, key[j]);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      b1 = kClosedKey;
      if (g.mine < a.groups)
        for (int i = lane % g.lanes; i < g.size; i += g.lanes) join(b1, b2, __builtin_bit_cast(int, room[g.mine * g.size + i]), kClosedKey);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (what is written into the room next comes after these reads)
    }
    // lanes 1, 2, 4, 8 away: swaps in a quad, mirrors of 8 and 16 (whose halves agree in themselves by then)
    if (g.lanes > 1) join(b1, b2, dpp<0xb1>(b1, b1), dpp<0xb1>(b2, b2));
    if (g.lanes > 2) join(b1, b2, dpp<0x4e>(b1, b1), dpp<0x4e>(b2, b2));
    if (g.lanes > 4) join(b1, b2, dpp<0x141>(b1, b1), dpp<0x141>(b2, b2));
    if (g.lanes > 8) join(b1, b2, dpp<0x140>(b1, b1), dpp<0x140>(b2, b2));
    if (g.lanes > 16) join(b1, b2, __shfl_xor(b1, 16), __shfl_xor(b2, 16));
    if (g.lanes > 32) join(b1, b2, __shfl_xor(b1, 32), __shfl_xor(b2, 32));
    const int total = a.best > 1 && b2 > kClosedKey ? ordered(unordered(b1) + unordered(b2)) : b1;
    int better = 0;
    for (int q = 0; q < a.groups; ++q) {
      const int other = __builtin_amdgcn_readlane(total, q * g.lanes);
      better += other > total || (other == total && q < g.mine) ? 1 : 0;
    }
    const unsigned long long open = __ballot(better < a.open && g.mine < a.groups);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (!((open >> g.at[j]) & 1)) key[j] = kClosedKey;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) room[first + j] = score[j];

  // exchanges of neighbours only, of unequal keys only: equal ones stay in the order of their experts
  int from[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) from[j] = j;
#pragma unroll
  for (int i = 0; i < PER - 1; ++i)
#pragma unroll
    for (int j = PER - 2; j >= i; --j) {
      const bool swap = key[j + 1] > key[j];
      const int k = imin(key[j], key[j + 1]), f = from[j];
      key[j] = imax(key[j], key[j + 1]);
      key[j + 1] = k;
      const int f1 = from[j + 1];
      from[j] = swap ? +f1 : +f;   // (values: a choice between array elements would make them memory)
      from[j + 1] = swap ? +f : +f1;
    }
  // the order as 4 bits an expert
  typedef typename std::conditional<(PER > 8), uint64_t, uint32_t>::type Order;
  Order order = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) order |= (Order)from[j] << (4 * j);

  int id = -1;
  for (int k = 0; k < a.topk; ++k) {
    const int m = max_over_wave(key[0]);
    if (m == kClosedKey) break;
    const int who = __builtin_ctzll(__ballot(key[0] == m));
    const int e = who * PER + __builtin_amdgcn_readlane((int)(order & 15), who);
    id = lane == k ? e : id;
    const bool mine = lane == who;
#pragma unroll
    for (int j = 0; j + 1 < PER; ++j) key[j] = mine ? +key[j + 1] : +key[j];
    key[PER - 1] = mine ? kClosedKey : +key[PER - 1];
    order = mine ? order >> 4 : order;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  float weight = id >= 0 ? room[id] : 0.0f;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (the next token's go there after this)
  if (a.renorm) {
    // up to 32 choices: the first two rows of 16 lanes
    float total = weight;
    total += dpp<kShr1>(0.0f, total);
    total += dpp<kShr2>(0.0f, total);
    total += dpp<kShr4>(0.0f, total);
    total += dpp<kShr8>(0.0f, total);
    const int bits = __builtin_bit_cast(int, total);
    total = __builtin_bit_cast(float, __builtin_amdgcn_readlane(bits, 15)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(bits, 31));
    weight = total > 0.0f ? weight / total : 0.0f;
  }
  *id_out = id;
  *weight_out = weight * a.scale;
}

// a workgroup has kRouteBlock tokens and counts the slots of each expert among them: hist [experts][workgroups]
template <int TYPE, int PER>
__global__ __launch_bounds__(1024) void k_route_choose(RouteArgs a)
{
  constexpr int WAVES = 16;
  __shared__ float room[WAVES][64 * PER];
  __shared__ int count[64 * PER];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int e = threadIdx.x; e < a.experts; e += 64 * WAVES) count[e] = 0;
  __syncthreads();
  const long long from = (long long)blockIdx.x * kRouteBlock, to = from + kRouteBlock < a.tokens ? from + kRouteBlock : a.tokens;
  const Fixed<PER> fixed = fixed_of<PER>(a);
  float x[PER], ahead[PER];
  if (from + wave < to) load_logits<TYPE, PER>(a, from + wave, ahead);
  int32_t *ids = a.ids + (from + wave) * a.topk + lane;
  float *weights = a.weights + (from + wave) * a.topk + lane;
  for (long long t = from + wave; t < to; t += WAVES) {
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = ahead[j];
    if (t + WAVES < to) load_logits<TYPE, PER>(a, t + WAVES, ahead);
    int id;
    float w;
    choose<PER>(a, fixed, x, room[wave], &id, &w);
    if (lane < a.topk) {
      *ids = id;
      *weights = w;
      if (id >= 0) atomicAdd(&count[id], 1);
    }
    ids += WAVES * a.topk;
    weights += WAVES * a.topk;
  }
  if (!a.hist) return;
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += 64 * WAVES) a.hist[(long long)e * gridDim.x + blockIdx.x] = count[e];
}

// sum of v over the lanes before this one; *all: over the wave
__device__ __forceinline__ int sum_before(int v, int *all)
{
  int s = v;
  s += dpp<kShr1>(0, s);
  s += dpp<kShr2>(0, s);
  s += dpp<kShr4>(0, s);
  s += dpp<kShr8>(0, s);
  s += dpp<kBcast15, 0xa>(0, s);
  s += dpp<kBcast31, 0xc>(0, s);
  *all = __builtin_amdgcn_readlane(s, 63);
  return s - v;
}

// one wave an expert: its counts over the workgroups before each, in place, and in totals[expert] all of them
__global__ __launch_bounds__(256) void k_route_sum(RouteArgs a, int blocks)
{
  const int e = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (e >= a.experts) return;
  int32_t *hist = a.hist + (long long)e * blocks;
  int before = 0;
  for (int b0 = 0; b0 < blocks; b0 += 256) {   // four a lane
    int n[4], own = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int b = b0 + lane * 4 + j;
      n[j] = b < blocks ? hist[b] : 0;
      own += n[j];
    }
    int all;
    int at = before + sum_before(own, &all);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int b = b0 + lane * 4 + j;
      if (b < blocks) hist[b] = at;
      at += n[j];
    }
    before += all;
  }
  if (lane == 0) a.totals[e] = before;
}

// 64 slots beside each other in a wave: how many before a lane's have the same expert, and how many have it in all.
// -1 has no expert
__device__ __forceinline__ int rank_in_wave(int id, int bits, int *same)
{
  unsigned long long peers = __ballot(id >= 0);
  for (int b = 0; b < bits; ++b) {
    const unsigned long long set = __ballot((id >> b) & 1);
    peers &= (id >> b) & 1 ? set : ~set;
  }
  *same = __popcll(peers);
  return __popcll(peers & ((1ull << (threadIdx.x & 63)) - 1));
}

// next[e] of the workgroup's first slot of each expert -> the slots of its tokens in place; one wave, in order
__device__ __forceinline__ void place(const RouteArgs &a, const int *ids, long long from, int count, int *next)
{
  const int lane = threadIdx.x & 63, bits = 32 - __builtin_clz(a.experts);
  for (int i = 0; i < count; i += 64) {
    const int id = i + lane < count ? ids[i + lane] : -1;
    int same;
    const int rank = rank_in_wave(id, bits, &same);
    if (id >= 0) {
      const int at = next[id];
      a.slots[at + rank] = (int)(from + i + lane);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (rank == same - 1) next[id] = at + same;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// exclusive sum over the experts of total[] into first[], by the first wave; the count of all comes back to that wave
__device__ __forceinline__ int sum_up(const int *total, int *first, int experts)
{
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    int all;
    const int at = sum_before(e0 + lane < experts ? total[e0 + lane] : 0, &all);
    if (e0 + lane < experts) first[e0 + lane] = before + at;
    before += all;
  }
  return before;
}

// The slots of a workgroup of k_route_choose in their places: four waves, each with a quarter of them, that count first
__global__ __launch_bounds__(256) void k_route_place(RouteArgs a)
{
  __shared__ int first[1024], next[4][1024], all;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long from = (long long)blockIdx.x * kRouteBlock * a.topk, end = a.tokens * a.topk;
  const int count = (int)(end - from < (long long)kRouteBlock * a.topk ? end - from : (long long)kRouteBlock * a.topk);
  const int quarter = (count + 255) / 256 * 64, mine = wave * quarter, to = mine + quarter < count ? mine + quarter : count;
  for (int e = threadIdx.x; e < a.experts; e += 256) {
    first[e] = a.totals[e];
#pragma unroll
    for (int w = 0; w < 4; ++w) next[w][e] = 0;
  }
  __syncthreads();
  for (int i = mine + lane; i < to; i += 64) {
    const int id = a.ids[from + i];
    if (id >= 0) atomicAdd(&next[wave][id], 1);
  }
  if (wave == 0) {
    const int n = sum_up(first, first, a.experts);
    if (lane == 0) all = n;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += 256) {
    if (blockIdx.x == 0) a.offsets[e] = first[e];
    int at = first[e] + a.hist[(long long)e * gridDim.x + blockIdx.x];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int n = next[w][e];
      next[w][e] = at;
      at += n;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[a.experts] = all;
  __syncthreads();
  if (mine < to) place(a, a.ids + from + mine, from + mine, to - mine, next[wave]);
  // behind the last expert's: none.  Every workgroup has its share of the places that could be left
  for (long long i = from + threadIdx.x; i < from + count; i += 256)
    if (i >= all) a.slots[i] = -1;
}

// at most kRouteBlock tokens: one workgroup does it all
template <int TYPE, int PER>
__global__ __launch_bounds__(1024) void k_route_few(RouteArgs a)
{
  constexpr int WAVES = 16;
  __shared__ float room[WAVES][64 * PER];
  __shared__ int count[64 * PER], next[64 * PER], ids[kRouteBlock * 32], all;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int e = threadIdx.x; e < a.experts; e += 1024) count[e] = 0;
  __syncthreads();
  const Fixed<PER> fixed = fixed_of<PER>(a);
  for (int t = wave; t < a.tokens; t += WAVES) {
    int id;
    float w;
    float x[PER];
    load_logits<TYPE, PER>(a, t, x);
    choose<PER>(a, fixed, x, room[wave], &id, &w);
    if (lane < a.topk) {
      a.ids[t * a.topk + lane] = id;
      a.weights[t * a.topk + lane] = w;
      ids[t * a.topk + lane] = id;
      if (id >= 0) atomicAdd(&count[id], 1);
    }
  }
  __syncthreads();
  const int slots = (int)a.tokens * a.topk;
  if (threadIdx.x < 64) {
    const int n = sum_up(count, next, a.experts);
    if (lane == 0) {
      all = n;
      a.offsets[a.experts] = n;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int e = lane; e < a.experts; e += 64) a.offsets[e] = next[e];
    place(a, ids, 0, slots, next);
  }
  __syncthreads();
  for (int i = all + threadIdx.x; i < slots; i += 1024) a.slots[i] = -1;
}

template <int TYPE, int PER>
hipError_t run(const RouteArgs &a, hipStream_t s)
{
  if (a.offsets && a.tokens <= kRouteBlock) {
    hipLaunchKernelGGL((k_route_few<TYPE, PER>), dim3(1), dim3(1024), 0, s, a);
    return hipGetLastError();
  }
  const unsigned blocks = (unsigned)((a.tokens + kRouteBlock - 1) / kRouteBlock);
  hipLaunchKernelGGL((k_route_choose<TYPE, PER>), dim3(blocks), dim3(1024), 0, s, a);
  if (a.offsets) {
    hipLaunchKernelGGL(k_route_sum, dim3((a.experts + 3) / 4), dim3(256), 0, s, a, (int)blocks);
    hipLaunchKernelGGL(k_route_place, dim3(blocks), dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

template <int TYPE>
hipError_t run_type(const RouteArgs &a, hipStream_t s)
{
  if (a.experts <= 64) return run<TYPE, 1>(a, s);
  if (a.experts <= 128) return run<TYPE, 2>(a, s);
  if (a.experts <= 256) return run<TYPE, 4>(a, s);
  if (a.experts <= 512) return run<TYPE, 8>(a, s);
  return run<TYPE, 16>(a, s);
}

}  // namespace

hipError_t launch_route(const RouteArgs &a, int type, hipStream_t s)
{
  switch (type) {
  case EHIP_F32: return run_type<EHIP_F32>(a, s);
  case EHIP_F16: return run_type<EHIP_F16>(a, s);
  default: return run_type<EHIP_BF16>(a, s);
  }
}

}  // namespace ehip
