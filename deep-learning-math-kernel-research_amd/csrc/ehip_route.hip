// The experts of each token, and the order of their work.
//
// A wave has a token, its lanes the experts in runs of PER.  Every score is the definition's single-precision value: exp, the
// sum over the experts in 64 bits (so that its order cannot show), one division; a choice is the largest key, by a maximum over
// the wave, of the lowest expert that has it.  The slots of an expert keep the order of the tokens: workgroups count theirs,
// and a second kernel places each behind those of the workgroups before it.  A few tokens take one workgroup and one launch.
#include "ehip_layers.hpp"

namespace ehip {
namespace {

constexpr float kClosed = -__builtin_inff();

__device__ __forceinline__ float max_over_wave(float v)
{
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

// One token: lane j < topk returns its j-th choice (-1: none) and that choice's weight
template <int TYPE, int PER>
__device__ __forceinline__ void choose(const RouteArgs &a, long long token, float *keys, int *id_out, float *weight_out)
{
  const int lane = threadIdx.x & 63, first = lane * PER;
  constexpr int size = TYPE == EHIP_F32 ? 4 : 2;
  const char *row = a.logits + token * a.ld + (long long)first * size;
  float x[PER], score[PER], key[PER];
  float top = kClosed;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    x[j] = kClosed;
    if (first + j < a.experts) x[j] = load_one(row + j * size, TYPE);
    if (!(x[j] > kClosed)) x[j] = kClosed;   // a NaN
    x[j] = fminf(x[j], 3.402823466e38f);
    top = fmaxf(top, x[j]);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] = 1.0f / (1.0f + expf(-x[j]));
  } else {
    top = max_over_wave(top);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      score[j] = x[j] > kClosed ? expf(x[j] - top) : 0.0f;
      sum += (double)score[j];
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    const float all = (float)sum;
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] /= all;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    key[j] = kClosed;
    if (x[j] > kClosed) {
      key[j] = a.bias ? score[j] + a.bias[first + j] : score[j];
      if (key[j] != key[j]) key[j] = kClosed;
    }
  }

  if (a.open < a.groups) {
    // the best one or two keys of each group: 64 / (groups rounded up to a power of two) lanes look through one
    const int size_g = a.experts / a.groups;
    int lanes = 64;
    while (lanes * a.groups > 64) lanes >>= 1;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (first + j < a.experts) keys[first + j] = key[j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int mine = lane / lanes;
    float b1 = kClosed, b2 = kClosed;
    if (mine < a.groups)
      for (int i = lane % lanes; i < size_g; i += lanes) {
        const float k = keys[mine * size_g + i];
        b2 = fmaxf(b2, fminf(b1, k));
        b1 = fmaxf(b1, k);
      }
    for (int d = 1; d < lanes; d <<= 1) {
      const float o1 = __shfl_xor(b1, d), o2 = __shfl_xor(b2, d);
      b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
      b1 = fmaxf(b1, o1);
    }
    const float total = a.best > 1 && b2 > kClosed ? b1 + b2 : b1;
    int better = 0;
    for (int q = 0; q < a.groups; ++q) {
      const float other = __shfl(total, q * lanes);
      better += other > total || (other == total && q < mine);
    }
    const unsigned long long open = __ballot(better < a.open && mine < a.groups);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (the next token's keys come after these reads)
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (first + j < a.experts && !((open >> ((first + j) / size_g * lanes)) & 1)) key[j] = kClosed;
  }

  int id = -1;
  float weight = 0.0f, total = 0.0f;
  for (int k = 0; k < a.topk; ++k) {
    float best = key[0], its = score[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < PER; ++j)
      if (key[j] > best) {
        best = key[j];
        its = score[j];
        at = j;
      }
    const float m = max_over_wave(best);
    if (!(m > kClosed)) break;
    const int who = __builtin_ctzll(__ballot(best == m));
    const float w = __shfl(its, who);
    const int e = who * PER + __shfl(at, who);
    total += w;
    if (lane == k) {
      id = e;
      weight = w;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (lane == who && j == at) key[j] = kClosed;
  }
  if (a.renorm) weight = total > 0.0f ? weight / total : 0.0f;
  *id_out = id;
  *weight_out = weight * a.scale;
}

// a workgroup has kRouteBlock tokens and counts the slots of each expert among them
template <int TYPE, int PER>
__global__ __launch_bounds__(512) void k_route_choose(RouteArgs a)
{
  constexpr int WAVES = 8;
  __shared__ float keys[WAVES][64 * PER];
  __shared__ int count[64 * PER];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int e = threadIdx.x; e < a.experts; e += 512) count[e] = 0;
  __syncthreads();
  const long long from = (long long)blockIdx.x * kRouteBlock, to = from + kRouteBlock < a.tokens ? from + kRouteBlock : a.tokens;
  for (long long t = from + wave; t < to; t += WAVES) {
    int id;
    float w;
    choose<TYPE, PER>(a, t, keys[wave], &id, &w);
    if (lane < a.topk) {
      a.ids[t * a.topk + lane] = id;
      a.weights[t * a.topk + lane] = w;
      if (id >= 0) atomicAdd(&count[id], 1);
    }
  }
  if (!a.hist) return;
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += 512) a.hist[(long long)blockIdx.x * a.experts + e] = count[e];
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
    const int n = e0 + lane < experts ? total[e0 + lane] : 0;
    int sum = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int t = __shfl_up(sum, d);
      if (lane >= d) sum += t;
    }
    if (e0 + lane < experts) first[e0 + lane] = before + sum - n;
    before += __shfl(sum, 63);
  }
  return before;
}

__global__ __launch_bounds__(512) void k_route_place(RouteArgs a, int blocks)
{
  __shared__ int total[1024], next[1024], first[1024], all;
  for (int e = threadIdx.x; e < a.experts; e += 512) {
    int sum = 0, before = 0;
    for (int b = 0; b < blocks; ++b) {
      const int n = a.hist[(long long)b * a.experts + e];
      before += b < (int)blockIdx.x ? n : 0;
      sum += n;
    }
    total[e] = sum;
    next[e] = before;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int n = sum_up(total, first, a.experts);
    if (threadIdx.x == 0) all = n;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += 512) {
    next[e] += first[e];
    if (blockIdx.x == 0) a.offsets[e] = first[e];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[a.experts] = all;
  __syncthreads();
  const long long from = (long long)blockIdx.x * kRouteBlock * a.topk, end = a.tokens * a.topk;
  const int count = (int)(end - from < (long long)kRouteBlock * a.topk ? end - from : (long long)kRouteBlock * a.topk);
  if (threadIdx.x < 64) place(a, a.ids + from, from, count, next);
  // behind the last expert's: none.  Every workgroup has its share of the places that could be left
  for (long long i = from + threadIdx.x; i < from + count; i += 512)
    if (i >= all) a.slots[i] = -1;
}

// at most kRouteBlock tokens: one workgroup does it all
template <int TYPE, int PER>
__global__ __launch_bounds__(1024) void k_route_few(RouteArgs a)
{
  constexpr int WAVES = 16;
  __shared__ float keys[WAVES][64 * PER];
  __shared__ int count[64 * PER], next[64 * PER], ids[kRouteBlock * 32], all;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int e = threadIdx.x; e < a.experts; e += 1024) count[e] = 0;
  __syncthreads();
  for (int t = wave; t < a.tokens; t += WAVES) {
    int id;
    float w;
    choose<TYPE, PER>(a, t, keys[wave], &id, &w);
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
  hipLaunchKernelGGL((k_route_choose<TYPE, PER>), dim3(blocks), dim3(512), 0, s, a);
  if (a.offsets) hipLaunchKernelGGL(k_route_place, dim3(blocks), dim3(512), 0, s, a, (int)blocks);
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
