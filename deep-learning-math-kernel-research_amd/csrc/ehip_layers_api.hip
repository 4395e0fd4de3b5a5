// C-ABI of the layers between convolutions (include/euler_hip.h): checks, packed weights, launches.  No kernels here.
#include <new>
#include <string>

#include "ehip_internal.hpp"
#include "ehip_layers.hpp"

using namespace ehip;

struct ehip_linear {
  ehip_linear_desc_t d;
  int elem = 0, tiles = 0, chunks = 0;
  int form = -1;   // EHIP_LINEAR_FORM: forces a kernel form (a gated product needs one with an even number of tiles)
  char *packed = nullptr;   // weights, and behind them the scales, the bias and 256 bytes of zeros
  float *scale = nullptr, *bias = nullptr;
  char *zeros = nullptr;
  bool prepared = false;
};
struct ehip_norm {
  ehip_norm_desc_t d;
};
struct ehip_route {
  ehip_route_desc_t d;
};

namespace {

int fail(int code, const char *msg)
{
  set_error(msg);
  return code;
}

// No exception leaves a C entry
template <typename F>
int guarded(F f)
{
  try {
    return f();
  } catch (...) {
    return EHIP_GENERAL_ERROR;
  }
}

#define LAYER_TRY(expr)                                                                            \
  do {                                                                                             \
    const hipError_t _e = (expr);                                                                  \
    if (_e != hipSuccess) {                                                                        \
      set_error(std::string(#expr) + ": " + hipGetErrorString(_e));                                \
      return EHIP_HIP_ERROR;                                                                       \
    }                                                                                              \
  } while (0)

constexpr int64_t kMaxRows = 1ll << 31, kMaxStride = 1ll << 32;

bool float_type(int t) { return t == EHIP_F32 || t == EHIP_F16 || t == EHIP_BF16; }
int size_of(int t) { return t == EHIP_F32 ? 4 : t == EHIP_S8 ? 1 : 2; }
bool flag(int v) { return v == 0 || v == 1; }
bool aligned(const void *p, int size) { return (uintptr_t)p % (unsigned)size == 0; }

// a stride in bytes; false: shorter than a row, or out of range
bool stride(int64_t given, int64_t cols, int size, long long *bytes)
{
  if (given == 0) given = cols;
  if (given < cols || given > kMaxStride) return false;
  *bytes = given * size;
  return true;
}

int linear_check(const ehip_linear_desc_t &d)
{
  if (d.ic < 1 || d.oc < 1 || d.ic > 1 << 24 || d.oc > 1 << 24) return fail(EHIP_GENERAL_ERROR, "linear: ic and oc are 1 .. 2^24");
  if (d.experts < 1 || d.experts > 1024) return fail(EHIP_GENERAL_ERROR, "linear: experts are 1 .. 1024");
  if (d.input_type != EHIP_F16 && d.input_type != EHIP_BF16 && d.input_type != EHIP_S8)
    return fail(EHIP_UNIMPLEMENTED, "linear: input f16, bf16 or s8");
  if (!float_type(d.output_type)) return fail(EHIP_UNIMPLEMENTED, "linear: output f32, f16 or bf16");
  if (d.activation < EHIP_ACT_NONE || d.activation > EHIP_ACT_SILU) return fail(EHIP_UNIMPLEMENTED, "linear: unknown activation");
  if (!flag(d.gated) || !flag(d.with_bias) || !flag(d.with_residual)) return fail(EHIP_GENERAL_ERROR, "linear: flags are 0 or 1");
  if (d.experts > 1 && d.with_residual) return fail(EHIP_UNIMPLEMENTED, "linear: no residual with experts");
  if (d.input_type == EHIP_S8 && d.ic > 131071) return fail(EHIP_UNIMPLEMENTED, "linear: s8 sums of more than 131071 products");
  return EHIP_OK;
}

// what the handle has for every call
LinearArgs constant_args(const ehip_linear *h)
{
  const ehip_linear_desc_t &d = h->d;
  LinearArgs a = {};
  a.w = h->packed;
  a.wscale = d.input_type == EHIP_S8 ? h->scale : nullptr;
  a.bias = d.with_bias ? h->bias : nullptr;
  a.zeros = h->zeros;
  a.oc = d.oc;
  a.kbytes = d.ic * h->elem;
  a.tiles = h->tiles;
  a.chunks = h->chunks;
  a.experts = d.experts;
  a.out_type = d.output_type;
  a.act = d.activation;
  a.gated = d.gated;
  a.res_scale = d.residual_scale;
  a.form = h->form;
  return a;
}

// what both executes check; fills the kernel's arguments
int linear_args(const ehip_linear *h, const ehip_linear_args_t &g, LinearArgs *a)
{
  const ehip_linear_desc_t &d = h->d;
  if (!h->prepared) return fail(EHIP_GENERAL_ERROR, "linear: not prepared");
  if (g.rows < 0 || g.rows >= kMaxRows) return fail(EHIP_GENERAL_ERROR, "linear: rows out of range");
  *a = constant_args(h);
  const int osize = size_of(d.output_type);
  if (!stride(g.input_stride, d.ic, h->elem, &a->ldx) || !stride(g.output_stride, d.oc, osize, &a->ldo) ||
      !stride(g.residual_stride, d.oc, osize, &a->ldr))
    return fail(EHIP_GENERAL_ERROR, "linear: a stride is shorter than a row or out of range");
  // what the descriptor has no place for would be left out without a word
  if (g.residual_dev && !d.with_residual) return fail(EHIP_GENERAL_ERROR, "linear: a residual, but not with_residual");
  if (g.input_scale_dev && d.input_type != EHIP_S8) return fail(EHIP_GENERAL_ERROR, "linear: input scales are for s8 rows");
  if (g.rows > 0) {
    if (!g.output_dev || !g.input_dev || (d.input_type == EHIP_S8 && !g.input_scale_dev) || (d.with_residual && !g.residual_dev))
      return fail(EHIP_GENERAL_ERROR, "linear: null argument");
    if (!aligned(g.output_dev, osize) || !aligned(g.input_dev, h->elem) || !aligned(g.residual_dev, osize) || !aligned(g.input_scale_dev, 4))
      return fail(EHIP_GENERAL_ERROR, "linear: an address is not a multiple of its elements' size");
  }
  a->x = static_cast<const char *>(g.input_dev);
  a->xscale = d.input_type == EHIP_S8 ? g.input_scale_dev : nullptr;
  a->out = static_cast<char *>(g.output_dev);
  a->res = d.with_residual ? static_cast<const char *>(g.residual_dev) : nullptr;
  a->rows = g.rows;
  return EHIP_OK;
}

}  // namespace

extern "C" {

EHIP_API int ehip_linear_create(const ehip_linear_desc_t *desc, ehip_linear_t **out)
{
  return guarded([&]() -> int {
    if (!desc || !out) return fail(EHIP_GENERAL_ERROR, "null argument");
    *out = nullptr;
    const int rc = linear_check(*desc);
    if (rc != EHIP_OK) return rc;
    ehip_linear *h = new (std::nothrow) ehip_linear;
    if (!h) return fail(EHIP_GENERAL_ERROR, "out of host memory");
    h->d = *desc;
    h->elem = size_of(desc->input_type);
    if (const char *env = getenv("EHIP_LINEAR_FORM")) h->form = atoi(env);
    h->tiles = desc->gated ? (desc->oc + 31) / 32 * 4 : (desc->oc + 63) / 64 * 4;
    h->chunks = (int)(((int64_t)desc->ic * h->elem + 127) / 128 * 2);
    const size_t blocks = (size_t)desc->experts * h->tiles * h->chunks, constants = (size_t)desc->experts * h->tiles * 16 * 4;
    if (blocks >= (size_t)1 << 33) {   // 8 TiB: more than a card holds
      delete h;
      return fail(EHIP_UNIMPLEMENTED, "linear: the weights are too large");
    }
    const hipError_t e = hipMalloc(reinterpret_cast<void **>(&h->packed), blocks * 1024 + 2 * constants + 256);
    if (e != hipSuccess) {
      (void)hipGetLastError();
      delete h;
      set_error(std::string("linear: hipMalloc: ") + hipGetErrorString(e));
      return EHIP_HIP_ERROR;
    }
    h->scale = reinterpret_cast<float *>(h->packed + blocks * 1024);
    h->bias = reinterpret_cast<float *>(h->packed + blocks * 1024 + constants);
    h->zeros = h->packed + blocks * 1024 + 2 * constants;
    *out = h;
    return EHIP_OK;
  });
}

EHIP_API int ehip_linear_destroy(ehip_linear_t *h)
{
  if (!h) return EHIP_OK;
  (void)hipFree(h->packed);
  delete h;
  return EHIP_OK;
}

EHIP_API int ehip_linear_prepare(ehip_linear_t *h, const void *weights_dev, const float *scale_dev, const float *bias_dev, void *hip_stream)
{
  return guarded([&]() -> int {
    if (!h || !weights_dev) return fail(EHIP_GENERAL_ERROR, "null argument");
    const ehip_linear_desc_t &d = h->d;
    if (d.input_type == EHIP_S8 && !scale_dev) return fail(EHIP_GENERAL_ERROR, "linear: s8 weights come with a scale per row");
    if (d.with_bias && !bias_dev) return fail(EHIP_GENERAL_ERROR, "linear: with_bias, but no bias");
    if (d.input_type != EHIP_S8 && scale_dev) return fail(EHIP_GENERAL_ERROR, "linear: scales are for s8 weights");
    if (!d.with_bias && bias_dev) return fail(EHIP_GENERAL_ERROR, "linear: a bias, but not with_bias");
    if (!aligned(weights_dev, h->elem) || !aligned(scale_dev, 4) || !aligned(bias_dev, 4))
      return fail(EHIP_GENERAL_ERROR, "linear: an address is not a multiple of its elements' size");
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    LAYER_TRY(launch_linear_pack(h->packed, weights_dev, d.experts, d.oc, d.ic, h->elem, d.gated, h->tiles, h->chunks, h->zeros, s));
    if (d.input_type == EHIP_S8) LAYER_TRY(launch_linear_constants(h->scale, scale_dev, d.experts, d.oc, d.gated, h->tiles, s));
    if (d.with_bias) LAYER_TRY(launch_linear_constants(h->bias, bias_dev, d.experts, d.oc, d.gated, h->tiles, s));
    h->prepared = true;
    return EHIP_OK;
  });
}

EHIP_API int ehip_linear_execute(const ehip_linear_t *h, const ehip_linear_args_t *args, void *hip_stream)
{
  return guarded([&]() -> int {
    if (!h || !args) return fail(EHIP_GENERAL_ERROR, "null argument");
    if (h->d.experts != 1) return fail(EHIP_GENERAL_ERROR, "linear: a handle of experts is executed with their offsets");
    if (args->slots_dev || args->offsets_dev) return fail(EHIP_GENERAL_ERROR, "linear: slots and offsets are for ehip_linear_execute_experts");
    LinearArgs a;
    const int rc = linear_args(h, *args, &a);
    if (rc != EHIP_OK || args->rows == 0) return rc;
    LAYER_TRY(launch_linear(a, h->d.input_type, static_cast<hipStream_t>(hip_stream)));
    return EHIP_OK;
  });
}

EHIP_API int ehip_linear_execute_experts(const ehip_linear_t *h, const ehip_linear_args_t *args, void *hip_stream)
{
  return guarded([&]() -> int {
    if (!h || !args) return fail(EHIP_GENERAL_ERROR, "null argument");
    const ehip_linear_args_t &g = *args;
    if (h->d.with_residual) return fail(EHIP_UNIMPLEMENTED, "linear: no residual with experts");
    if (g.topk < 1 || g.rows % g.topk) return fail(EHIP_GENERAL_ERROR, "linear: rows are tokens * topk");
    if (g.input_rows < EHIP_ROWS_SORTED || g.input_rows > EHIP_ROWS_SLOT || (g.output_rows != EHIP_ROWS_SORTED && g.output_rows != EHIP_ROWS_SLOT))
      return fail(EHIP_GENERAL_ERROR, "linear: input rows sorted, by token or by slot; output rows sorted or by slot");
    LinearArgs a;
    const int rc = linear_args(h, g, &a);
    if (rc != EHIP_OK || g.rows == 0) return rc;
    if (!g.slots_dev || !g.offsets_dev) return fail(EHIP_GENERAL_ERROR, "linear: null argument");
    if (!aligned(g.slots_dev, 4) || !aligned(g.offsets_dev, 4))
      return fail(EHIP_GENERAL_ERROR, "linear: an address is not a multiple of its elements' size");
    if (g.rows >= 1 << 30) return fail(EHIP_UNIMPLEMENTED, "linear: 2^30 slots and more");
    a.slots = g.slots_dev;
    a.offsets = g.offsets_dev;
    a.topk = g.topk;
    a.in_rows = g.input_rows;
    a.out_rows = g.output_rows;
    LAYER_TRY(launch_linear(a, h->d.input_type, static_cast<hipStream_t>(hip_stream)));
    return EHIP_OK;
  });
}

EHIP_API const char *ehip_linear_kernel_name(const ehip_linear_t *h, int64_t rows)
{
  if (!h || rows < 1 || rows >= kMaxRows) return "";
  LinearArgs a = constant_args(h);
  a.rows = rows;
  // (of these only whether there are any is asked)
  static const int32_t none = 0;
  if (h->d.experts > 1) a.offsets = &none;
  if (h->d.with_residual) a.res = h->packed;
  return linear_kernel_name(a);
}

EHIP_API int ehip_norm_create(const ehip_norm_desc_t *desc, ehip_norm_t **out)
{
  return guarded([&]() -> int {
    if (!desc || !out) return fail(EHIP_GENERAL_ERROR, "null argument");
    *out = nullptr;
    const ehip_norm_desc_t &d = *desc;
    if (d.cols < 1 || d.parts < 1 || d.rows_per_gate < 0) return fail(EHIP_GENERAL_ERROR, "norm: cols and parts are positive, rows_per_gate is not negative");
    if (d.cols > 65536 || d.parts > 64) return fail(EHIP_UNIMPLEMENTED, "norm: more than 65536 columns or 64 parts");
    if (!float_type(d.data_type)) return fail(EHIP_UNIMPLEMENTED, "norm: data f32, f16 or bf16");
    if (d.output_type != d.data_type && d.output_type != EHIP_S8) return fail(EHIP_UNIMPLEMENTED, "norm: output of the data's type or s8");
    if (d.post < EHIP_NORM_NONE || d.post > EHIP_NORM_LAYER || d.pre < EHIP_NORM_NONE || d.pre > EHIP_NORM_LAYER)
      return fail(EHIP_UNIMPLEMENTED, "norm: unknown kind of norm");
    if (!(d.post_eps >= 0.0f) || !(d.pre_eps >= 0.0f)) return fail(EHIP_GENERAL_ERROR, "norm: eps is not negative");
    ehip_norm *h = new (std::nothrow) ehip_norm;
    if (!h) return fail(EHIP_GENERAL_ERROR, "out of host memory");
    h->d = d;
    *out = h;
    return EHIP_OK;
  });
}

EHIP_API int ehip_norm_destroy(ehip_norm_t *h)
{
  delete h;
  return EHIP_OK;
}

EHIP_API int ehip_norm_execute(const ehip_norm_t *h, const ehip_norm_args_t *args, void *hip_stream)
{
  return guarded([&]() -> int {
    if (!h || !args) return fail(EHIP_GENERAL_ERROR, "null argument");
    const ehip_norm_desc_t &d = h->d;
    const ehip_norm_args_t &g = *args;
    const int size = size_of(d.data_type), osize = size_of(d.output_type);
    NormArgs a = {};
    if (g.rows < 0 || g.rows >= kMaxRows) return fail(EHIP_GENERAL_ERROR, "norm: rows out of range");
    if (!stride(g.output_stride, d.cols, osize, &a.ldo) || !stride(g.sum_stride, d.cols, size, &a.lds) ||
        !stride(g.block_stride, d.cols, size, &a.ldb) || !stride(g.residual_stride, d.cols, size, &a.ldr) ||
        !stride(g.gate_stride, d.cols, size, &a.ldg))
      return fail(EHIP_GENERAL_ERROR, "norm: a stride is shorter than a row or out of range");
    if (g.output_scale_dev && d.output_type != EHIP_S8) return fail(EHIP_GENERAL_ERROR, "norm: output scales are for s8 rows");
    if (g.rows == 0) return EHIP_OK;
    if (!g.block_dev || (!g.output_dev && !g.sum_dev) || (d.parts > 1 && !g.part_weights_dev) ||
        (d.output_type == EHIP_S8 && g.output_dev && !g.output_scale_dev))
      return fail(EHIP_GENERAL_ERROR, "norm: null argument");
    if (!aligned(g.output_dev, osize) || !aligned(g.sum_dev, size) || !aligned(g.block_dev, size) || !aligned(g.residual_dev, size) ||
        !aligned(g.gate_dev, size) || !aligned(g.output_scale_dev, 4) || !aligned(g.part_weights_dev, 4) || !aligned(g.post_weight_dev, 4) ||
        !aligned(g.post_bias_dev, 4) || !aligned(g.pre_weight_dev, 4) || !aligned(g.pre_bias_dev, 4))
      return fail(EHIP_GENERAL_ERROR, "norm: an address is not a multiple of its elements' size");
    a.out = static_cast<char *>(g.output_dev);
    a.out_scale = g.output_scale_dev;
    a.sum = static_cast<char *>(g.sum_dev);
    a.block = static_cast<const char *>(g.block_dev);
    a.res = static_cast<const char *>(g.residual_dev);
    a.gate = static_cast<const char *>(g.gate_dev);
    a.pw = g.part_weights_dev;
    a.w1 = g.post_weight_dev;
    a.b1 = g.post_bias_dev;
    a.w2 = g.pre_weight_dev;
    a.b2 = g.pre_bias_dev;
    a.rows = g.rows;
    a.cols = d.cols;
    a.parts = d.parts;
    a.post = d.post;
    a.pre = d.pre;
    a.rows_per_gate = d.rows_per_gate;
    a.block_scale = d.block_scale;
    a.res_scale = d.residual_scale;
    a.eps1 = d.post_eps;
    a.eps2 = d.pre_eps;
    LAYER_TRY(launch_norm(a, d.data_type, d.output_type == EHIP_S8, static_cast<hipStream_t>(hip_stream)));
    return EHIP_OK;
  });
}

EHIP_API int ehip_route_create(const ehip_route_desc_t *desc, ehip_route_t **out)
{
  return guarded([&]() -> int {
    if (!desc || !out) return fail(EHIP_GENERAL_ERROR, "null argument");
    *out = nullptr;
    const ehip_route_desc_t &d = *desc;
    if (d.experts < 1 || d.topk < 1 || d.topk > d.experts) return fail(EHIP_GENERAL_ERROR, "route: topk is 1 .. experts");
    if (d.experts > 1024 || d.topk > 32 || d.groups > 64) return fail(EHIP_UNIMPLEMENTED, "route: more than 1024 experts, 32 choices or 64 groups");
    if (d.groups < 1 || d.experts % d.groups || d.open_groups < 1 || d.open_groups > d.groups)
      return fail(EHIP_GENERAL_ERROR, "route: groups divide the experts, open_groups is 1 .. groups");
    if (d.group_best != 1 && d.group_best != 2) return fail(EHIP_UNIMPLEMENTED, "route: group_best is 1 or 2");
    if (!float_type(d.logits_type)) return fail(EHIP_UNIMPLEMENTED, "route: logits f32, f16 or bf16");
    if (d.score != EHIP_SCORE_SOFTMAX && d.score != EHIP_SCORE_SIGMOID) return fail(EHIP_UNIMPLEMENTED, "route: unknown score");
    if (!flag(d.renormalize)) return fail(EHIP_GENERAL_ERROR, "route: flags are 0 or 1");
    ehip_route *h = new (std::nothrow) ehip_route;
    if (!h) return fail(EHIP_GENERAL_ERROR, "out of host memory");
    h->d = d;
    *out = h;
    return EHIP_OK;
  });
}

EHIP_API int ehip_route_destroy(ehip_route_t *h)
{
  delete h;
  return EHIP_OK;
}

EHIP_API int64_t ehip_route_plan_ints(const ehip_route_t *h, int64_t tokens)
{
  if (!h || tokens < 0 || tokens > kRouteTokens || tokens * h->d.topk >= 1ll << 30) return -1;
  const int64_t kept = tokens > kRouteBlock ? (1 + (tokens + kRouteBlock - 1) / kRouteBlock) * h->d.experts : 0;
  return h->d.experts + 1 + tokens * h->d.topk + kept;
}

EHIP_API int ehip_route_execute(const ehip_route_t *h, const ehip_route_args_t *args, void *hip_stream)
{
  return guarded([&]() -> int {
    if (!h || !args) return fail(EHIP_GENERAL_ERROR, "null argument");
    const ehip_route_desc_t &d = h->d;
    const ehip_route_args_t &g = *args;
    const int size = size_of(d.logits_type);
    RouteArgs a = {};
    if (ehip_route_plan_ints(h, g.tokens) < 0) return fail(EHIP_GENERAL_ERROR, "route: tokens out of range");
    if (!stride(g.logits_stride, d.experts, size, &a.ld)) return fail(EHIP_GENERAL_ERROR, "route: a stride is shorter than a row or out of range");
    if (g.tokens > 0 && (!g.ids_dev || !g.weights_dev || !g.logits_dev)) return fail(EHIP_GENERAL_ERROR, "route: null argument");
    if (!aligned(g.ids_dev, 4) || !aligned(g.weights_dev, 4) || !aligned(g.plan_dev, 4) || !aligned(g.bias_dev, 4) || !aligned(g.logits_dev, size))
      return fail(EHIP_GENERAL_ERROR, "route: an address is not a multiple of its elements' size");
    if (g.tokens == 0 && !g.plan_dev) return EHIP_OK;
    a.ids = g.ids_dev;
    a.weights = g.weights_dev;
    if (g.plan_dev) {
      a.offsets = g.plan_dev;
      a.slots = a.offsets + d.experts + 1;
      a.totals = a.slots + g.tokens * d.topk;
      a.hist = a.totals + d.experts;
    }
    a.logits = static_cast<const char *>(g.logits_dev);
    a.bias = g.bias_dev;
    a.tokens = g.tokens;
    a.experts = d.experts;
    a.topk = d.topk;
    a.groups = d.groups;
    a.open = d.open_groups;
    a.best = d.group_best;
    a.sigmoid = d.score == EHIP_SCORE_SIGMOID;
    a.renorm = d.renormalize;
    a.scale = d.scale;
    LAYER_TRY(launch_route(a, d.logits_type, static_cast<hipStream_t>(hip_stream)));
    return EHIP_OK;
  });
}

}  // extern "C"
