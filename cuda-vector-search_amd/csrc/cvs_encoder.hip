// C entry points of the text-encoder operators: argument checks, plans, launches.
// As in cvs_capi.hip, nothing here allocates, synchronises or throws.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "cvs.h"
#include "cvs_encoder.h"
#include "cvs_host.h"

using namespace cvs;

namespace {

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int64_t up256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

int gfx950(int device, DevInfo* di) {
  const int rc = dev_info(device, di);
  if (rc != CVS_OK) return rc;
  if (!di->gfx950) return fail(CVS_ERR_INVALID, "libcvs_hip targets gfx950 (MI355X); device %d is %s", device, di->arch);
  return CVS_OK;
}

int check_workspace(const void* ws, int64_t have, int64_t need) {
  if (need > 0 && (ws == nullptr || reinterpret_cast<uintptr_t>(ws) % 256 != 0))
    return fail(CVS_ERR_INVALID, "workspace must be 256-byte aligned");
  if (have < need) return fail(CVS_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)have, (long long)need);
  return CVS_OK;
}

int done(hipError_t e, const char* what) { return e == hipSuccess ? CVS_OK : hip_fail(e, what); }

// ---- layer norm ------------------------------------------------------------------

int check_norm(int64_t n, int64_t d, int type) {
  if (type != CVS_TYPE_F16 && type != CVS_TYPE_BF16 && type != CVS_TYPE_F32)
    return fail(CVS_ERR_INVALID, "layer norm takes float16, bfloat16 or float32");
  if (d < 1 || d > (1 << 24)) return fail(CVS_ERR_INVALID, "layer norm takes widths of 1 to 2^24");
  if (n < 0 || n >= INT_MAX) return fail(CVS_ERR_INVALID, "too many rows");
  return CVS_OK;
}

int64_t norm_ws(int64_t n, int64_t d, int type, int cus) {
  return n == 0 ? 0 : up256((int64_t)norm_backward_parts(n, d, type, cus) * 2 * d * 4);
}

// ---- matrix product ----------------------------------------------------------------

int check_linear(int64_t m, int64_t k, int64_t n) {
  if (m < 0 || m > INT_MAX - 255) return fail(CVS_ERR_INVALID, "too many rows");  // (rows of the last tile count on past m)
  if (k < 8 || n < 8 || k % 8 != 0 || n % 8 != 0)
    return fail(CVS_ERR_INVALID, "linear takes feature counts that are multiples of 8 (zero-pad them)");
  if (k > (1 << 20) || n > (1 << 20)) return fail(CVS_ERR_INVALID, "linear takes at most 2^20 features");
  if (m * std::max(k, n) > ((int64_t)1 << 36)) return fail(CVS_ERR_INVALID, "linear: more than 2^36 values in a matrix");
  return CVS_OK;
}

int check_plan(const GemmPlan& p) {
  return p.splits > 0 ? CVS_OK : fail(CVS_ERR_INVALID, "linear: too many rows and features for a launch");
}

int check_linear_types(int act, int type) {
  if (type != CVS_TYPE_F16 && type != CVS_TYPE_BF16) return fail(CVS_ERR_INVALID, "linear takes float16 or bfloat16");
  if (act < CVS_ACT_NONE || act > CVS_ACT_TANH) return fail(CVS_ERR_INVALID, "unknown activation %d", act);
  return CVS_OK;
}

int check_rows(const void* p, int64_t stride, int64_t width, const char* what) {
  if (!aligned16(p)) return fail(CVS_ERR_INVALID, "%s must be 16-byte aligned", what);
  if (stride < width || stride % 8 != 0 || stride > (1 << 21))
    return fail(CVS_ERR_INVALID, "%s: row stride must be a multiple of 8, at least its width and at most 2^21", what);
  return CVS_OK;
}

struct LinearBackwardPlan {
  GemmPlan dx, dw;
  int parts;
  int64_t dz, partial, gemm, gemm_dw, bytes;  // offsets, then all
};

LinearBackwardPlan plan_linear_backward(int64_t m, int64_t k, int64_t n, int act, int cus) {
  LinearBackwardPlan p;
  p.dx = plan_gemm(m, k, n, cus);
  p.dw = plan_gemm(n, k, m, cus);
  p.parts = act_grad_parts(m, n, cus);
  int64_t at = 0;
  p.dz = at, at += act == CVS_ACT_NONE ? 0 : up256(m * n * 2);
  p.partial = at, at += up256((int64_t)p.parts * n * 4);
  p.gemm = at, at += up256(p.dx.ws_bytes);
  p.gemm_dw = at, at += up256(p.dw.ws_bytes);
  p.bytes = at;
  return p;
}

// ---- gated product -----------------------------------------------------------------

int check_gated_types(int act, int type) {
  if (type != CVS_TYPE_F16 && type != CVS_TYPE_BF16) return fail(CVS_ERR_INVALID, "gated linear takes float16 or bfloat16");
  if (act < CVS_ACT_NONE || act > CVS_ACT_SIGMOID) return fail(CVS_ERR_INVALID, "unknown activation %d", act);
  return CVS_OK;
}

// (twice n values a row: dz, pre)
int check_gated(int64_t m, int64_t k, int64_t n) {
  const int rc = check_linear(m, k, n);
  return rc == CVS_OK && n > (1 << 19) ? fail(CVS_ERR_INVALID, "gated linear takes at most 2^19 output features") : rc;
}

struct GatedBackwardPlan {
  GemmPlan dx, dw, one;  // one: a single weight's gradient
  int parts;
  bool rests;     // dz's rows twice: rounded, and what that took off
  int64_t rows;   // of dz
  int64_t dz, twice, partial, peaks, unit, gemm, bytes;  // offsets, then all
};

GatedBackwardPlan plan_gated_backward(int64_t m, int64_t k, int64_t n, int cus) {
  GatedBackwardPlan p;
  p.rests = gated_few_rows(m);
  p.rows = p.rests ? 2 * m : m;
  p.dx = plan_two_parts(p.rows, k, n, p.rests, cus);
  p.dw = plan_gemm(2 * n, k, p.rows, cus);
  p.one = plan_gemm(n, k, p.rows, cus);
  p.parts = gated_grad_parts(m, n, cus);
  int64_t at = 0;
  p.dz = at, at += up256(2 * p.rows * n * 2);
  p.twice = at, at += p.rests ? up256(p.rows * k * 2) : 0;
  p.partial = at, at += up256((int64_t)p.parts * 2 * n * 4);
  p.peaks = at, at += up256(gated_grad_workgroups(m, n, p.parts) * 4);
  p.unit = at, at += up256(4);
  p.gemm = at, at += up256(std::max({p.dx.ws_bytes, p.dw.ws_bytes, p.one.ws_bytes}));  // (one product after the other)
  p.bytes = at;
  return p;
}

int check_gated_plan(const GatedBackwardPlan& p) {
  int rc = check_plan(p.dx);
  if (rc == CVS_OK) rc = check_plan(p.dw);
  return rc == CVS_OK ? check_plan(p.one) : rc;
}

// ---- 8-bit product -----------------------------------------------------------------

int check_quantize(int64_t n, int64_t d, int type) {
  if (type != CVS_TYPE_F16 && type != CVS_TYPE_BF16) return fail(CVS_ERR_INVALID, "8-bit rows are made of float16 or bfloat16");
  if (n < 0 || n > INT_MAX - 255) return fail(CVS_ERR_INVALID, "too many rows");
  if (d < 16 || d % 16 != 0 || d > (1 << 17))
    return fail(CVS_ERR_INVALID, "8-bit rows have a multiple of 16 values, at most 2^17 (zero-pad them)");
  // (a launch has fewer than 2^32 threads: rows of a wave each, or a workgroup)
  if (n * (d <= 4096 ? 64 : 256) + 256 >= ((int64_t)1 << 32)) return fail(CVS_ERR_INVALID, "too many rows");
  return CVS_OK;
}

int check_int8(int64_t m, int64_t k, int64_t n, int act, int type) {
  int rc = check_quantize(m, k, type);
  if (rc == CVS_OK) rc = check_linear(m, k, n);
  if (rc == CVS_OK) rc = check_linear_types(act, type);
  return rc;
}

struct Int8Plan {
  GemmPlan product;
  bool few;  // one launch, without a workspace
  int64_t values, scales, gemm, bytes;  // offsets, then all
};

Int8Plan plan_linear_int8(int64_t m, int64_t k, int64_t n, int cus) {
  Int8Plan p = {};
  p.product = plan_int8(m, n, k, cus);
  p.few = int8_few_rows(m, n, k, p.product, cus);
  if (p.few) return p;
  int64_t at = 0;
  p.values = at, at += up256(m * k);
  p.scales = at, at += up256(m * 4);
  p.gemm = at, at += up256(p.product.ws_bytes);
  p.bytes = at;
  return p;
}

// ---- attention ---------------------------------------------------------------------

int check_attention(const cvs_attention* p) {
  if (p == nullptr) return fail(CVS_ERR_INVALID, "attention: null arguments");
  if (p->type != CVS_TYPE_F16 && p->type != CVS_TYPE_BF16) return fail(CVS_ERR_INVALID, "attention takes float16 or bfloat16");
  if (p->width < 8 || p->width > 128 || p->width % 8 != 0)
    return fail(CVS_ERR_INVALID, "attention takes head widths that are multiples of 8, at most 128");
  if (p->batch < 0 || p->q_len < 0 || p->k_len < 0 || p->q_len >= (1 << 29) || p->k_len >= (1 << 29))
    return fail(CVS_ERR_INVALID, "attention: bad batch or length");
  if (p->heads < 1 || p->k_heads < 1 || p->heads % p->k_heads != 0)
    return fail(CVS_ERR_INVALID, "attention: query heads must be a multiple of key heads");
  if (p->heads > 65536 || p->batch > INT_MAX / p->heads)
    return fail(CVS_ERR_INVALID, "attention: too many heads");
  for (const int64_t len : {p->q_len, p->k_len})
    if ((len + kAttnRows - 1) / kAttnRows * p->batch * p->heads >= (1 << 23))  // (a launch has fewer than 2^32 threads)
      return fail(CVS_ERR_INVALID, "attention: too many rows");
  // (the kernels hold biases in units of unscaled scores, bias / scale)
  if (!(p->scale >= 0x1p-100 && p->scale <= 0x1p100)) return fail(CVS_ERR_INVALID, "attention: scale must be positive, from 2^-100 to 2^100");
  if (p->bias_table != nullptr) {
    const int64_t one = p->causal ? p->buckets : p->buckets / 2;
    if (p->buckets < 4 || p->buckets > kMaxBuckets || p->buckets % 2 != 0)
      return fail(CVS_ERR_INVALID, "attention: an even number of 4 to %d buckets", kMaxBuckets);
    if (p->max_distance <= one / 2 || p->max_distance > kMaxDistance)
      return fail(CVS_ERR_INVALID, "attention: max_distance must be more than %lld (buckets of one distance) and at most %d",
                  (long long)(one / 2), kMaxDistance);
  }
  return CVS_OK;
}

int check_heads(const void* p, const int64_t* stride, const char* what) {
  if (!aligned16(p)) return fail(CVS_ERR_INVALID, "%s must be 16-byte aligned", what);
  for (int i = 0; i < 3; ++i)
    if (stride[i] < 0 || stride[i] % 8 != 0) return fail(CVS_ERR_INVALID, "%s: strides must be multiples of 8", what);
  if (stride[1] > (1 << 23)) return fail(CVS_ERR_INVALID, "%s: a position's stride must be at most 2^23", what);
  return CVS_OK;
}

// (positions are below 2^28 + 2^29, query_start being brought to +-2^29: every sum of the kernels' fits an int)
int check_window(const cvs_attention* p, const cvs_attention_window* w) {
  if (w == nullptr) return CVS_OK;
  if (w->before < 0 || w->after < 0 || w->sinks < 0) return fail(CVS_ERR_INVALID, "attention: a window's sizes must not be negative");
  if (p->q_len >= (1 << 28) || p->k_len >= (1 << 28)) return fail(CVS_ERR_INVALID, "attention: windows take lengths below 2^28");
  return CVS_OK;
}

AttnArgs attn_args(const cvs_attention* p, const cvs_attention_window* w) {
  AttnArgs a = {};
  a.type = p->type;
  a.batch = (int)p->batch, a.lq = (int)p->q_len, a.lk = (int)p->k_len;
  a.heads = (int)p->heads, a.k_heads = (int)p->k_heads, a.d = (int)p->width;
  a.q = p->q, a.k = p->k, a.v = p->v;
  for (int i = 0; i < 3; ++i) a.qs[i] = p->q_stride[i], a.ks[i] = p->k_stride[i], a.vs[i] = p->v_stride[i];
  a.scale = (float)p->scale;
  a.causal = p->causal != 0;
  a.key_lengths = p->key_lengths, a.query_lengths = p->query_lengths, a.query_start = p->query_start;
  a.table = p->bias_table;
  a.buckets = (int)p->buckets, a.max_distance = (int)p->max_distance;
  a.splits = 1;
  if (w != nullptr) {
    constexpr int64_t kAll = (int64_t)3 << 28;  // no position is further from a key
    a.windowed = 1;
    a.before = (int)std::min(w->before, kAll);
    a.after = a.causal ? 0 : (int)std::min(w->after, kAll);
    a.sinks = (int)std::min(w->sinks, p->k_len);
  }
  if (a.table != nullptr) {
    a.one_way = a.causal ? a.buckets : a.buckets / 2;
    const int exact = a.one_way / 2, wide = a.one_way - exact;
    for (int u = 0; u <= exact; ++u) a.edges[u] = (unsigned short)u;
    // (the powers that are whole numbers may come out a hair above them)
    for (int t = 1; t < wide; ++t)
      a.edges[exact + t] = (unsigned short)std::ceil(exact * std::pow((double)a.max_distance / exact, (double)t / wide) - 1e-9);
    a.edges[a.one_way] = (unsigned short)(a.max_distance + 1);
    a.far = a.edges[a.one_way - 1];
    for (int dist = 0, u = 0; dist <= a.max_distance; ++dist) {
      while (u + 1 < a.one_way && a.edges[u + 1] <= dist) ++u;
      a.bucket_of[dist] = (unsigned char)u;
    }
  }
  return a;
}

struct AttnPlan {
  int splits = 1, table_parts = 0, kv_parts = 1, q_parts = 1, sink_parts = 1;
  int64_t part_sinks = 0, part_kv = 0, part_q = 0, part_out = 0, part_ml = 0, delta = 0, part_peak = 0, part_table = 0, bytes = 0;
};

AttnPlan plan_attention(const AttnArgs& a, bool backward, int cus) {
  AttnPlan p;
  int64_t at = 0;
  const int64_t rows = (int64_t)a.batch * a.heads * a.lq;
  if (backward) {
    p.delta = at, at += up256(rows * 4);
    p.q_parts = rows == 0 ? 1 : attn_q_parts(a, cus);
    if (p.q_parts > 1) p.part_q = at, at += up256(p.q_parts * rows * a.d * 4);
    if (a.type == CVS_TYPE_F16)
      p.part_peak = at, at += up256((int64_t)a.batch * a.heads * p.q_parts * ((a.lq + kAttnRows - 1) / kAttnRows) * 4);
    if (a.table != nullptr) {
      p.table_parts = a.batch * p.q_parts * ((a.lq + kAttnRows - 1) / kAttnRows);
      p.part_table = at, at += up256((int64_t)a.heads * p.table_parts * a.buckets * 4);
    }
    p.kv_parts = rows == 0 || a.lk == 0 ? 1 : attn_kv_parts(a, cus);
    if (p.kv_parts > 1) p.part_kv = at, at += up256((int64_t)p.kv_parts * 2 * a.batch * a.lk * a.k_heads * a.d * 4);
    if (rows > 0 && a.sinks > 0) p.sink_parts = attn_sink_parts(a, p.kv_parts, cus);
    if (p.sink_parts > 1) p.part_sinks = at, at += up256((int64_t)p.sink_parts * 2 * a.batch * a.sinks * a.k_heads * a.d * 4);
  } else {
    p.splits = rows == 0 ? 1 : attn_splits(a, cus);
    if (p.splits > 1) {
      p.part_out = at, at += up256(p.splits * rows * a.d * 4);
      p.part_ml = at, at += up256(p.splits * rows * 8);
    }
  }
  p.bytes = at;
  return p;
}

// (dk's and dv's launch has workgroups for the first keys, and fewer than 2^32 threads)
int check_first_keys(const AttnArgs& a, const AttnPlan& plan) {
  AttnArgs b = a;
  b.sink_parts = plan.sink_parts;
  return attn_key_workgroups(b) < (1 << 24) ? CVS_OK : fail(CVS_ERR_INVALID, "attention: too many first keys for a backward pass");
}

int attention_plan(const cvs_attention* p, const cvs_attention_window* w, int backward, int device, int64_t* workspace_bytes) {
  DevInfo di;
  int rc = dev_info(device, &di);
  if (rc == CVS_OK) rc = check_attention(p);
  if (rc == CVS_OK) rc = check_window(p, w);
  if (rc != CVS_OK) return rc;
  const AttnArgs a = attn_args(p, w);
  const AttnPlan plan = plan_attention(a, backward != 0, di.cus);
  if (backward != 0) rc = check_first_keys(a, plan);
  if (rc == CVS_OK && workspace_bytes != nullptr) *workspace_bytes = plan.bytes;
  return rc;
}

int attention_forward(const cvs_attention* p, const cvs_attention_window* w, void* out, float* lse, void* workspace,
                      int64_t workspace_bytes, int device, void* stream) {
  DevInfo di;
  int rc = gfx950(device, &di);
  if (rc == CVS_OK) rc = check_attention(p);
  if (rc == CVS_OK) rc = check_window(p, w);
  if (rc != CVS_OK || p->batch == 0 || p->q_len == 0) return rc;
  if (p->q == nullptr || (p->k_len > 0 && (p->k == nullptr || p->v == nullptr)) || out == nullptr)
    return fail(CVS_ERR_INVALID, "attention: null pointer");
  rc = check_heads(p->q, p->q_stride, "q");
  if (rc == CVS_OK) rc = check_heads(p->k, p->k_stride, "k");
  if (rc == CVS_OK) rc = check_heads(p->v, p->v_stride, "v");
  if (rc == CVS_OK && !aligned16(out)) rc = fail(CVS_ERR_INVALID, "out must be 16-byte aligned");
  if (rc != CVS_OK) return rc;
  AttnArgs a = attn_args(p, w);
  const AttnPlan plan = plan_attention(a, false, di.cus);
  rc = check_workspace(workspace, workspace_bytes, plan.bytes);
  if (rc != CVS_OK) return rc;
  DeviceGuard guard(device);
  if (guard.err != hipSuccess) return hip_fail(guard.err, "hipSetDevice");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  a.out = out, a.lse = lse;
  a.splits = plan.splits;
  a.part_out = reinterpret_cast<float*>(ws + plan.part_out);
  a.part_ml = reinterpret_cast<float*>(ws + plan.part_ml);
  return done(launch_attn_forward(a, s), "attention launch");
}

int attention_backward(const cvs_attention* p, const cvs_attention_window* w, const void* dout, const int64_t* dout_stride,
                       const void* out, const float* lse, void* dq, void* dk, void* dv, void* dbias_table, void* workspace,
                       int64_t workspace_bytes, int device, void* stream) {
  DevInfo di;
  int rc = gfx950(device, &di);
  if (rc == CVS_OK) rc = check_attention(p);
  if (rc == CVS_OK) rc = check_window(p, w);
  if (rc != CVS_OK || p->batch == 0 || (p->q_len == 0 && p->k_len == 0)) return rc;
  const bool rows = p->q_len > 0, keys = p->k_len > 0;
  if (dout_stride == nullptr || (rows && (p->q == nullptr || dout == nullptr || out == nullptr || lse == nullptr || dq == nullptr)) ||
      (keys && (p->k == nullptr || p->v == nullptr || dk == nullptr || dv == nullptr)) ||
      (p->bias_table != nullptr && dbias_table == nullptr))
    return fail(CVS_ERR_INVALID, "attention: null pointer");
  rc = check_heads(p->q, p->q_stride, "q");
  if (rc == CVS_OK) rc = check_heads(p->k, p->k_stride, "k");
  if (rc == CVS_OK) rc = check_heads(p->v, p->v_stride, "v");
  if (rc == CVS_OK) rc = check_heads(dout, dout_stride, "dout");
  if (rc == CVS_OK && !(aligned16(out) && aligned16(dq) && aligned16(dk) && aligned16(dv)))
    rc = fail(CVS_ERR_INVALID, "attention: pointers must be 16-byte aligned");
  if (rc != CVS_OK) return rc;
  AttnArgs a = attn_args(p, w);
  const AttnPlan plan = plan_attention(a, true, di.cus);
  rc = check_first_keys(a, plan);
  if (rc == CVS_OK) rc = check_workspace(workspace, workspace_bytes, plan.bytes);
  if (rc != CVS_OK) return rc;
  DeviceGuard guard(device);
  if (guard.err != hipSuccess) return hip_fail(guard.err, "hipSetDevice");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  a.out = const_cast<void*>(out), a.lse = const_cast<float*>(lse), a.dout = dout;
  for (int i = 0; i < 3; ++i) a.dos[i] = dout_stride[i];
  a.dq = dq, a.dk = dk, a.dv = dv, a.dtable = dbias_table;
  a.delta = reinterpret_cast<float*>(ws + plan.delta);
  a.part_peak = reinterpret_cast<float*>(ws + plan.part_peak);
  a.part_table = reinterpret_cast<float*>(ws + plan.part_table);
  a.table_parts = plan.table_parts;
  a.kv_parts = plan.kv_parts, a.q_parts = plan.q_parts, a.sink_parts = plan.sink_parts;
  a.part_sinks = reinterpret_cast<float*>(ws + plan.part_sinks);
  a.part_q = reinterpret_cast<float*>(ws + plan.part_q);
  a.part_kv = reinterpret_cast<float*>(ws + plan.part_kv);
  return done(launch_attn_backward(a, s), "attention backward launch");
}

}  // namespace

extern "C" {

int cvs_layer_norm(const void* x, const void* weight, const void* bias, int64_t n, int64_t d, int64_t x_stride,
                   double eps, int type, void* y, float* mean, float* rstd, int device, void* stream) {
  DevInfo di;
  int rc = gfx950(device, &di);
  if (rc == CVS_OK) rc = check_norm(n, d, type);
  if (rc != CVS_OK || n == 0) return rc;
  if (x == nullptr || weight == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr))
    return fail(CVS_ERR_INVALID, "layer norm: null pointer");
  if (x_stride < d && n > 1) return fail(CVS_ERR_INVALID, "layer norm: rows overlap");
  DeviceGuard guard(device);
  if (guard.err != hipSuccess) return hip_fail(guard.err, "hipSetDevice");
  NormArgs a = {};
  a.type = type, a.n = n, a.d = (int)d, a.x = x, a.x_stride = x_stride, a.weight = weight, a.bias = bias;
  a.eps = (float)eps, a.y = y, a.mean = mean, a.rstd = rstd;
  return done(launch_norm_forward(a, reinterpret_cast<hipStream_t>(stream)), "layer norm launch");
}

int cvs_layer_norm_backward_plan(int64_t n, int64_t d, int type, int device, int64_t* workspace_bytes) {
  DevInfo di;
  int rc = dev_info(device, &di);
  if (rc == CVS_OK) rc = check_norm(n, d, type);
  if (rc == CVS_OK && workspace_bytes != nullptr) *workspace_bytes = norm_ws(n, d, type, di.cus);
  return rc;
}

int cvs_layer_norm_backward(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd,
                            int64_t n, int64_t d, int64_t dy_stride, int64_t x_stride, int type, void* dx, void* dweight,
                            void* dbias, void* workspace, int64_t workspace_bytes, int device, void* stream) {
  DevInfo di;
  int rc = gfx950(device, &di);
  if (rc == CVS_OK) rc = check_norm(n, d, type);
  if (rc != CVS_OK) return rc;
  rc = check_workspace(workspace, workspace_bytes, norm_ws(n, d, type, di.cus));
  if (rc != CVS_OK || n == 0) return rc;
  if (dy == nullptr || x == nullptr || weight == nullptr || mean == nullptr || rstd == nullptr || dx == nullptr)
    return fail(CVS_ERR_INVALID, "layer norm: null pointer");
  if ((x_stride < d || dy_stride < d) && n > 1) return fail(CVS_ERR_INVALID, "layer norm: rows overlap");
  DeviceGuard guard(device);
  if (guard.err != hipSuccess) return hip_fail(guard.err, "hipSetDevice");
  NormArgs a = {};
  a.type = type, a.n = n, a.d = (int)d, a.x = x, a.x_stride = x_stride, a.weight = weight;
  a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
  a.dy = dy, a.dy_stride = dy_stride, a.dx = dx, a.dweight = dweight, a.dbias = dbias;
  a.partial = reinterpret_cast<float*>(workspace);
  a.parts = norm_backward_parts(n, d, type, di.cus);
  return done(launch_norm_backward(a, reinterpret_cast<hipStream_t>(stream)), "layer norm backward launch");
}

int cvs_linear_plan(int64_t m, int64_t k, int64_t n, int device, int64_t* workspace_bytes) {
  DevInfo di;
  int rc = dev_info(device, &di);
  if (rc == CVS_OK) rc = check_linear(m, k, n);
  GemmPlan p = {};
  if (rc == CVS_OK && m > 0) rc = check_plan(p = plan_gemm(m, n, k, di.cus));
  if (rc == CVS_OK && workspace_bytes != nullptr) *workspace_bytes = p.ws_bytes;
  return rc;
}

int cvs_linear(const void* x, const void* w, const void* bias, const void* residual, int64_t m, int64_t k, int64_t n,
               int64_t x_stride, int64_t residual_stride, int act, int type, void* y, void* pre, void* workspace,
               int64_t workspace_bytes, int device, void* stream) {
  DevInfo di;
  int rc = gfx950(device, &di);
  if (rc == CVS_OK) rc = check_linear(m, k, n);
  if (rc == CVS_OK) rc = check_linear_types(act, type);
  if (rc != CVS_OK || m == 0) return rc;
  if (x == nullptr || w == nullptr || y == nullptr) return fail(CVS_ERR_INVALID, "linear: null pointer");
  rc = check_rows(x, x_stride, k, "x");
  if (rc == CVS_OK && residual != nullptr) rc = check_rows(residual, residual_stride, n, "residual");
  if (rc != CVS_OK) return rc;
  if (!aligned16(w) || !aligned16(bias) || !aligned16(y) || !aligned16(pre))
    return fail(CVS_ERR_INVALID, "linear: pointers must be 16-byte aligned");
  const GemmPlan p = plan_gemm(m, n, k, di.cus);
  rc = check_plan(p);
  if (rc == CVS_OK) rc = check_workspace(workspace, workspace_bytes, p.ws_bytes);
  if (rc != CVS_OK) return rc;
  DeviceGuard guard(device);
  if (guard.err != hipSuccess) return hip_fail(guard.err, "hipSetDevice");
  GemmArgs a = {};
  a.type = type, a.m = (int)m, a.n = (int)n, a.k = (int)k;
  a.M = x, a.ldm = x_stride, a.N = w, a.ldn = k;
  a.bias = bias, a.residual = residual, a.ld_res = residual_stride, a.act = act;
  a.pre = pre, a.out = y, a.partial = reinterpret_cast<float*>(workspace), a.splits = p.splits;
  return done(launch_gemm(a, p, reinterpret_cast<hipStream_t>(stream)), "linear launch");
}

int cvs_linear_backward_plan(int64_t m, int64_t k, int64_t n, int act, int device, int64_t* workspace_bytes) {
  DevInfo di;
  int rc = dev_info(device, &di);
  if (rc == CVS_OK) rc = check_linear(m, k, n);
  LinearBackwardPlan p = {};
  if (rc == CVS_OK && m > 0) {
    p = plan_linear_backward(m, k, n, act, di.cus);
    rc = check_plan(p.dx);
    if (rc == CVS_OK) rc = check_plan(p.dw);
  }
  if (rc == CVS_OK && workspace_bytes != nullptr) *workspace_bytes = p.bytes;
  return rc;
}

int cvs_linear_backward(const void* dy, const void* x, const void* w, const void* pre, int64_t m, int64_t k, int64_t n,
                        int64_t dy_stride, int64_t x_stride, int act, int type, void* dx, void* dw, void* dbias,
                        void* workspace, int64_t workspace_bytes, int device, void* stream) {
  DevInfo di;
  int rc = gfx950(device, &di);
  if (rc == CVS_OK) rc = check_linear(m, k, n);
  if (rc == CVS_OK) rc = check_linear_types(act, type);
  if (rc != CVS_OK || m == 0) return rc;
  if (dy == nullptr || x == nullptr || w == nullptr || (act != CVS_ACT_NONE && pre == nullptr))
    return fail(CVS_ERR_INVALID, "linear: null pointer");
  rc = check_rows(dy, dy_stride, n, "dy");
  if (rc == CVS_OK) rc = check_rows(x, x_stride, k, "x");
  if (rc != CVS_OK) return rc;
  if (!aligned16(w) || !aligned16(pre) || !aligned16(dx) || !aligned16(dw) || !aligned16(dbias))
    return fail(CVS_ERR_INVALID, "linear: pointers must be 16-byte aligned");
  const LinearBackwardPlan p = plan_linear_backward(m, k, n, act, di.cus);
  rc = check_plan(p.dx);
  if (rc == CVS_OK) rc = check_plan(p.dw);
  if (rc == CVS_OK) rc = check_workspace(workspace, workspace_bytes, p.bytes);
  if (rc != CVS_OK) return rc;
  DeviceGuard guard(device);
  if (guard.err != hipSuccess) return hip_fail(guard.err, "hipSetDevice");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  const void* dz = dy;
  int64_t dz_stride = dy_stride;
  if (act != CVS_ACT_NONE || dbias != nullptr) {
    ActGradArgs g = {};
    g.type = type, g.act = act, g.m = m, g.n = (int)n, g.dy = dy, g.dy_stride = dy_stride, g.pre = pre;
    g.dbias = dbias, g.partial = reinterpret_cast<float*>(ws + p.partial), g.parts = p.parts;
    if (act != CVS_ACT_NONE) {
      g.dz = ws + p.dz;
      dz = g.dz, dz_stride = n;
    }
    const hipError_t e = launch_act_grad(g, s);
    if (e != hipSuccess) return hip_fail(e, "linear backward launch");
  }
  GemmArgs x_args = {}, w_args = {};
  x_args.type = w_args.type = type;
  // dx = dz [m, n] x w [n, k]
  x_args.m = (int)m, x_args.n = (int)k, x_args.k = (int)n;
  x_args.M = dz, x_args.ldm = dz_stride, x_args.m_strided = false, x_args.N = w, x_args.ldn = k, x_args.n_strided = true;
  x_args.out = dx, x_args.splits = p.dx.splits, x_args.partial = reinterpret_cast<float*>(ws + p.gemm);
  // dw = dz^T [n, m] x x [m, k]
  w_args.m = (int)n, w_args.n = (int)k, w_args.k = (int)m;
  w_args.M = dz, w_args.ldm = dz_stride, w_args.m_strided = true, w_args.N = x, w_args.ldn = x_stride, w_args.n_strided = true;
  w_args.out = dw, w_args.splits = p.dw.splits, w_args.partial = reinterpret_cast<float*>(ws + p.gemm_dw);
  hipError_t e = hipSuccess;
  if (dx != nullptr && dw != nullptr)
    e = launch_gemm_pair(x_args, p.dx, w_args, p.dw, s);
  else if (dx != nullptr)
    e = launch_gemm(x_args, p.dx, s);
  else if (dw != nullptr)
    e = launch_gemm(w_args, p.dw, s);
  return done(e, "linear backward launch");
}

int cvs_gated_linear_plan(int64_t m, int64_t k, int64_t n, int device, int64_t* workspace_bytes) {
  DevInfo di;
  int rc = dev_info(device, &di);
  if (rc == CVS_OK) rc = check_gated(m, k, n);
  GemmPlan p = {};
  if (rc == CVS_OK && m > 0) rc = check_plan(p = plan_gated(m, n, k, di.cus));
  if (rc == CVS_OK && workspace_bytes != nullptr) *workspace_bytes = p.ws_bytes;
  return rc;
}

int cvs_gated_linear(const void* x, const void* gate, const void* up, const void* gate_bias, const void* up_bias, int64_t m,
                     int64_t k, int64_t n, int64_t x_stride, int act, int type, void* y, void* pre, void* workspace,
                     int64_t workspace_bytes, int device, void* stream) {
  DevInfo di;
  int rc = gfx950(device, &di);
  if (rc == CVS_OK) rc = check_gated(m, k, n);
  if (rc == CVS_OK) rc = check_gated_types(act, type);
  if (rc != CVS_OK || m == 0) return rc;
  if (x == nullptr || gate == nullptr || up == nullptr || y == nullptr) return fail(CVS_ERR_INVALID, "gated linear: null pointer");
  rc = check_rows(x, x_stride, k, "x");
  if (rc != CVS_OK) return rc;
  if (!aligned16(gate) || !aligned16(up) || !aligned16(gate_bias) || !aligned16(up_bias) || !aligned16(y) || !aligned16(pre))
    return fail(CVS_ERR_INVALID, "gated linear: pointers must be 16-byte aligned");
  const GemmPlan p = plan_gated(m, n, k, di.cus);
  rc = check_plan(p);
  if (rc == CVS_OK) rc = check_workspace(workspace, workspace_bytes, p.ws_bytes);
  if (rc != CVS_OK) return rc;
  DeviceGuard guard(device);
  if (guard.err != hipSuccess) return hip_fail(guard.err, "hipSetDevice");
  GemmKindArgs a = {};
  a.type = type, a.m = (int)m, a.n = (int)n, a.k = (int)k;
  a.M = x, a.ldm = x_stride, a.N = gate, a.N2 = up, a.ldn = k;
  a.bias = gate_bias, a.bias2 = up_bias, a.act = act;
  a.pre = pre, a.out = y, a.partial = reinterpret_cast<float*>(workspace), a.splits = p.splits;
  return done(launch_gated(a, p, reinterpret_cast<hipStream_t>(stream)), "gated linear launch");
}

int cvs_gated_linear_backward_plan(int64_t m, int64_t k, int64_t n, int device, int64_t* workspace_bytes) {
  DevInfo di;
  int rc = dev_info(device, &di);
  if (rc == CVS_OK) rc = check_gated(m, k, n);
  GatedBackwardPlan p = {};
  if (rc == CVS_OK && m > 0) rc = check_gated_plan(p = plan_gated_backward(m, k, n, di.cus));
  if (rc == CVS_OK && workspace_bytes != nullptr) *workspace_bytes = p.bytes;
  return rc;
}

int cvs_gated_linear_backward(const void* dy, const void* x, const void* gate, const void* up, const void* pre, int64_t m,
                              int64_t k, int64_t n, int64_t dy_stride, int64_t x_stride, int act, int type, void* dx,
                              void* dgate, void* dup, void* dgate_bias, void* dup_bias, void* workspace,
                              int64_t workspace_bytes, int device, void* stream) {
  DevInfo di;
  int rc = gfx950(device, &di);
  if (rc == CVS_OK) rc = check_gated(m, k, n);
  if (rc == CVS_OK) rc = check_gated_types(act, type);
  if (rc != CVS_OK || m == 0) return rc;
  if (dy == nullptr || x == nullptr || gate == nullptr || up == nullptr || pre == nullptr)
    return fail(CVS_ERR_INVALID, "gated linear: null pointer");
  rc = check_rows(dy, dy_stride, n, "dy");
  if (rc == CVS_OK) rc = check_rows(x, x_stride, k, "x");
  if (rc != CVS_OK) return rc;
  if (!aligned16(gate) || !aligned16(up) || !aligned16(pre) || !aligned16(dx) || !aligned16(dgate) || !aligned16(dup) ||
      !aligned16(dgate_bias) || !aligned16(dup_bias))
    return fail(CVS_ERR_INVALID, "gated linear: pointers must be 16-byte aligned");
  const GatedBackwardPlan p = plan_gated_backward(m, k, n, di.cus);
  rc = check_gated_plan(p);
  if (rc == CVS_OK) rc = check_workspace(workspace, workspace_bytes, p.bytes);
  if (rc != CVS_OK) return rc;
  DeviceGuard guard(device);
  if (guard.err != hipSuccess) return hip_fail(guard.err, "hipSetDevice");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  GatedGradArgs g = {};
  g.type = type, g.act = act, g.m = m, g.n = (int)n, g.dy = dy, g.dy_stride = dy_stride, g.pre = pre;
  g.dz = ws + p.dz, g.dgate_bias = dgate_bias, g.dup_bias = dup_bias;
  g.partial = reinterpret_cast<float*>(ws + p.partial), g.parts = p.parts, g.rests = p.rests;
  g.peaks = reinterpret_cast<float*>(ws + p.peaks), g.unit = reinterpret_cast<float*>(ws + p.unit);
  if (p.rests && (dgate != nullptr || dup != nullptr)) g.x = x, g.x_stride = x_stride, g.k = (int)k, g.twice = ws + p.twice;
  hipError_t e = launch_gated_grad(g, s);
  float* sums = reinterpret_cast<float*>(ws + p.gemm);
  const float* unit = type == CVS_TYPE_F16 ? g.unit : nullptr;
  if (e == hipSuccess && dx != nullptr) {  // dx = dg [m, n] gate [n, k] + du up
    GemmKindArgs a = {};
    a.type = type, a.m = (int)p.rows, a.n = (int)k, a.k = (int)n;
    a.M = g.dz, a.ldm = 2 * n, a.m_second = n, a.N = gate, a.N2 = up, a.ldn = k, a.n_strided = true;
    a.out = dx, a.m_first = a.m, a.partial = sums, a.splits = p.dx.splits, a.unit = unit;
    e = launch_two_parts(a, p.dx, p.rests, s);
  }
  // dgate = dg^T x, dup = du^T x: one product of 2 n rows
  auto weights = [&](int64_t first, int64_t rows, const GemmPlan& plan, void* out, void* out2) {
    GemmKindArgs a = {};
    a.type = type, a.m = (int)rows, a.n = (int)k, a.k = (int)p.rows;
    a.M = static_cast<unsigned char*>(g.dz) + 2 * first, a.ldm = 2 * n, a.m_strided = true;
    a.N = p.rests ? g.twice : x, a.ldn = p.rests ? k : x_stride, a.n_strided = true;
    a.out = out, a.out2 = out2, a.m_first = (int)n, a.partial = sums, a.splits = plan.splits, a.unit = unit;
    return launch_weights(a, plan, s);
  };
  if (e == hipSuccess && dgate != nullptr && dup != nullptr)
    e = weights(0, 2 * n, p.dw, dgate, dup);
  else if (e == hipSuccess && dgate != nullptr)
    e = weights(0, n, p.one, dgate, nullptr);
  else if (e == hipSuccess && dup != nullptr)
    e = weights(n, n, p.one, dup, nullptr);
  return done(e, "gated linear backward launch");
}

int cvs_quantize_rows(const void* x, int64_t n, int64_t d, int64_t x_stride, int type, void* values, float* scales, int device,
                      void* stream) {
  DevInfo di;
  int rc = gfx950(device, &di);
  if (rc == CVS_OK) rc = check_quantize(n, d, type);
  if (rc != CVS_OK || n == 0) return rc;
  if (x == nullptr || values == nullptr || scales == nullptr) return fail(CVS_ERR_INVALID, "quantize rows: null pointer");
  rc = check_rows(x, x_stride, d, "x");
  if (rc == CVS_OK && !aligned16(values)) rc = fail(CVS_ERR_INVALID, "quantize rows: values must be 16-byte aligned");
  if (rc != CVS_OK) return rc;
  DeviceGuard guard(device);
  if (guard.err != hipSuccess) return hip_fail(guard.err, "hipSetDevice");
  QuantArgs a = {};
  a.type = type, a.n = n, a.d = (int)d, a.x = x, a.x_stride = x_stride;
  a.values = static_cast<signed char*>(values), a.scales = scales;
  return done(launch_quantize(a, reinterpret_cast<hipStream_t>(stream)), "quantize rows launch");
}

int cvs_linear_int8_plan(int64_t m, int64_t k, int64_t n, int device, int64_t* workspace_bytes) {
  DevInfo di;
  int rc = dev_info(device, &di);
  if (rc == CVS_OK) rc = check_int8(m, k, n, CVS_ACT_NONE, CVS_TYPE_F16);
  Int8Plan p = {};
  if (rc == CVS_OK && m > 0) rc = check_plan((p = plan_linear_int8(m, k, n, di.cus)).product);
  if (rc == CVS_OK && workspace_bytes != nullptr) *workspace_bytes = p.bytes;
  return rc;
}

int cvs_linear_int8(const void* x, const void* w, const float* w_scales, const void* bias, const void* residual, int64_t m,
                    int64_t k, int64_t n, int64_t x_stride, int64_t residual_stride, int act, int type, void* y,
                    void* workspace, int64_t workspace_bytes, int device, void* stream) {
  DevInfo di;
  int rc = gfx950(device, &di);
  if (rc == CVS_OK) rc = check_int8(m, k, n, act, type);
  if (rc != CVS_OK || m == 0) return rc;
  if (x == nullptr || w == nullptr || w_scales == nullptr || y == nullptr) return fail(CVS_ERR_INVALID, "linear int8: null pointer");
  rc = check_rows(x, x_stride, k, "x");
  if (rc == CVS_OK && residual != nullptr) rc = check_rows(residual, residual_stride, n, "residual");
  if (rc != CVS_OK) return rc;
  if (!aligned16(w) || !aligned16(w_scales) || !aligned16(bias) || !aligned16(y))
    return fail(CVS_ERR_INVALID, "linear int8: pointers must be 16-byte aligned");
  const Int8Plan p = plan_linear_int8(m, k, n, di.cus);
  rc = check_plan(p.product);
  if (rc == CVS_OK) rc = check_workspace(workspace, workspace_bytes, p.bytes);
  if (rc != CVS_OK) return rc;
  DeviceGuard guard(device);
  if (guard.err != hipSuccess) return hip_fail(guard.err, "hipSetDevice");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  GemmKindArgs a = {};
  a.type = type, a.m = (int)m, a.n = (int)n, a.N = w, a.col_scale = w_scales;
  a.bias = bias, a.residual = residual, a.ld_res = residual_stride, a.act = act, a.out = y;
  if (p.few) return done(launch_int8_rows(a, x, x_stride, (int)k, s), "linear int8 launch");
  QuantArgs q = {};
  q.type = type, q.n = m, q.d = (int)k, q.x = x, q.x_stride = x_stride;
  q.values = reinterpret_cast<signed char*>(ws + p.values), q.scales = reinterpret_cast<float*>(ws + p.scales);
  hipError_t e = launch_quantize(q, s);
  if (e != hipSuccess) return hip_fail(e, "linear int8 launch");
  a.k = (int)(k / 2), a.M = q.values, a.ldm = k / 2, a.ldn = k / 2;
  a.row_scale = q.scales;
  a.partial = reinterpret_cast<float*>(ws + p.gemm), a.splits = p.product.splits;
  return done(launch_int8(a, p.product, s), "linear int8 launch");
}

int cvs_attention_plan(const cvs_attention* p, int backward, int device, int64_t* workspace_bytes) {
  return attention_plan(p, nullptr, backward, device, workspace_bytes);
}

int cvs_attention_forward(const cvs_attention* p, void* out, float* lse, void* workspace, int64_t workspace_bytes,
                          int device, void* stream) {
  return attention_forward(p, nullptr, out, lse, workspace, workspace_bytes, device, stream);
}

int cvs_attention_backward(const cvs_attention* p, const void* dout, const int64_t* dout_stride, const void* out,
                           const float* lse, void* dq, void* dk, void* dv, void* dbias_table, void* workspace,
                           int64_t workspace_bytes, int device, void* stream) {
  return attention_backward(p, nullptr, dout, dout_stride, out, lse, dq, dk, dv, dbias_table, workspace, workspace_bytes, device,
                            stream);
}

int cvs_attention_window_plan(const cvs_attention* p, const cvs_attention_window* w, int backward, int device,
                              int64_t* workspace_bytes) {
  if (w == nullptr) return fail(CVS_ERR_INVALID, "attention: null window");
  return attention_plan(p, w, backward, device, workspace_bytes);
}

int cvs_attention_window_forward(const cvs_attention* p, const cvs_attention_window* w, void* out, float* lse, void* workspace,
                                 int64_t workspace_bytes, int device, void* stream) {
  if (w == nullptr) return fail(CVS_ERR_INVALID, "attention: null window");
  return attention_forward(p, w, out, lse, workspace, workspace_bytes, device, stream);
}

int cvs_attention_window_backward(const cvs_attention* p, const cvs_attention_window* w, const void* dout,
                                  const int64_t* dout_stride, const void* out, const float* lse, void* dq, void* dk, void* dv,
                                  void* dbias_table, void* workspace, int64_t workspace_bytes, int device, void* stream) {
  if (w == nullptr) return fail(CVS_ERR_INVALID, "attention: null window");
  return attention_backward(p, w, dout, dout_stride, out, lse, dq, dk, dv, dbias_table, workspace, workspace_bytes, device, stream);
}

}  // extern "C"
