// Argument blocks and launchers of the text-encoder kernels: layer norm, matrix
// product with an epilogue, attention (internal to libcvs_hip.so).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cvs {

enum ElemType : int { kF16 = 0, kBF16 = 1, kF32 = 2 };
enum Activation : int { kActNone = 0, kActGelu = 1, kActRelu = 2, kActTanh = 3, kActSilu = 4, kActSigmoid = 5 };  // (the last two: gates)

// ---- layer norm ----------------------------------------------------------------
struct NormArgs {
  int type;
  int64_t n;
  int d;
  const void* x;
  int64_t x_stride;        // elements between rows
  const void* weight;      // [d]
  const void* bias;        // [d] or null
  float eps;
  void* y;                 // [n, d]
  float* mean;             // [n] or null (with rstd)
  float* rstd;
  // backward: mean and rstd are inputs
  const void* dy;
  int64_t dy_stride;
  void* dx;                // [n, d]
  void* dweight;           // [d]
  void* dbias;             // [d]
  float* partial;          // [parts, 2, d] sums of the row groups
  int parts;
};
// Row groups (workgroups) of the backward pass, each with its own partial sums.
int norm_backward_parts(int64_t n, int64_t d, int type, int cus);
hipError_t launch_norm_forward(const NormArgs& a, hipStream_t s);
hipError_t launch_norm_backward(const NormArgs& a, hipStream_t s);

// ---- matrix product ------------------------------------------------------------
// out[i, j] = sum_r M(i, r) N(j, r), i < m, j < n, r < k, with the epilogue
// z = sum + bias[j] (-> pre), out = act(z) + residual[i, j].  An operand is stored
// either [rows, k] (its reduction contiguous) or [k, rows] (strided).
struct GemmArgs {
  int type;
  int m, n, k;
  const void* M;
  int64_t ldm;
  bool m_strided;
  const void* N;
  int64_t ldn;
  bool n_strided;
  const void* bias;       // [n] or null
  const void* residual;   // [m, n] or null
  int64_t ld_res;
  int act;
  void* pre;              // [m, n] or null
  void* out;              // [m, n]
  float* partial;         // [splits, m, n] when splits > 1
  int splits;
};
// The other kinds of product (cvs_gemm_tile.h); partial is [splits, m, 2, n] when gated, whole numbers when int8.
struct GemmKindArgs : GemmArgs {
  const void* N2;         // gated: the second factor's weight; two parts: N of the second part
  const void* bias2;      // gated: [n] or null
  int64_t m_second;       // two parts: elements from M's first part to its second
  const float* unit;      // two parts, weights: what the sums are in units of, or null
  int m_first;            // weights: rows of out, those after them are out2's
  void* out2;
  const float* row_scale; // int8: [m]
  const float* col_scale; // int8: [n]
};
struct GemmPlan {
  int tile, tile_n;  // rows and columns of a workgroup's tile
  int splits;        // parts of the reduction
  int64_t ws_bytes;
};
struct TileChoice { int m, n, wgs, threads; double stage; };  // a tile, workgroups of it a CU, us a stage
// The choice of least estimated time; sums: fp32 sums of an output where the reduction is split.
GemmPlan plan_tiles(const TileChoice* choices, int count, int64_t m, int64_t n, int64_t stages, int sums, int cus);
GemmPlan plan_gemm(int64_t m, int64_t n, int64_t k, int cus);
hipError_t launch_gemm(const GemmArgs& a, const GemmPlan& p, hipStream_t s);
// Two products, with partial sums apart; one launch where their tiles are alike.  a: N strided, b: both.
hipError_t launch_gemm_pair(const GemmArgs& a, const GemmPlan& pa, const GemmArgs& b, const GemmPlan& pb, hipStream_t s);

// The gated product's forward pass (out [m, n], pre [m, 2 n] or null) and dx of its backward pass:
// dz [m, 2 n] times both weights.
GemmPlan plan_gated(int64_t m, int64_t n, int64_t k, int cus);
hipError_t launch_gated(const GemmKindArgs& a, const GemmPlan& p, hipStream_t s);
GemmPlan plan_two_parts(int64_t m, int64_t n, int64_t k, bool rests, int cus);
hipError_t launch_two_parts(const GemmKindArgs& a, const GemmPlan& p, bool rests, hipStream_t s);
// The weights' gradients, dz^T x, one behind the other's rows: plan_gemm's tiles, both operands strided.
hipError_t launch_weights(const GemmKindArgs& a, const GemmPlan& p, hipStream_t s);

// dz = [dy up act'(gate), dy act(gate)] ([m, 2 n], contiguous) of pre = [gate, up], and dz's column sums.
struct GatedGradArgs {
  int type, act;
  int64_t m;
  int n;
  const void* dy;
  int64_t dy_stride;
  const void* pre;
  void* dz;
  void* dgate_bias;       // [n] or null
  void* dup_bias;
  float* partial;         // [parts, 2, n] when either is not null
  int parts;
  bool rests;             // dz is [2 m, 2 n]: what rounding took off its rows behind them
  float* peaks;           // float16: [gated_grad_workgroups] largest finite |dz|
  float* unit;            // float16: dz is held times 1 / unit
  const void* x;          // and x is copied to twice [2 m, k], to go with them, or null
  int64_t x_stride;
  int k;
  void* twice;
};
// Of so few rows what dz loses to 16 bits is kept (cvs_gated.hip).
inline bool gated_few_rows(int64_t m) { return m <= 32; }
int gated_grad_parts(int64_t m, int64_t n, int cus);
int64_t gated_grad_workgroups(int64_t m, int64_t n, int parts);
hipError_t launch_gated_grad(const GatedGradArgs& a, hipStream_t s);

// Rows in 8-bit whole numbers with a scale each, and the product of such operands (ldm, ldn and k in
// 16-bit units: pairs of values).
struct QuantArgs {
  int type;
  int64_t n;
  int d;
  const void* x;
  int64_t x_stride;
  signed char* values;    // [n, d]
  float* scales;          // [n]
};
hipError_t launch_quantize(const QuantArgs& a, hipStream_t s);
// Few rows: one launch, of rows x (m of d values), whole numbers and product.
bool int8_few_rows(int64_t m, int64_t n, int64_t k, const GemmPlan& tiles, int cus);
hipError_t launch_int8_rows(const GemmKindArgs& a, const void* x, int64_t x_stride, int d, hipStream_t s);
GemmPlan plan_int8(int64_t m, int64_t n, int64_t k, int cus);
hipError_t launch_int8(const GemmKindArgs& a, const GemmPlan& p, hipStream_t s);

// dz = dy act'(pre) ([m, n], when act is not none and dz not null) and the column
// sums of dz (dbias, when not null).
struct ActGradArgs {
  int type, act;
  int64_t m;
  int n;
  const void* dy;
  int64_t dy_stride;
  const void* pre;        // [m, n] contiguous
  void* dz;
  void* dbias;
  float* partial;         // [parts, n] when parts > 1
  int parts;
};
int act_grad_parts(int64_t m, int64_t n, int cus);
hipError_t launch_act_grad(const ActGradArgs& a, hipStream_t s);

// Column sums of fp32 partial rows, sum_p partial[p * stride + j]: the first n1 columns to
// out, the n2 after them to out2.
hipError_t launch_column_sums(const float* partial, int parts, int64_t stride, int n1, int n2, int type, void* out, void* out2,
                              hipStream_t s);

// ---- attention -----------------------------------------------------------------
constexpr int kMaxBuckets = 128;
constexpr int kMaxDistance = 256;

struct AttnArgs {
  int type;
  int batch, lq, lk, heads, k_heads, d;
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];    // batch, position, head strides in elements
  float scale;
  int causal;
  const int* key_lengths;         // [batch] or null
  const int* query_lengths;
  const int* query_start;         // [batch] key position of query 0, or null: lk - lq
  // learned bias by relative position
  const void* table;              // [buckets, heads] or null
  int buckets, max_distance;
  int far;                             // smallest distance of the last bucket
  int one_way;                          // buckets of one direction
  unsigned char bucket_of[kMaxDistance + 1];   // a direction's bucket by distance (the last: all further ones)
  unsigned short edges[kMaxBuckets + 1];       // smallest distance of each, then one past max_distance
  // forward
  void* out;                      // [batch, lq, heads, d]
  float* lse;                     // [batch, heads, lq] or null
  int splits;                     // parts of the keys (forward, few query rows)
  float* part_out;                // [splits, batch, heads, lq, d]
  float* part_ml;                 // [splits, batch, heads, lq, 2]: maximum and sum
  // backward
  const void* dout;
  int64_t dos[3];
  float* delta;                   // [batch, heads, lq] sum(dout out)
  void *dq, *dk, *dv, *dtable;
  int q_parts;                    // parts of the keys that dq is summed over
  float* part_q;                  // [q_parts, batch, lq, heads, d] when q_parts > 1
  float* part_peak;               // [batch, heads, q_parts, query blocks] largest |ds| (float16)
  float* part_table;              // [heads, batch * q_parts * query blocks, buckets]
  int table_parts;
  int kv_parts;                   // parts of the queries that dk and dv are summed over
  float* part_kv;                 // [kv_parts, 2, batch, lk, k_heads, d] when kv_parts > 1
  // sliding window: a row at position p sees keys p - before .. p + after (causal: after is 0) and the first `sinks`
  int windowed, before, after, sinks;  // sinks <= lk
  int sink_parts;                 // parts of the queries that dk and dv of the first keys are summed over
  float* part_sinks;              // [sink_parts, 2, batch, sinks, k_heads, d] when sink_parts > 1
};
constexpr int kAttnRows = 128;    // query (or key) rows of a workgroup
int attn_q_parts(const AttnArgs& a, int cus);
int attn_kv_parts(const AttnArgs& a, int cus);
int attn_sink_parts(const AttnArgs& a, int kv_parts, int cus);
int attn_splits(const AttnArgs& a, int cus);
int64_t attn_key_workgroups(const AttnArgs& a);  // of dk's and dv's launch, a part of its rows
hipError_t launch_attn_forward(const AttnArgs& a, hipStream_t s);
hipError_t launch_attn_backward(const AttnArgs& a, hipStream_t s);

}  // namespace cvs
