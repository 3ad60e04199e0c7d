// Argument blocks and launchers of the text-encoder kernels: layer norm, matrix
// product with an epilogue, attention (internal to libcvs_hip.so).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cvs {

enum ElemType : int { kF16 = 0, kBF16 = 1, kF32 = 2 };
enum Activation : int { kActNone = 0, kActGelu = 1, kActRelu = 2, kActTanh = 3 };

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
struct GemmPlan {
  int tile, tile_n;  // rows and columns of a workgroup's tile
  int splits;        // parts of the reduction
  int64_t ws_bytes;
};
GemmPlan plan_gemm(int64_t m, int64_t n, int64_t k, int cus);
hipError_t launch_gemm(const GemmArgs& a, const GemmPlan& p, hipStream_t s);
// Two products, with partial sums apart; one launch where their tiles are alike.  a: N strided, b: both.
hipError_t launch_gemm_pair(const GemmArgs& a, const GemmPlan& pa, const GemmArgs& b, const GemmPlan& pb, hipStream_t s);

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
};
constexpr int kAttnRows = 128;    // query (or key) rows of a workgroup
int attn_q_parts(const AttnArgs& a, int cus);
int attn_kv_parts(const AttnArgs& a, int cus);
int attn_splits(const AttnArgs& a, int cus);
hipError_t launch_attn_forward(const AttnArgs& a, hipStream_t s);
hipError_t launch_attn_backward(const AttnArgs& a, hipStream_t s);

}  // namespace cvs
