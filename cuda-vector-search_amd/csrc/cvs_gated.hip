// The gated feed-forward block: both projections, the activation and the product in one
// kernel, and its backward pass.
//
//   y = act(g) * u,  g = x Wg^T + bg,  u = x Wu^T + bu  (pre = [g, u], rounded, for the backward pass)
//   dg = dy * u * act'(g),  du = dy * act(g)            (dz = [dg, du], rounded, and its column sums)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// Forward, a tile of the product has as many columns of g as of u, the same ones, so that g and
// u meet in a wave's registers.  Backward, dx is one sum over two reductions and both weights'
// gradients are one product whose rows are dz's 2 n columns.
#include <algorithm>

#include "cvs_gemm_tile.h"

namespace cvs {

namespace {

template <class T, int WM, int WN, int BM, int BN, int RING, int WGS, int KIND>
__global__ __launch_bounds__(64 * WM * WN, WGS) void gemm_kind_kernel(GemmKindArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[gemm_lds<WM, WN, BM, BN, RING>()];
  __shared__ __attribute__((aligned(16))) float vectors[gemm_vectors<KIND, WM * BM * 32, WN * BN * 16>()];
  gemm_tile<T, WM, WN, BM, BN, RING, KIND == kWeights, KIND != kGated, KIND>(a, blockIdx.x, smem, vectors);
}

// Adds the parts of a split reduction, in order, and finishes: 8 columns a thread.
template <class T>
__global__ __launch_bounds__(kBlock) void gated_join_kernel(GemmKindArgs a) {
  const int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  const int pieces = a.n / 8;
  const int64_t i = at / pieces;
  if (i >= a.m) return;
  const int j = (int)(at - i * pieces) * 8;
  const int64_t plane = (int64_t)a.m * a.n * 2;
  float z[2][8], h[8], bias[2][8];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) z[u][e] = 0.f;
  const float* p = a.partial + i * 2 * a.n + j;
  for (int s = 0; s < a.splits; ++s, p += plane)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float* from = p + (u == 0 ? 0 : a.n);
      const f32x4 lo = *reinterpret_cast<const f32x4*>(from), hi = *reinterpret_cast<const f32x4*>(from + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) z[u][e] += lo[e], z[u][4 + e] += hi[e];
    }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const T* from = (const T*)(u == 0 ? a.bias : a.bias2);
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[u][e] = 0.f;
    if (from != nullptr) load8(from + j, bias[u]);
  }
  finish_gated8(a.act, bias[0], bias[1], z[0], z[1], h);
  if (a.pre != nullptr) {
    store8((T*)a.pre + i * 2 * a.n + j, z[0]);
    store8((T*)a.pre + i * 2 * a.n + a.n + j, z[1]);
  }
  store8((T*)a.out + i * a.n + j, h);
}

// The same of two parts and of weights (halves: the second half of the rows is what rounding took off the first).
template <class T>
__global__ __launch_bounds__(kBlock) void sums_join_kernel(GemmKindArgs a, int halves) {
  const int64_t at = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * 8, plane = (int64_t)a.m / halves * a.n;
  if (at >= plane) return;
  float z[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] = 0.f;
  const float* p = a.partial + at;
  for (int s = 0; s < a.splits * halves; ++s, p += plane) {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] += lo[e], z[4 + e] += hi[e];
  }
  if (a.unit != nullptr) {
    const float unit = *a.unit;
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] *= unit;
  }
  const int64_t first = (int64_t)a.m_first * a.n;
  store8(at < first ? (T*)a.out + at : (T*)a.out2 + (at - first), z);
}

template <class T, int WM, int WN, int BM, int BN, int RING, int WGS, int KIND>
void launch_tiles(const GemmKindArgs& a, hipStream_t s) {
  const dim3 grid(gemm_grid(a, WM * BM * 32, WN * BN * (KIND == kGated ? 16 : 32))), block(64 * WM * WN);
  hipLaunchKernelGGL((gemm_kind_kernel<T, WM, WN, BM, BN, RING, WGS, KIND>), grid, block, 0, s, a);
}

dim3 join_grid(const GemmKindArgs& a) { return dim3((unsigned)(((int64_t)a.m * (a.n / 8) + kBlock - 1) / kBlock)); }

template <class T>
hipError_t gated(const GemmKindArgs& a, const GemmPlan& p, hipStream_t s) {
  if (p.tile == 256)
    launch_tiles<T, 4, 2, 2, 4, 2, 1, kGated>(a, s);
  else if (p.tile == 128)
    launch_tiles<T, 2, 2, 2, 2, 2, 2, kGated>(a, s);
  else
    launch_tiles<T, 2, 2, 1, 2, 3, 2, kGated>(a, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL(gated_join_kernel<T>, join_grid(a), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

template <class T, int KIND>
hipError_t sums(const GemmKindArgs& a, const GemmPlan& p, int halves, hipStream_t s) {
  if (p.tile == 256 && p.tile_n == 256)
    launch_tiles<T, 4, 2, 2, 4, 2, 1, KIND>(a, s);
  else if (p.tile == 256)
    launch_tiles<T, 4, 2, 2, 3, 2, 1, KIND>(a, s);
  else if (p.tile == 128)
    launch_tiles<T, 2, 2, 2, 2, 2, 2, KIND>(a, s);
  else
    launch_tiles<T, 2, 2, 1, 1, 3, 2, KIND>(a, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL(sums_join_kernel<T>, join_grid(a), dim3(kBlock), 0, s, a, halves);
  return hipGetLastError();
}

// du = dy act(g) and dg = dy u act'(g) of 8 values (the same branch for a whole launch).
__device__ __forceinline__ void gate_grads8(const float* dy, const float* g, const float* u, int act, float* dg, float* du) {
#pragma unroll
  for (int e = 0; e < 8; ++e) dg[e] = dy[e] * u[e];
  if (act == kActSilu || act == kActSigmoid) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // s and 1 - s, each with its digits however small
      const float x = __builtin_amdgcn_exp2f(fabsf(g[e]) * -kLog2e), r = __builtin_amdgcn_rcpf(1.f + x);
      const float s = g[e] < 0.f ? x * r : r, rest = g[e] < 0.f ? r : x * r;
      du[e] = dy[e] * (act == kActSilu ? g[e] * s : s);
      dg[e] *= act == kActSilu ? s * fmaf(g[e], rest, 1.f) : s * rest;
    }
  } else if (act == kActNone) {
#pragma unroll
    for (int e = 0; e < 8; ++e) du[e] = dy[e] * g[e];
  } else {
    float h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = g[e];
    activate8(h, act);
#pragma unroll
    for (int e = 0; e < 8; ++e) du[e] = dy[e] * h[e];
    times_slope8(dg, g, act);
  }
}

// Pieces of 8 columns of a workgroup, as act_grad_kernel's: few for few rows.
__host__ __device__ inline int gated_grad_width(int64_t m, int n) { return m <= 256 ? 16 : min(n / 8, kBlock); }

// float16 holds small gradients as subnormals, of few digits, which sums over many rows are not (of 4096 rows and dy of
// 2^-18 dgate was off by 0.7%), and none past 65504, which products with small weights are not.  So dz is held there times 2^4,
// or, where that brings its largest value past 2^15 or leaves it below 2^-2, times what brings it to 2^14 to 2^15, and
// the products' sums are taken back: a dz loses 2^-23 of the largest at most beside its own rounding.  The largest is known
// once all are made: gated_grad_kernel makes them times 2^4 and leaves each workgroup's largest, and a launch after it,
// REFIT, looks at these and makes dz again where they do not fit (the pass of 16384 rows of 2 x 2048, k = 768: 297 us,
// 359 where dz is made again, 295 without any of this; 23 rows of 2 x 1536, k = 384 30.5 and 30.6, in bfloat16 28).
template <class T>
constexpr bool kFits = true;
template <>
constexpr bool kFits<_Float16> = false;
constexpr int kDzLift = 4;

// The largest of a workgroup's values, in every thread (red: 4 floats of LDS).
__device__ __forceinline__ float workgroup_max(float v, float* red) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor(v, s));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// The largest magnitude of 16 values, of those that are finite.
__device__ __forceinline__ float finite_max8(const float* v, const float* w) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = fabsf(v[e]), y = fabsf(w[e]);
    top = fmaxf(top, fmaxf(x < __builtin_inff() ? x : 0.f, y < __builtin_inff() ? y : 0.f));
  }
  return top;
}

// What rounding to T took off 8 values; nothing of those that it made infinite.
template <class T>
__device__ __forceinline__ void rest8(float* v) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float left = v[e] - (float)(T)v[e];
    v[e] = fabsf(left) < __builtin_inff() ? left : 0.f;
  }
}

// dz and its column sums, bound by memory: three values in, two out (16384 rows of 2 x 2048 61 us, 5.5 TB/s).  A
// workgroup has up to 256 pieces of 8 columns (blockIdx.x) and as many of its part's rows at a time as its
// threads cover.  The products take dz in 16 bits, and sums over many rows and columns average what that loses: dx and the
// weights' gradients are sqrt(2) times as far off as rounding them alone makes them.  Of few rows they may
// be further off (one row of 384 features 1.66 times), so there dz's rounding errors are 16-bit rows of their own, behind
// its rows: up to 32 rows the products' tiles and stages of 64 hold both without another one (23 x 2 x 1536, k = 384: 26 us
// both ways; 32 x 2 x 4096, k = 1024: 32 for 27).
template <class T, bool REFIT>
__global__ __launch_bounds__(kBlock) void gated_grad_kernel(GatedGradArgs a) {
  __shared__ float red[kBlock * 8];
  const int64_t wg = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  float lift = kFits<T> ? 1.f : (float)(1 << kDzLift), peak = 0.f;
  if constexpr (REFIT) {
    const int64_t all = (int64_t)gridDim.x * gridDim.y;
    float top = 0.f;
    for (int64_t t = threadIdx.x; t < all; t += kBlock) top = fmaxf(top, a.peaks[t]);
    top = workgroup_max(top, red);
    const bool fits = top == 0.f || (top * lift < 32768.f && top * lift >= 0.25f);
    if (!fits) lift = ldexpf(1.f, min(15 - __builtin_amdgcn_frexp_expf(top), 60));
    if (wg == 0 && threadIdx.x == 0) *a.unit = 1.f / lift;
    if (fits) return;
  }
  const int width = gated_grad_width(a.m, a.n);
  const int pieces = min(a.n / 8 - (int)blockIdx.x * width, width), lanes = kBlock / pieces;
  const int p = threadIdx.x % pieces, rl = threadIdx.x / pieces;
  const int c = (blockIdx.x * width + p) * 8;
  float sum[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[0][e] = sum[1][e] = 0.f;
  const int64_t r0 = a.m * blockIdx.y / gridDim.y, r1 = a.m * (blockIdx.y + 1) / gridDim.y;
  if (rl < lanes) {
    constexpr int U = 4;  // rows under way
    for (int64_t r = r0 + rl; r < r1; r += U * lanes) {
      typename Frag<T>::V d[U], g[U], z[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = min(r + u * lanes, r1 - 1);
        d[u] = *reinterpret_cast<const typename Frag<T>::V*>((const T*)a.dy + row * a.dy_stride + c);
        g[u] = *reinterpret_cast<const typename Frag<T>::V*>((const T*)a.pre + row * 2 * a.n + c);
        z[u] = *reinterpret_cast<const typename Frag<T>::V*>((const T*)a.pre + row * 2 * a.n + a.n + c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = r + u * lanes;
        if (row < r1) {
          float df[8], gf[8], uf[8], dg[8], du[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) df[e] = (float)d[u][e], gf[e] = (float)g[u][e], uf[e] = (float)z[u][e];
          gate_grads8(df, gf, uf, a.act, dg, du);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[0][e] += dg[e], sum[1][e] += du[e];
          if constexpr (!kFits<T>) {
            if constexpr (!REFIT) peak = fmaxf(peak, finite_max8(dg, du));
#pragma unroll
            for (int e = 0; e < 8; ++e) dg[e] *= lift, du[e] *= lift;
          }
          store8((T*)a.dz + row * 2 * a.n + c, dg);
          store8((T*)a.dz + row * 2 * a.n + a.n + c, du);
          if (a.rests) {
            rest8<T>(dg), rest8<T>(du);
            store8((T*)a.dz + (a.m + row) * 2 * a.n + c, dg);
            store8((T*)a.dz + (a.m + row) * 2 * a.n + a.n + c, du);
          }
        }
      }
    }
  }
  if constexpr (REFIT) return;
  if constexpr (!kFits<T>) {
    peak = workgroup_max(peak, red);
    if (threadIdx.x == 0) a.peaks[wg] = peak;
  }
  if (a.rests && a.x != nullptr) {
    const int64_t pieces_x = a.k / 8, all = a.m * pieces_x, step = (int64_t)gridDim.x * kBlock;
    for (int64_t t = (int64_t)blockIdx.x * kBlock + threadIdx.x; t < all; t += step) {
      const u32x4 v = *reinterpret_cast<const u32x4*>((const T*)a.x + t / pieces_x * a.x_stride + t % pieces_x * 8);
      reinterpret_cast<u32x4*>(a.twice)[t] = v;
      reinterpret_cast<u32x4*>(a.twice)[all + t] = v;
    }
  }
  if (a.dgate_bias == nullptr && a.dup_bias == nullptr) return;
  const int64_t col0 = (int64_t)blockIdx.x * width * 8;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) red[threadIdx.x * 8 + e] = sum[u][e];
    __syncthreads();
    T* out = (T*)(u == 0 ? a.dgate_bias : a.dup_bias);
    for (int t = threadIdx.x; t < pieces * 8; t += kBlock) {
      float s = 0.f;
      for (int l = 0; l < lanes; ++l) s += red[l * pieces * 8 + t];
      if (gridDim.y > 1)
        a.partial[((int64_t)blockIdx.y * 2 + u) * a.n + col0 + t] = s;
      else if (out != nullptr)
        out[col0 + t] = (T)s;
    }
  }
}

}  // namespace

// Tiles of 256 x (128 + 128) (8 waves, one workgroup a CU), 128 x (64 + 64) (two) and 64 x (64 + 64) (two),
// with the costs of plan_gemm's products of as many blocks.  16384 x 2 x 2048, k = 768, three results: 127 us, 0.81 PFLOP/s,
// of the first passes, 144 to 159 of those after them; 10007 x 2 x 2664, k = 1000: 143 us, 0.75; 23 x 2 x 1536, k = 384: 6.6 us,
// a launch's latency; dx of two sums 16384 x 768, k = 2 x 2048 115 us, 0.89.  The clock falls under load, to 2.1 to 2.2 of
// 2.4 GHz, and the matrix cores are busy in 30 to 35% of its cycles: a wave waits 37% of its time at barriers and for loads, and
// 38% for an instruction's turn (a stage is 64 steps of a short reduction, and no other workgroup's work is on the CU).
GemmPlan plan_gated(int64_t m, int64_t n, int64_t k, int cus) {
  static constexpr TileChoice kTiles[] = {{256, 128, 1, 512, 1.8}, {128, 64, 2, 256, 1.2}, {64, 64, 2, 256, 0.9}};
  return plan_tiles(kTiles, 3, m, n, (k + kDepth - 1) / kDepth, 2, cus);
}

hipError_t launch_gated(const GemmKindArgs& a, const GemmPlan& p, hipStream_t s) {
  return a.type == kF16 ? gated<_Float16>(a, p, s) : gated<__bf16>(a, p, s);
}

GemmPlan plan_two_parts(int64_t m, int64_t n, int64_t k, bool rests, int cus) {
  static constexpr TileChoice kTiles[] = {{256, 256, 1, 512, 1.8}, {256, 192, 1, 512, 1.7}, {128, 128, 2, 256, 1.2}, {64, 64, 3, 256, 0.9}};
  GemmPlan p = plan_tiles(kTiles, 4, m, n, 2 * ((k + kDepth - 1) / kDepth), 1, cus);
  if (rests && p.splits == 1) p.splits = 2, p.ws_bytes = 2 * m * n * 4;  // (the join adds the halves; there are two stages at least)
  return p;
}

hipError_t launch_two_parts(const GemmKindArgs& a, const GemmPlan& p, bool rests, hipStream_t s) {
  const int halves = rests ? 2 : 1;
  return a.type == kF16 ? sums<_Float16, kTwoParts>(a, p, halves, s) : sums<__bf16, kTwoParts>(a, p, halves, s);
}

hipError_t launch_weights(const GemmKindArgs& a, const GemmPlan& p, hipStream_t s) {
  return a.type == kF16 ? sums<_Float16, kWeights>(a, p, 1, s) : sums<__bf16, kWeights>(a, p, 1, s);
}

int64_t gated_grad_workgroups(int64_t m, int64_t n, int parts) {
  const int64_t width = gated_grad_width(m, (int)n);
  return (n / 8 + width - 1) / width * parts;
}

int gated_grad_parts(int64_t m, int64_t n, int cus) {
  if (m <= 256) return 1;
  const int64_t width = gated_grad_width(m, (int)n);
  const int64_t blocks = (n / 8 + width - 1) / width, lanes = kBlock / width;
  return (int)std::max<int64_t>(1, std::min<int64_t>((m + lanes - 1) / lanes, 3 * cus / blocks));
}

hipError_t launch_gated_grad(const GatedGradArgs& a, hipStream_t s) {
  const int width = gated_grad_width(a.m, a.n);
  const dim3 grid((a.n / 8 + width - 1) / width, a.parts), block(kBlock);
  if (a.type == kF16) {
    hipLaunchKernelGGL((gated_grad_kernel<_Float16, false>), grid, block, 0, s, a);
    hipLaunchKernelGGL((gated_grad_kernel<_Float16, true>), grid, block, 0, s, a);
  } else {
    hipLaunchKernelGGL((gated_grad_kernel<__bf16, false>), grid, block, 0, s, a);
  }
  hipError_t e = hipGetLastError();
  const int first = a.dgate_bias != nullptr ? a.n : 0, second = a.dup_bias != nullptr ? a.n : 0;
  if (e == hipSuccess && a.parts > 1 && first + second > 0)
    e = launch_column_sums(a.partial + (first > 0 ? 0 : a.n), a.parts, 2 * a.n, first > 0 ? first : second, first > 0 ? second : 0,
                           a.type, first > 0 ? a.dgate_bias : a.dup_bias, first > 0 ? a.dup_bias : nullptr, s);
  return e;
}

}  // namespace cvs
