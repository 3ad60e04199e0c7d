// Matrix product with bias, activation and residual in its epilogue, and the
// products of its backward pass, for 16-bit operands with fp32 sums (the tile is
// in cvs_gemm_tile.h).
#include <algorithm>

#include "cvs_gemm_tile.h"

namespace cvs {

namespace {

constexpr int64_t kLaunchThreads = (int64_t)1 << 32;

template <class T, int WM, int WN, int BM, int BN, int RING, bool MS, bool NS>
__global__ __launch_bounds__(64 * WM * WN, (WM * BM + WN * BN) * RING <= 16 ? 2 : 1) void gemm_kernel(GemmArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[gemm_lds<WM, WN, BM, BN, RING>()];
  gemm_tile<T, WM, WN, BM, BN, RING, MS, NS>(a, blockIdx.x, smem);
}

// Two products that share an operand, dx (first) and dW, in one launch: neither fills the GPU
// where the rows are few.
template <class T, int WM, int WN, int BM, int BN, int RING>
__global__ __launch_bounds__(64 * WM * WN, (WM * BM + WN * BN) * RING <= 16 ? 2 : 1) void gemm_pair_kernel(GemmArgs a, GemmArgs b) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[gemm_lds<WM, WN, BM, BN, RING>()];
  const int first = gemm_grid(a, WM * BM * 32, WN * BN * 32);
  if ((int)blockIdx.x < first)
    gemm_tile<T, WM, WN, BM, BN, RING, false, true>(a, blockIdx.x, smem);
  else
    gemm_tile<T, WM, WN, BM, BN, RING, true, true>(b, blockIdx.x - first, smem);
}

// Adds the parts of a split reduction, in order, and finishes: 8 columns a thread.
template <class T>
__global__ __launch_bounds__(kBlock) void gemm_join_kernel(GemmArgs a) {
  const int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  const int pieces = a.n / 8;
  const int64_t i = at / pieces;
  if (i >= a.m) return;
  const int j = (int)(at - i * pieces) * 8;
  const int64_t plane = (int64_t)a.m * a.n;
  const float* p = a.partial + i * a.n + j;
  float z[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] = 0.f;
  for (int s = 0; s < a.splits; ++s, p += plane) {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] += lo[e], z[4 + e] += hi[e];
  }
  float pre[8];
  finish8<T>(a, (int)i, j, z, pre);
  if (a.pre != nullptr) store8((T*)a.pre + i * a.n + j, pre);
  store8((T*)a.out + i * a.n + j, z);
}

template <class T>
hipError_t launch_join(const GemmArgs& a, hipStream_t s) {
  const int64_t threads = (int64_t)a.m * (a.n / 8);
  hipLaunchKernelGGL((gemm_join_kernel<T>), dim3((unsigned)((threads + kBlock - 1) / kBlock)), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

template <class T, int WM, int WN, int BM, int BN, int RING>
hipError_t launch_tiles(const GemmArgs& a, hipStream_t s) {
  const dim3 grid(gemm_grid(a, WM * BM * 32, WN * BN * 32)), block(64 * WM * WN);
  if (a.m_strided && a.n_strided)
    hipLaunchKernelGGL((gemm_kernel<T, WM, WN, BM, BN, RING, true, true>), grid, block, 0, s, a);
  else if (a.n_strided)
    hipLaunchKernelGGL((gemm_kernel<T, WM, WN, BM, BN, RING, false, true>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((gemm_kernel<T, WM, WN, BM, BN, RING, false, false>), grid, block, 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess && a.splits > 1 ? launch_join<T>(a, s) : e;
}

template <class T, int WM, int WN, int BM, int BN, int RING>
hipError_t launch_pair(const GemmArgs& a, const GemmArgs& b, hipStream_t s) {
  constexpr int TM = WM * BM * 32, TN = WN * BN * 32;
  hipLaunchKernelGGL((gemm_pair_kernel<T, WM, WN, BM, BN, RING>), dim3(gemm_grid(a, TM, TN) + gemm_grid(b, TM, TN)),
                     dim3(64 * WM * WN), 0, s, a, b);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.splits > 1) e = launch_join<T>(a, s);
  if (e == hipSuccess && b.splits > 1) e = launch_join<T>(b, s);
  return e;
}

template <class T>
hipError_t launch_typed(const GemmArgs& a, const GemmPlan& p, hipStream_t s) {
  if (p.tile == 256) return p.tile_n == 256 ? launch_tiles<T, 4, 2, 2, 4, 2>(a, s) : launch_tiles<T, 4, 2, 2, 3, 2>(a, s);
  if (p.tile == 128) return launch_tiles<T, 2, 2, 2, 2, 2>(a, s);
  return launch_tiles<T, 2, 2, 1, 1, 3>(a, s);
}

template <class T>
hipError_t launch_typed_pair(const GemmArgs& a, const GemmArgs& b, const GemmPlan& p, hipStream_t s) {
  if (p.tile == 128) return launch_pair<T, 2, 2, 2, 2, 2>(a, b, s);
  return launch_pair<T, 2, 2, 1, 1, 3>(a, b, s);
}

// Pieces of 8 columns of a workgroup of act_grad_kernel: few for few rows, which one part then
// has, so that it writes dbias itself.
__host__ __device__ inline int act_grad_width(int64_t m, int n) { return m <= 256 ? 16 : min(n / 8, kBlock); }

// dz = dy act'(pre) and its column sums, bound by memory.  A workgroup has up to 256
// pieces of 8 columns (blockIdx.x) and as many of its part's rows at a time as its threads
// cover; it adds its row lanes' sums in LDS and writes one partial row.
template <class T>
__global__ __launch_bounds__(kBlock) void act_grad_kernel(ActGradArgs a) {
  __shared__ float red[kBlock * 8];
  const int width = act_grad_width(a.m, a.n);
  const int pieces = min(a.n / 8 - (int)blockIdx.x * width, width), lanes = kBlock / pieces;
  const int p = threadIdx.x % pieces, rl = threadIdx.x / pieces;
  const int c = (blockIdx.x * width + p) * 8;
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  const int64_t r0 = a.m * blockIdx.y / gridDim.y, r1 = a.m * (blockIdx.y + 1) / gridDim.y;
  if (rl < lanes) {
    const bool act = a.act != kActNone;
    constexpr int U = 4;  // rows under way
    for (int64_t r = r0 + rl; r < r1; r += U * lanes) {
      typename Frag<T>::V g[U], z[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = min(r + u * lanes, r1 - 1);
        g[u] = *reinterpret_cast<const typename Frag<T>::V*>((const T*)a.dy + row * a.dy_stride + c);
        if (act) z[u] = *reinterpret_cast<const typename Frag<T>::V*>((const T*)a.pre + row * a.n + c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = r + u * lanes;
        if (row < r1) {
          float gf[8], zf[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) gf[e] = (float)g[u][e];
          if (act) {
#pragma unroll
            for (int e = 0; e < 8; ++e) zf[e] = (float)z[u][e];
            times_slope8(gf, zf, a.act);
            store8((T*)a.dz + row * a.n + c, gf);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] += gf[e];
        }
      }
    }
  }
  if (a.dbias == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[threadIdx.x * 8 + e] = sum[e];
  __syncthreads();
  const int64_t col0 = (int64_t)blockIdx.x * width * 8;
  for (int t = threadIdx.x; t < pieces * 8; t += kBlock) {
    float s = 0.f;
    for (int l = 0; l < lanes; ++l) s += red[l * pieces * 8 + t];
    if (gridDim.y == 1)
      ((T*)a.dbias)[col0 + t] = (T)s;
    else
      a.partial[(int64_t)blockIdx.y * a.n + col0 + t] = s;
  }
}

}  // namespace

// Tiles of 256 x 256 and 256 x 192 (8 waves, one workgroup a CU), 128 x 128 and 64 x 64 (4 waves,
// two and three workgroups a CU), and parts of the reduction where the tiles leave CUs idle: the
// choice of least estimated time.  A CU runs its workgroups in rounds; every XCD has an eighth of
// the tiles, rounded up, and all their parts (33 tiles in 7 parts are 35 workgroups on 32 CUs, two
// rounds: 100 us where 128 x 128 takes 60).  A stage of a round costs what was
// measured on long reductions (8192 x 8192, k = 2048: 1080, 850 and 480 TFLOP/s, that is 1.8 to
// 2.0, 1.2 and 0.9 us with 1, 2 and 3 workgroups; 256 x 192 has 1.7), a round 3 us more to fill
// and finish, and a split 3 us and its sums' way to memory and back.  At 16384 x 2048, k = 768
// that gives 256 x 256 (calls of the product alone, back to back: 54 us, with 128 x 128 58), at
// 16384 x 768, k = 2048 256 x 192 (its 256 tiles 48 us, 192 of 256 x 256 52), at 10007 x 768, k = 2048
// 128 x 128 (35, 256 x 256 47), at 2048 x 768, k = 16384 128 x 128 in 5 parts (61 with the join,
// 256 x 192 in parts 65).
//
// A launch has fewer than 2^32 threads: choices of more are passed over, and where that leaves none
// (splits 0), there is no plan.
GemmPlan plan_tiles(const TileChoice* choices, int count, int64_t m, int64_t n, int64_t stages, int sums, int cus) {
  GemmPlan best = {};
  double least = 1e30;
  for (const TileChoice* t = choices; t < choices + count; ++t) {
    const int64_t tiles = ((m + t->m - 1) / t->m) * ((n + t->n - 1) / t->n);
    for (int64_t splits = 1; splits <= 16 && (splits == 1 || splits * 8 <= stages); ++splits) {
      const int64_t wgs = (tiles + 7) / 8 * 8 * splits, full = wgs / (t->wgs * (int64_t)cus);
      if (wgs * t->threads >= kLaunchThreads || (splits > 1 && m * (n / 8) + kBlock > kLaunchThreads)) break;
      // a last round of few workgroups has more of a CU for each, but not below a stage's latency
      const int64_t rest = (wgs - full * t->wgs * cus + cus - 1) / cus;
      const double per = full * t->stage + (rest > 0 ? std::max(rest * t->stage / t->wgs, 0.5) : 0.0);
      double us = (stages + splits - 1) / splits * per + 3.0 * (full + (rest > 0));
      if (splits > 1) us += 3.0 + 2.0 * splits * m * n * sums * 4 / 4e6;
      if (us < least) {
        least = us;
        best.tile = t->m, best.tile_n = t->n, best.splits = (int)splits;
        best.ws_bytes = splits > 1 ? splits * m * n * sums * 4 : 0;
      }
    }
  }
  return best;
}

GemmPlan plan_gemm(int64_t m, int64_t n, int64_t k, int cus) {
  static constexpr TileChoice kTiles[] = {{256, 256, 1, 512, 1.8}, {256, 192, 1, 512, 1.7}, {128, 128, 2, 256, 1.2}, {64, 64, 3, 256, 0.9}};
  return plan_tiles(kTiles, 4, m, n, (k + kDepth - 1) / kDepth, 1, cus);
}

hipError_t launch_gemm(const GemmArgs& a, const GemmPlan& p, hipStream_t s) {
  return a.type == kF16 ? launch_typed<_Float16>(a, p, s) : launch_typed<__bf16>(a, p, s);
}

hipError_t launch_gemm_pair(const GemmArgs& a, const GemmPlan& pa, const GemmArgs& b, const GemmPlan& pb, hipStream_t s) {
  const int64_t both = (int64_t)gemm_grid(a, pa.tile, pa.tile_n) + gemm_grid(b, pb.tile, pb.tile_n);
  if (pa.tile == pb.tile && pa.tile < 256 && both * 256 < kLaunchThreads)
    return a.type == kF16 ? launch_typed_pair<_Float16>(a, b, pa, s) : launch_typed_pair<__bf16>(a, b, pa, s);
  const hipError_t e = launch_gemm(a, pa, s);
  return e == hipSuccess ? launch_gemm(b, pb, s) : e;
}

int act_grad_parts(int64_t m, int64_t n, int cus) {
  const int64_t width = act_grad_width(m, (int)n);
  if (m <= 256) return 1;
  const int64_t blocks = (n / 8 + width - 1) / width, lanes = kBlock / width;
  return (int)std::max<int64_t>(1, std::min<int64_t>((m + lanes - 1) / lanes, 3 * cus / blocks));
}

hipError_t launch_act_grad(const ActGradArgs& a, hipStream_t s) {
  const int width = act_grad_width(a.m, a.n);
  const dim3 grid((a.n / 8 + width - 1) / width, a.parts), block(kBlock);
  if (a.type == kF16)
    hipLaunchKernelGGL(act_grad_kernel<_Float16>, grid, block, 0, s, a);
  else
    hipLaunchKernelGGL(act_grad_kernel<__bf16>, grid, block, 0, s, a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.dbias != nullptr && a.parts > 1)
    e = launch_column_sums(a.partial, a.parts, a.n, a.n, 0, a.type, a.dbias, nullptr, s);
  return e;
}

}  // namespace cvs
