// Matrix product of 8-bit whole numbers: each row of x (a token) is taken in units of
// its own scale, each row of the weight (a channel) comes in units of its own, and
//
//   y[i, j] = act(sx_i sw_j sum_r qx(i, r) qw(j, r) + bias[j]) + residual[i, j],
//   sx_i = max_r |x(i, r)| / 127,  qx(i, r) = x(i, r) / sx_i to the nearest whole number, ties to the even one.
//
// The sum is whole and exact in 32 bits up to k = 2^17 (127 * 128 * 2^17 < 2^31), in any order.
#include <algorithm>

#include "cvs_gemm_tile.h"

namespace cvs {

namespace {

// The largest magnitude of 16-bit floats by their bits: NaN and infinities come out on top.
template <class T>
struct Top;
template <>
struct Top<_Float16> {
  static constexpr uint32_t kInf = 0x7c00;
  static __device__ __forceinline__ float value(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits); }
};
template <>
struct Top<__bf16> {
  static constexpr uint32_t kInf = 0x7f80;
  static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits << 16); }
};

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ u16x2 top_of(const u32x4& v, u16x2 top) {
#pragma unroll
  for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[e] & 0x7fff7fffu));
  return top;
}

// A row's scale and what turns its values into whole numbers.  The quotient 127 x / top is exact
// where it is a tie: 127 x is (18 bits), the division's remainder too, and one step of it from the
// reciprocal's estimate leaves an error far below a tie's distance from any other quotient (2^-12 at
// least: top has 11 bits).  Both are brought to where top is 0.5 to 1, out of the subnormals.
struct RowUnit {
  float scale, top, inv;
  int shift;
  bool finite;

  template <class T>
  __device__ __forceinline__ static RowUnit of(uint32_t bits) {
    RowUnit u;
    u.finite = bits < Top<T>::kInf;
    const float top = u.finite ? Top<T>::value(bits) : 0.f;
    u.scale = u.finite ? top / 127.f : __builtin_nanf("");
    u.shift = -__builtin_amdgcn_frexp_expf(top);
    u.top = ldexpf(top, u.shift);
    u.inv = top > 0.f ? __builtin_amdgcn_rcpf(u.top) : 0.f;
    return u;
  }
  // The whole number in the low byte (of the sum with 1.5 * 2^23, whose spacing is 1).
  __device__ __forceinline__ uint32_t whole(float x) const {
    const float t = 127.f * ldexpf(x, shift);
    const float q = t * inv;
    return __float_as_uint(fmaf(fmaf(-q, top, t), inv, q) + 12582912.f);
  }
  template <class T>
  __device__ __forceinline__ u32x4 whole16(const u32x4& lo, const u32x4& hi) const {
    const auto a = __builtin_bit_cast(typename Frag<T>::V, lo), b = __builtin_bit_cast(typename Frag<T>::V, hi);
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = whole((float)(e < 2 ? a[4 * e + i] : b[4 * e - 8 + i]));
      const uint32_t low = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400u), high = __builtin_amdgcn_perm(w[3], w[2], 0x04000c0cu);
      r[e] = finite ? low | high : 0u;
    }
    return r;
  }
};

// Rows of up to 1024 P values, a wave each, held in registers.  Bound by memory: 10007 x 2048 12.2 us, 5.0 TB/s,
// 32768 x 1024 26.4 us, 3.8.
template <class T, int P>
__global__ __launch_bounds__(kBlock) void quantize_kernel(QuantArgs a) {
  const int64_t row = (int64_t)blockIdx.x * (kBlock / kWave) + (threadIdx.x >> 6);
  if (row >= a.n) return;
  const int lane = threadIdx.x & 63;
  const T* x = (const T*)a.x + row * a.x_stride;
  u32x4 lo[P], hi[P];
  u16x2 top = {0, 0};
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int c = (p * 64 + lane) * 16;
    lo[p] = hi[p] = u32x4{0, 0, 0, 0};
    if (c < a.d) {
      lo[p] = *reinterpret_cast<const u32x4*>(x + c);
      hi[p] = *reinterpret_cast<const u32x4*>(x + c + 8);
    }
  }
#pragma unroll
  for (int p = 0; p < P; ++p) top = top_of(hi[p], top_of(lo[p], top));
  uint32_t bits = max((uint32_t)top[0], (uint32_t)top[1]);
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, s));
  const RowUnit u = RowUnit::of<T>(bits);
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int c = (p * 64 + lane) * 16;
    if (c < a.d) *reinterpret_cast<u32x4*>(a.values + row * a.d + c) = u.whole16<T>(lo[p], hi[p]);
  }
  if (lane == 0) a.scales[row] = u.scale;
}

// Longer rows, a workgroup each, read twice.
template <class T>
__global__ __launch_bounds__(kBlock) void quantize_long_kernel(QuantArgs a) {
  __shared__ uint32_t tops[4];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.x_stride;
  u16x2 top = {0, 0};
  for (int c = threadIdx.x * 16; c < a.d; c += kBlock * 16)
    top = top_of(*reinterpret_cast<const u32x4*>(x + c + 8), top_of(*reinterpret_cast<const u32x4*>(x + c), top));
  uint32_t bits = max((uint32_t)top[0], (uint32_t)top[1]);
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, s));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = bits;
  __syncthreads();
  const RowUnit u = RowUnit::of<T>(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
  for (int c = threadIdx.x * 16; c < a.d; c += kBlock * 16)
    *reinterpret_cast<u32x4*>(a.values + row * a.d + c) =
        u.whole16<T>(*reinterpret_cast<const u32x4*>(x + c), *reinterpret_cast<const u32x4*>(x + c + 8));
  if (threadIdx.x == 0) a.scales[row] = u.scale;
}

template <class T>
void quantize(const QuantArgs& a, hipStream_t s) {
  const dim3 waves((unsigned)((a.n + 3) / 4)), block(kBlock);
  if (a.d <= 1024)
    hipLaunchKernelGGL((quantize_kernel<T, 1>), waves, block, 0, s, a);
  else if (a.d <= 2048)
    hipLaunchKernelGGL((quantize_kernel<T, 2>), waves, block, 0, s, a);
  else if (a.d <= 4096)
    hipLaunchKernelGGL((quantize_kernel<T, 4>), waves, block, 0, s, a);
  else
    hipLaunchKernelGGL(quantize_long_kernel<T>, dim3((unsigned)a.n), block, 0, s, a);
}

// Few rows (single tokens, a query), one launch: a workgroup has 32 columns of the weight, its waves a quarter of
// their depth each, straight from memory to the matrix cores, and takes all rows in whole numbers itself, while the
// weight is on its way.  Bound by latency: a launch, the rows, the weight (loaded together), and the waves' join; 7.2 us
// of 1 x 2048, k = 768, 8.2 of 23 x 1536, k = 384.
//
// Calls of it (one after the other, bound by the host or the GPU) against the quantising launch and the tiles, us:
//   up to 1024 values a row   32 x 256, k = 768 9.1, 13.0; 32 x 8192, k = 1024 9.5, 13.0; 16 x 16384, k = 1024 10.1, 13.1;
//                             32 x 16384, k = 1024 12.4, 12.9; 1 x 24576, k = 1024 12.4, 12.6; 8 x 32768, k = 768 14.2, 12.4;
//                             1 x 131072, k = 768 44.3, 23.8: every workgroup takes all the rows, so the columns may
//                             fill the CUs once, or twice of half as many rows;
//   up to 2048, read twice    18 x 768, k = 1040 12.7, 12.9; 18 x 8192, k = 1920 12.1, 13.0; 20 x 768, k = 1040 14.6, 12.8;
//                             24 x 512, k = 1280 13.3, 13.0; 32 x 4096, k = 1792 14.4, 12.9; 8 x 16384, k = 2048 13.0, 12.6;
//   and tiles in parts        28 x 8192, k = 2048 14.9, 15.7 (a third launch joins them);
//   deeper                    8 x 4096, k = 4096 16.6, 16.0; 4 x 2048, k = 8192 23.2, 16.0.
// (In a captured graph, where launches cost the host nothing, the tiles are ahead from some 16 rows: 32 x 4096, k = 1024 8.9, 7.6.)
constexpr int kFewRows = 32;     // columns of a block
constexpr int kFewDepth = 2048;  // the weight past the first 1024 values of a row comes after the rows

// Bytes of LDS between rows: depth padded to whole blocks of 128 (four waves' 32), and 16 so that rows start in other banks.
__host__ __device__ inline int few_stride(int d) { return (d + 127) / 128 * 128 + 16; }

template <class T>
__global__ __launch_bounds__(kBlock) void int8_rows_kernel(GemmKindArgs a, const void* x, int64_t x_stride, int d) {
  extern __shared__ __attribute__((aligned(16))) unsigned char rows[];  // [m][few_stride]; then the waves' sums
  __shared__ float scale[kFewRows];
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int stride = few_stride(d), n0 = blockIdx.x * 32;
  const int steps = (d + 127) / 128;  // blocks of 32 values of each wave
  constexpr int AHEAD = 8;            // the weight's first loads, under way before the rows are looked at
  const unsigned char* w = (const unsigned char*)a.N + (int64_t)min(n0 + tile_row(l32), a.n - 1) * d;
  auto weight = [&](int s) -> i32x4 {
    const int c = (s * 4 + wave) * 32 + 16 * g;
    i32x4 v = {0, 0, 0, 0};
    if (c < d) v = *reinterpret_cast<const i32x4*>(w + c);
    return v;
  };
  // the epilogue's: 8 columns a thread of the first 128
  const int half = threadIdx.x >> 6 & 1, i = l32, j = n0 + 16 * half + 8 * g;
  const bool mine = threadIdx.x < 128 && i < a.m && j < a.n;
  typename Frag<T>::V bias = {}, res = {};
  f32x4 col[2] = {};
  if (mine) {
    col[0] = *reinterpret_cast<const f32x4*>(a.col_scale + j);
    col[1] = *reinterpret_cast<const f32x4*>(a.col_scale + j + 4);
    if (a.bias != nullptr) bias = *reinterpret_cast<const typename Frag<T>::V*>((const T*)a.bias + j);
    if (a.residual != nullptr) res = *reinterpret_cast<const typename Frag<T>::V*>((const T*)a.residual + (int64_t)i * a.ld_res + j);
  }
  i32x4 first[AHEAD];
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) first[s] = s < steps ? weight(s) : i32x4{0, 0, 0, 0};

  // this wave's rows, every fourth: their loads go together (and again where a row is longer than a wave)
  constexpr int R = kFewRows / 4;
  u32x4 lo[R], hi[R];
  auto load = [&](int c) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      lo[r] = hi[r] = u32x4{0, 0, 0, 0};
      if (wave + 4 * r < a.m && c < d) {
        const T* row = (const T*)x + (wave + 4 * r) * x_stride + c;
        lo[r] = *reinterpret_cast<const u32x4*>(row);
        hi[r] = *reinterpret_cast<const u32x4*>(row + 8);
      }
    }
  };
  u16x2 top[R];
#pragma unroll
  for (int r = 0; r < R; ++r) top[r] = u16x2{0, 0};
  for (int c = lane * 16; c < d + lane * 16; c += 1024) {
    load(c);
#pragma unroll
    for (int r = 0; r < R; ++r) top[r] = top_of(hi[r], top_of(lo[r], top[r]));
  }
  RowUnit unit[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    uint32_t bits = max((uint32_t)top[r][0], (uint32_t)top[r][1]);
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, s));
    unit[r] = RowUnit::of<T>(bits);
    if (lane == 0 && wave + 4 * r < a.m) scale[wave + 4 * r] = unit[r].scale;
  }
  for (int c = lane * 16; c < stride - 16 + lane * 16; c += 1024) {
    if (d > 1024) load(c);
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (wave + 4 * r < a.m && c < stride - 16)
        *reinterpret_cast<u32x4*>(rows + (wave + 4 * r) * stride + c) = unit[r].whole16<T>(lo[r], hi[r]);
  }
  __syncthreads();

  i32x16 sum;
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] = 0;
  const unsigned char* from = rows + min(l32, a.m - 1) * stride + wave * 32 + 16 * g;
  auto multiply = [&](int s, i32x4 v) {
    sum = __builtin_amdgcn_mfma_i32_32x32x32_i8(v, *reinterpret_cast<const i32x4*>(from + s * 128), sum, 0, 0, 0);
  };
#pragma unroll
  for (int s = 0; s < AHEAD; ++s)
    if (s < steps) multiply(s, first[s]);
  for (int s = AHEAD; s < steps; s += AHEAD) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) first[u] = s + u < steps ? weight(s + u) : i32x4{0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (s + u < steps) multiply(s + u, first[u]);
  }
  __syncthreads();  // the rows have been read
  // lane: row l32's columns 8 g .. 8 g + 7 and 16 + those
  i32x4* sums = reinterpret_cast<i32x4*>(rows);  // [wave][16-byte piece][lane]
#pragma unroll
  for (int q = 0; q < 4; ++q) sums[(wave * 4 + q) * 64 + lane] = i32x4{sum[4 * q], sum[4 * q + 1], sum[4 * q + 2], sum[4 * q + 3]};
  __syncthreads();
  if (!mine) return;
  float z[8], scales[8], add[8];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    i32x4 t = sums[(2 * half + q) * 64 + lane];
#pragma unroll
    for (int v = 1; v < 4; ++v) t += sums[(v * 4 + 2 * half + q) * 64 + lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[4 * q + e] = (float)t[e], scales[4 * q + e] = col[q][e], add[4 * q + e] = (float)bias[4 * q + e];
  }
  finish_int8(a.act, scale[i], scales, add, z);
  if (a.residual != nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += (float)res[e];
  }
  store8((T*)a.out + (int64_t)i * a.n + j, z);
}

template <class T, int WM, int WN, int BM, int BN, int RING, int WGS>
__global__ __launch_bounds__(64 * WM * WN, WGS) void gemm_int8_kernel(GemmKindArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[gemm_lds<WM, WN, BM, BN, RING>()];
  __shared__ __attribute__((aligned(16))) float vectors[gemm_vectors<kInt8, WM * BM * 32, WN * BN * 32>()];
  gemm_tile<T, WM, WN, BM, BN, RING, false, false, kInt8>(a, blockIdx.x, smem, vectors);
}

// Adds the parts of a split reduction and finishes: 8 columns a thread.
template <class T>
__global__ __launch_bounds__(kBlock) void int8_join_kernel(GemmKindArgs a) {
  const int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  const int pieces = a.n / 8;
  const int64_t i = at / pieces;
  if (i >= a.m) return;
  const int j = (int)(at - i * pieces) * 8;
  const int64_t plane = (int64_t)a.m * a.n;
  i32x4 lo = {0, 0, 0, 0}, hi = lo;
  const float* p = a.partial + i * a.n + j;
  for (int s = 0; s < a.splits; ++s, p += plane) {
    lo += *reinterpret_cast<const i32x4*>(p);
    hi += *reinterpret_cast<const i32x4*>(p + 4);
  }
  float z[8], col[8], more[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) z[e] = (float)lo[e], z[4 + e] = (float)hi[e], more[e] = more[4 + e] = 0.f;
  take8(a.col_scale + j, col);
  if (a.bias != nullptr) load8((const T*)a.bias + j, more);
  finish_int8(a.act, a.row_scale[i], col, more, z);
  if (a.residual != nullptr) {
    load8((const T*)a.residual + i * a.ld_res + j, more);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += more[e];
  }
  store8((T*)a.out + i * a.n + j, z);
}

template <class T, int WM, int WN, int BM, int BN, int RING, int WGS>
void launch_tiles(const GemmKindArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((gemm_int8_kernel<T, WM, WN, BM, BN, RING, WGS>), dim3(gemm_grid(a, WM * BM * 32, WN * BN * 32)),
                     dim3(64 * WM * WN), 0, s, a);
}

template <class T>
hipError_t product(const GemmKindArgs& a, const GemmPlan& p, hipStream_t s) {
  if (p.tile == 256 && p.tile_n == 256)
    launch_tiles<T, 4, 2, 2, 4, 2, 1>(a, s);
  else if (p.tile == 256)
    launch_tiles<T, 4, 2, 2, 3, 2, 1>(a, s);
  else if (p.tile == 128)
    launch_tiles<T, 2, 2, 2, 2, 2, 2>(a, s);
  else
    launch_tiles<T, 2, 2, 1, 1, 3, 2>(a, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL(int8_join_kernel<T>, dim3((unsigned)(((int64_t)a.m * (a.n / 8) + kBlock - 1) / kBlock)), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize(const QuantArgs& a, hipStream_t s) {
  if (a.type == kF16)
    quantize<_Float16>(a, s);
  else
    quantize<__bf16>(a, s);
  return hipGetLastError();
}

// plan_gemm's tiles: a stage of 64 16-bit units is 128 values.  10007 x 768, k = 2048 in 128 x 128 tiles 24 us, 1.3 POP/s;
// 32768 x 4096, k = 1024 in 256 x 256 tiles 215 to 230 us, 1.2 to 1.3 POP/s: 2.1 to 2.2 of 2.4 GHz, of whose cycles the matrix
// cores are busy in 27%; a wave waits 35% of its time at barriers and for loads, and vector instructions are 26%.
GemmPlan plan_int8(int64_t m, int64_t n, int64_t k, int cus) {
  static constexpr TileChoice kTiles[] = {{256, 256, 1, 512, 1.8}, {256, 192, 1, 512, 1.7}, {128, 128, 2, 256, 1.2}, {64, 64, 3, 256, 0.9}};
  return plan_tiles(kTiles, 4, m, n, (k / 2 + kDepth - 1) / kDepth, 1, cus);
}

bool int8_few_rows(int64_t m, int64_t n, int64_t k, const GemmPlan& tiles, int cus) {
  const int64_t rounds = ((n + 31) / 32 + cus - 1) / cus;
  if (k <= 1024) return rounds <= 2 && m * rounds <= kFewRows;
  return k <= kFewDepth && rounds == 1 && m <= (tiles.splits > 1 ? 28 : 18);  // (57 KiB of rows at most)
}

hipError_t launch_int8_rows(const GemmKindArgs& a, const void* x, int64_t x_stride, int d, hipStream_t s) {
  const dim3 grid((unsigned)((a.n + 31) / 32)), block(kBlock);
  const size_t lds = std::max(a.m * few_stride(d), 4 * 4096);
  if (a.type == kF16)
    hipLaunchKernelGGL(int8_rows_kernel<_Float16>, grid, block, lds, s, a, x, x_stride, d);
  else
    hipLaunchKernelGGL(int8_rows_kernel<__bf16>, grid, block, lds, s, a, x, x_stride, d);
  return hipGetLastError();
}

hipError_t launch_int8(const GemmKindArgs& a, const GemmPlan& p, hipStream_t s) {
  return a.type == kF16 ? product<_Float16>(a, p, s) : product<__bf16>(a, p, s);
}

}  // namespace cvs
