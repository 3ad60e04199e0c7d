// Layer norm of rows and its backward pass.
//
// Forward: y = (x - mean) rstd weight + bias, rstd = 1 / sqrt(mean((x - mean)^2) + eps).
// Backward, with xhat = (x - mean) rstd and g = dy weight:
//   dx = rstd (g - mean(g) - xhat mean(g xhat)), dweight = sum dy xhat, dbias = sum dy.
//
// Both are bound by memory: a row is read once, by one wave, and stays in its
// registers; the variance is the mean of squared differences (no cancellation),
// and every sum is fp32.  The backward pass's waves keep the columns' sums of all
// their rows in registers, a workgroup adds its waves' in LDS and writes one row of
// partial sums; a second launch adds those in a fixed order (no atomics).
#include <algorithm>

#include "cvs_common.h"
#include "cvs_encoder.h"

namespace cvs {

namespace {

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

template <class T, int VEC>
struct Vec {
  typedef T V __attribute__((ext_vector_type(VEC)));
};
template <class T>
struct Vec<T, 1> {
  typedef T V;
};

template <class T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  if constexpr (VEC == 1) {
    f[0] = (float)*p;
  } else {
    const auto v = *reinterpret_cast<const typename Vec<T, VEC>::V*>(p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = (float)v[j];
  }
}

template <class T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  if constexpr (VEC == 1) {
    *p = (T)f[0];
  } else {
    typename Vec<T, VEC>::V v;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (T)f[j];
    *reinterpret_cast<typename Vec<T, VEC>::V*>(p) = v;
  }
}

// One wave a row, P pieces of VEC columns a lane (23 x 384 in fp16: 3.7 us, latency).
template <class T, int VEC, int P>
__global__ __launch_bounds__(kBlock) void norm_forward_kernel(NormArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * (kBlock / kWave) + (threadIdx.x >> 6);
  if (row >= a.n) return;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
  const T* w = reinterpret_cast<const T*>(a.weight);
  const T* b = reinterpret_cast<const T*>(a.bias);
  float v[P][VEC];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (lane + 64 * i) * VEC;
    if (c < a.d) {
      load_vec<T, VEC>(x + c, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += v[i][j];
  const float inv_d = 1.f / (float)a.d;
  const float mean = wave_sum(s) * inv_d;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const bool in = (lane + 64 * i) * VEC < a.d;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      v[i][j] -= mean;
      if (in) q = fmaf(v[i][j], v[i][j], q);
    }
  }
  const float rstd = 1.f / sqrtf(wave_sum(q) * inv_d + a.eps);
  T* y = reinterpret_cast<T*>(a.y) + row * a.d;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (lane + 64 * i) * VEC;
    if (c < a.d) {
      float wf[VEC], bf[VEC], o[VEC];
      load_vec<T, VEC>(w + c, wf);
      if (b != nullptr) {
        load_vec<T, VEC>(b + c, bf);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) bf[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) o[j] = fmaf(v[i][j] * rstd, wf[j], bf[j]);
      store_vec<T, VEC>(y + c, o);
    }
  }
  if (a.mean != nullptr && lane == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < kBlock / kWave; ++w) t += scratch[w];
  return t;
}

// Rows wider than the registers hold: a workgroup a row, three passes over it.
template <class T>
__global__ __launch_bounds__(kBlock) void norm_forward_wide_kernel(NormArgs a) {
  __shared__ float scratch[kBlock / kWave];
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
  const T* w = reinterpret_cast<const T*>(a.weight);
  const T* b = reinterpret_cast<const T*>(a.bias);
  float s = 0.f;
  for (int c = threadIdx.x; c < a.d; c += kBlock) s += (float)x[c];
  const float inv_d = 1.f / (float)a.d;
  const float mean = block_sum(s, scratch) * inv_d;
  float q = 0.f;
  for (int c = threadIdx.x; c < a.d; c += kBlock) {
    const float t = (float)x[c] - mean;
    q = fmaf(t, t, q);
  }
  const float rstd = 1.f / sqrtf(block_sum(q, scratch) * inv_d + a.eps);
  T* y = reinterpret_cast<T*>(a.y) + row * a.d;
  for (int c = threadIdx.x; c < a.d; c += kBlock)
    y[c] = (T)fmaf(((float)x[c] - mean) * rstd, (float)w[c], b != nullptr ? (float)b[c] : 0.f);
  if (a.mean != nullptr && threadIdx.x == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

// Backward: workgroup g takes rows g * 4 + wave, then every 4 * gridDim.x further, a row's loads
// under way while the one before is summed.  16384 x 768 in bf16: 18 us, 4.2 TB/s (and 7 for the
// partial sums, which are latency); 50021 x 1000 in fp32: 116 us, 5.2 TB/s.
template <class T, int VEC, int P>
__global__ __launch_bounds__(kBlock) void norm_backward_kernel(NormArgs a) {
  constexpr int kWaves = kBlock / kWave;
  __shared__ float red[kWaves][64 * VEC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T* w = reinterpret_cast<const T*>(a.weight);
  float wf[P][VEC], dw[P][VEC], db[P][VEC];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (lane + 64 * i) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) wf[i][j] = dw[i][j] = db[i][j] = 0.f;
    if (c < a.d) load_vec<T, VEC>(w + c, wf[i]);
  }
  const float inv_d = 1.f / (float)a.d;
  const int64_t step = (int64_t)gridDim.x * kWaves;
  typename Vec<T, VEC>::V xr[P], gr[P];  // the next row, under way while this one is computed
  float mean_r = 0.f, rstd_r = 0.f;
  auto fetch = [&](int64_t row) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.dy_stride;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (lane + 64 * i) * VEC;
      if (c < a.d) {
        xr[i] = *reinterpret_cast<const typename Vec<T, VEC>::V*>(x + c);
        gr[i] = *reinterpret_cast<const typename Vec<T, VEC>::V*>(dy + c);
      }
    }
    mean_r = a.mean[row];
    rstd_r = a.rstd[row];
  };
  int64_t row = (int64_t)blockIdx.x * kWaves + wave;
  if (row < a.n) fetch(row);
  for (; row < a.n; row += step) {
    const float mean = mean_r, rstd = rstd_r;
    float h[P][VEC], g[P][VEC];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const bool in = (lane + 64 * i) * VEC < a.d;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if constexpr (VEC == 1) {
          h[i][j] = in ? (float)xr[i] : mean;
          g[i][j] = in ? (float)gr[i] : 0.f;
        } else {
          h[i][j] = in ? (float)xr[i][j] : mean;
          g[i][j] = in ? (float)gr[i][j] : 0.f;
        }
      }
    }
    if (row + step < a.n) fetch(row + step);
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        h[i][j] = (h[i][j] - mean) * rstd;
        db[i][j] += g[i][j];
        dw[i][j] = fmaf(g[i][j], h[i][j], dw[i][j]);
        g[i][j] *= wf[i][j];
        sg += g[i][j];
        sgh = fmaf(g[i][j], h[i][j], sgh);
      }
    const float mg = wave_sum(sg) * inv_d, mgh = wave_sum(sgh) * inv_d;
    T* dx = reinterpret_cast<T*>(a.dx) + row * a.d;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (lane + 64 * i) * VEC;
      if (c < a.d) {
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = rstd * (g[i][j] - mg - h[i][j] * mgh);
        store_vec<T, VEC>(dx + c, o);
      }
    }
  }
  float* part = a.partial + (int64_t)blockIdx.x * 2 * a.d;
  const bool alone = gridDim.x == 1;  // the sums are the gradients
#pragma unroll
  for (int i = 0; i < P; ++i) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < VEC; ++j) red[wave][lane * VEC + j] = which ? db[i][j] : dw[i][j];
      __syncthreads();
      for (int t = threadIdx.x; t < 64 * VEC; t += kBlock) {
        const int c = i * 64 * VEC + t;
        if (c < a.d) {
          const float s = (red[0][t] + red[1][t]) + (red[2][t] + red[3][t]);
          T* out = reinterpret_cast<T*>(which ? a.dbias : a.dweight);
          if (!alone)
            part[which * (int64_t)a.d + c] = s;
          else if (out != nullptr)
            out[c] = (T)s;
        }
      }
    }
  }
}

// dx of rows wider than the registers hold.
template <class T>
__global__ __launch_bounds__(kBlock) void norm_backward_wide_kernel(NormArgs a) {
  __shared__ float scratch[kBlock / kWave];
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.dy_stride;
    const T* w = reinterpret_cast<const T*>(a.weight);
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sg = 0.f, sgh = 0.f;
    for (int c = threadIdx.x; c < a.d; c += kBlock) {
      const float g = (float)dy[c] * (float)w[c];
      sg += g;
      sgh = fmaf(g, ((float)x[c] - mean) * rstd, sgh);
    }
    const float inv_d = 1.f / (float)a.d;
    const float mg = block_sum(sg, scratch) * inv_d;
    const float mgh = block_sum(sgh, scratch) * inv_d;
    T* dx = reinterpret_cast<T*>(a.dx) + row * a.d;
    for (int c = threadIdx.x; c < a.d; c += kBlock)
      dx[c] = (T)(rstd * ((float)dy[c] * (float)w[c] - mg - ((float)x[c] - mean) * rstd * mgh));
  }
}

// Partial column sums of wide rows: workgroup (x: 256 columns, y: part of the rows).
template <class T>
__global__ __launch_bounds__(kBlock) void norm_columns_kernel(NormArgs a) {
  const int c = blockIdx.x * kBlock + threadIdx.x;
  if (c >= a.d) return;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* dy = reinterpret_cast<const T*>(a.dy);
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.y; r < a.n; r += gridDim.y) {
    const float g = (float)dy[r * a.dy_stride + c];
    db += g;
    dw = fmaf(g, ((float)x[r * a.x_stride + c] - a.mean[r]) * a.rstd[r], dw);
  }
  float* part = a.partial + (int64_t)blockIdx.y * 2 * a.d;
  part[c] = dw;
  part[a.d + c] = db;
}

// Adds partial rows in a fixed order: 16 columns a workgroup, 64 threads a column, whose loads
// (16 of them for 1024 rows: 7.2 us for 2 x 768 columns, in two turns of 8 7.6) are under way
// together; then a tree in LDS.
template <class T>
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* partial, int parts, int64_t stride, int n, T* out,
                                                           T* out2, int n1) {
  __shared__ float red[64][17];
  const int col = threadIdx.x & 15, lane = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + col;
  float s[16];
#pragma unroll
  for (int u = 0; u < 16; ++u) s[u] = 0.f;
  if (c < n)
    for (int p = lane; p < parts; p += 1024)
#pragma unroll
      for (int u = 0; u < 16; ++u)
        if (p + 64 * u < parts) s[u] += partial[(p + 64 * u) * stride + c];
#pragma unroll
  for (int half = 8; half > 0; half >>= 1)
#pragma unroll
    for (int u = 0; u < half; ++u) s[u] += s[u + half];
  red[lane][col] = s[0];
#pragma unroll
  for (int half = 32; half > 0; half >>= 1) {
    __syncthreads();
    if (lane < half) red[lane][col] += red[lane + half][col];
  }
  if (lane == 0 && c < n) {
    T* to = c < n1 ? out + c : out2 + (c - n1);
    *to = (T)red[0][col];
  }
}

template <class T>
bool aligned_rows(const NormArgs& a, int vec, bool backward) {
  auto ok = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % (vec * sizeof(T)) == 0; };
  if (a.d % vec != 0 || a.x_stride % vec != 0 || !ok(a.x) || !ok(a.weight)) return false;
  if (backward) return a.dy_stride % vec == 0 && ok(a.dy) && ok(a.dx);
  return ok(a.bias) && ok(a.y);
}

constexpr int kRegWidth = 2048;  // columns a wave holds: 32 a lane

template <class T, int VEC, int P>
void launch_rows(const NormArgs& a, bool backward, hipStream_t s) {
  if (backward)
    hipLaunchKernelGGL((norm_backward_kernel<T, VEC, P>), dim3(a.parts), dim3(kBlock), 0, s, a);
  else
    hipLaunchKernelGGL((norm_forward_kernel<T, VEC, P>), dim3((unsigned)((a.n + 3) / 4)), dim3(kBlock), 0, s, a);
}

// The fewest columns a lane that hold the row: pieces of 4, or of 2, where every row starts on
// one, single elements otherwise.  (Pieces of 8 of 16-bit rows leave a quarter of the lanes'
// second piece empty at width 768, the registers with it.)
template <class T>
void launch_narrow(const NormArgs& a, bool backward, hipStream_t s) {
  const int lanes = (a.d + 63) / 64;
  if (aligned_rows<T>(a, 4, backward)) {
    if (lanes <= 4)
      launch_rows<T, 4, 1>(a, backward, s);
    else if (lanes <= 8)
      launch_rows<T, 4, 2>(a, backward, s);
    else if (lanes <= 12)
      launch_rows<T, 4, 3>(a, backward, s);
    else if (lanes <= 16)
      launch_rows<T, 4, 4>(a, backward, s);
    else if (lanes <= 24)
      launch_rows<T, 4, 6>(a, backward, s);
    else
      launch_rows<T, 4, 8>(a, backward, s);
  } else if (aligned_rows<T>(a, 2, backward)) {
    if (lanes <= 6)
      launch_rows<T, 2, 3>(a, backward, s);
    else if (lanes <= 16)
      launch_rows<T, 2, 8>(a, backward, s);
    else
      launch_rows<T, 2, 16>(a, backward, s);
  } else {
    if (lanes <= 6)
      launch_rows<T, 1, 6>(a, backward, s);
    else if (lanes <= 16)
      launch_rows<T, 1, 16>(a, backward, s);
    else
      launch_rows<T, 1, 32>(a, backward, s);
  }
}

template <class T>
void forward(const NormArgs& a, hipStream_t s) {
  if (a.d <= kRegWidth)
    launch_narrow<T>(a, false, s);
  else
    hipLaunchKernelGGL(norm_forward_wide_kernel<T>, dim3((unsigned)a.n), dim3(kBlock), 0, s, a);
}

template <class T>
void backward(const NormArgs& a, hipStream_t s) {
  if (a.d <= kRegWidth) {
    launch_narrow<T>(a, true, s);
  } else {
    hipLaunchKernelGGL(norm_backward_wide_kernel<T>, dim3((unsigned)std::min<int64_t>(a.n, 1 << 20)), dim3(kBlock), 0, s, a);
    hipLaunchKernelGGL(norm_columns_kernel<T>, dim3((a.d + kBlock - 1) / kBlock, a.parts), dim3(kBlock), 0, s, a);
  }
}

}  // namespace

int norm_backward_parts(int64_t n, int64_t d, int type, int cus) {
  (void)type;
  if (d > kRegWidth) return (int)std::min<int64_t>(n, 64);
  if (n <= 32) return 1;  // a launch for the sums would take longer than eight rows a wave
  // four workgroups a CU hide each other's latency; over many rows two do, and leave fewer
  // partial sums (50021 x 1000 in fp32: 122 us against 127 with four, 50021 x 768 in bf16 43 against 46;
  // of narrow rows, 120000 x 256 in fp16, four would take 41 for 44, and of 16384 x 768 in bf16,
  // which has four, two 23 for 25)
  return (int)std::min<int64_t>((n + 3) / 4, n > 128 * (int64_t)cus ? 2 * cus : 4 * cus);
}

hipError_t launch_column_sums(const float* partial, int parts, int64_t stride, int n1, int n2, int type, void* out, void* out2,
                              hipStream_t s) {
  const int n = n1 + n2;
  const dim3 grid((n + 15) / 16), block(1024);
  if (type == kF16)
    hipLaunchKernelGGL(column_sums_kernel<_Float16>, grid, block, 0, s, partial, parts, stride, n, (_Float16*)out, (_Float16*)out2, n1);
  else if (type == kBF16)
    hipLaunchKernelGGL(column_sums_kernel<__bf16>, grid, block, 0, s, partial, parts, stride, n, (__bf16*)out, (__bf16*)out2, n1);
  else
    hipLaunchKernelGGL(column_sums_kernel<float>, grid, block, 0, s, partial, parts, stride, n, (float*)out, (float*)out2, n1);
  return hipGetLastError();
}

hipError_t launch_norm_forward(const NormArgs& all, hipStream_t s) {
  // (a launch has fewer than 2^32 threads: rows in pieces)
  constexpr int64_t kRows = 1 << 23;
  const int64_t size = all.type == kF32 ? 4 : 2;
  for (int64_t r = 0; r < all.n; r += kRows) {
    NormArgs a = all;
    a.n = std::min(kRows, all.n - r);
    a.x = static_cast<const char*>(all.x) + r * all.x_stride * size;
    a.y = static_cast<char*>(all.y) + r * all.d * size;
    if (all.mean != nullptr) a.mean = all.mean + r, a.rstd = all.rstd + r;
    if (a.type == kF16)
      forward<_Float16>(a, s);
    else if (a.type == kBF16)
      forward<__bf16>(a, s);
    else
      forward<float>(a, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_norm_backward(const NormArgs& a, hipStream_t s) {
  if (a.type == kF16)
    backward<_Float16>(a, s);
  else if (a.type == kBF16)
    backward<__bf16>(a, s);
  else
    backward<float>(a, s);
  hipError_t e = hipGetLastError();
  if (a.parts == 1 && a.d <= kRegWidth) return e;
  // the partial rows hold dweight's columns, then dbias's: one launch adds both
  const int64_t stride = 2 * (int64_t)a.d;
  if (e == hipSuccess && a.dweight != nullptr && a.dbias != nullptr)
    return launch_column_sums(a.partial, a.parts, stride, a.d, a.d, a.type, a.dweight, a.dbias, s);
  if (e == hipSuccess && a.dweight != nullptr)
    e = launch_column_sums(a.partial, a.parts, stride, a.d, 0, a.type, a.dweight, nullptr, s);
  if (e == hipSuccess && a.dbias != nullptr)
    e = launch_column_sums(a.partial + a.d, a.parts, stride, a.d, 0, a.type, a.dbias, nullptr, s);
  return e;
}

}  // namespace cvs
