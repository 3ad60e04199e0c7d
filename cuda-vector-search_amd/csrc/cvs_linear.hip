// Matrix product with bias, activation and residual in its epilogue, and the
// products of its backward pass, for 16-bit operands with fp32 sums.
//
//   out[i, j] = act(sum_r M(i, r) N(j, r) + bias[j]) + residual[i, j]
//
// Either operand may be stored with its reduction contiguous ([rows, k]) or strided
// ([k, rows]): y = x W^T reads x and W so, dx = dz W takes W strided, dW = dz^T x
// both.  Stages of 64 reduction steps come into LDS as lines of 128 bytes, straight
// from memory (buffer loads into LDS; a lane past the operand's edge gets an
// offset past the buffer's end, which reads as zero); strided operands are turned
// on the way out of LDS by transposing reads.
#include <algorithm>

#include "cvs_encoder.h"
#include "cvs_mfma.h"

namespace cvs {

namespace {

constexpr int kDepth = 64;                    // reduction steps of a stage
constexpr uint32_t kOutside = 0x80000000u;    // a byte offset past every buffer

typedef int i32x4s __attribute__((ext_vector_type(4)));

// 16 bytes a lane from base + voff into LDS at lds + 16 * lane; zeros where voff >= kOutside.
__device__ __forceinline__ void load_lds(uint32_t voff, const unsigned char* base, uint32_t lds) {
  const uint64_t b = (uint64_t)(uintptr_t)base;
  const i32x4s rsrc = {__builtin_amdgcn_readfirstlane((int)(uint32_t)b),
                       __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32) & 0xffff), (int)kOutside, 0x00020000};
  const uint32_t m = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(m), "v"(voff), "s"(rsrc)
      : "memory");
}

__device__ __forceinline__ float activate(float z, int act) {
  if (act == kActGelu) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if (act == kActRelu) return z > 0.f ? z : (z != z ? z : 0.f);
  if (act == kActTanh) return tanhf(z);
  return z;
}

__device__ __forceinline__ float slope(float z, int act) {
  if (act == kActGelu) return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
  if (act == kActRelu) return z > 0.f ? 1.f : 0.f;
  if (act == kActTanh) {
    const float t = tanhf(z);
    return 1.f - t * t;
  }
  return 1.f;
}

template <class T>
__device__ __forceinline__ void load8(const T* p, float* f) {
  const auto v = *reinterpret_cast<const typename Frag<T>::V*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)v[j];
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float* f) {
  typename Frag<T>::V v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (T)f[j];
  *reinterpret_cast<typename Frag<T>::V*>(p) = v;
}

// The epilogue of 8 neighbouring sums of row i, columns j .. j + 7.
template <class T>
__device__ __forceinline__ void finish8(const GemmArgs& a, int i, int j, float* z) {
  if (a.bias != nullptr) {
    float b[8];
    load8((const T*)a.bias + j, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += b[e];
  }
  const int64_t at = (int64_t)i * a.n + j;
  if (a.pre != nullptr) store8((T*)a.pre + at, z);
  if (a.act != kActNone) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = activate(z[e], a.act);
  }
  if (a.residual != nullptr) {
    float r[8];
    load8((const T*)a.residual + (int64_t)i * a.ld_res + j, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += r[e];
  }
  store8((T*)a.out + at, z);
}

template <class T, int TM, int TN, int RING, bool MS, bool NS>
__global__ __launch_bounds__(kBlock, 2) void gemm_kernel(GemmArgs a) {
  constexpr int LM = TM / 32, LN = TN / 32;           // 1 KiB loads a wave and stage
  constexpr int BM = TM / 64, BN = TN / 64;           // 32 x 32 blocks a wave: 2 x 2 waves
  constexpr int MBYTES = TM * 128, STAGE = (TM + TN) * 128;
  typedef typename Frag<T>::V V;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[RING * STAGE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int l32 = lane & 31, g = lane >> 5;
  const int p16 = lane >> 4, s16 = lane & 15;

  // Tiles in an order that gives each XCD (consecutive workgroups go round the 8 of
  // them) neighbouring tiles, columns first: they share rows of M in its L2.
  const int tiles_n = (a.n + TN - 1) / TN, tiles_m = (a.m + TM - 1) / TM;
  const int tiles = tiles_n * tiles_m;
  const int per = (tiles + 7) / 8;
  const int local = blockIdx.x >> 3;
  const int tile = (blockIdx.x & 7) * per + local;
  if (local >= per || tile >= tiles) return;
  const int m0 = tile / tiles_n * TM, n0 = tile % tiles_n * TN;

  const int stages = (a.k + kDepth - 1) / kDepth;
  const int s_begin = (int)((int64_t)stages * blockIdx.y / a.splits);
  const int s_end = (int)((int64_t)stages * (blockIdx.y + 1) / a.splits);

  // This lane's place in each 1 KiB load: line and 16-byte piece of the tile.
  uint32_t vm[LM], vn[LN];
  int km[LM], kn[LN];  // reduction step of the load within a stage
  auto place = [&](int j, bool strided, int64_t ld, int first, int rows, uint32_t* voff, int* step) {
    const int line = (wave + 4 * j) * 8 + (lane >> 3);
    const int piece = (lane & 7) ^ piece_swizzle(line);
    if (strided) {
      const int col = line / 64 * 64 + piece * 8;
      *voff = (uint32_t)((line & 63) * ld * 2) + (uint32_t)(col * 2);
      if (first + col >= rows) *voff = kOutside;
      *step = line & 63;
    } else {
      *voff = (uint32_t)(line * ld * 2) + (uint32_t)(piece * 16);
      if (first + line >= rows) *voff = kOutside;
      *step = piece * 8;
    }
  };
#pragma unroll
  for (int j = 0; j < LM; ++j) place(j, MS, a.ldm, m0, a.m, &vm[j], &km[j]);
#pragma unroll
  for (int j = 0; j < LN; ++j) place(j, NS, a.ldn, n0, a.n, &vn[j], &kn[j]);
  const unsigned char* mbase = (const unsigned char*)a.M + 2 * (MS ? (int64_t)m0 : m0 * a.ldm);
  const unsigned char* nbase = (const unsigned char*)a.N + 2 * (NS ? (int64_t)n0 : n0 * a.ldn);
  const int64_t mstep = 2 * (MS ? kDepth * a.ldm : (int64_t)kDepth), nstep = 2 * (NS ? kDepth * a.ldn : (int64_t)kDepth);
  mbase += s_begin * mstep;
  nbase += s_begin * nstep;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)smem;

  int load_s = s_begin, load_buf = 0;
  auto load_stage = [&]() {
    const uint32_t at = lds0 + (uint32_t)(load_buf * STAGE + wave * 1024);
    const int left = a.k - load_s * kDepth;  // reduction steps from this stage on
#pragma unroll
    for (int j = 0; j < LM; ++j) load_lds(km[j] < left ? vm[j] : kOutside, mbase, at + j * 4096);
#pragma unroll
    for (int j = 0; j < LN; ++j) load_lds(kn[j] < left ? vn[j] : kOutside, nbase, at + MBYTES + j * 4096);
    mbase += mstep;
    nbase += nstep;
    ++load_s;
    load_buf = load_buf + 1 == RING ? 0 : load_buf + 1;
  };

  // Operand fragments of depth step ks (16 of the stage's 64), rows r0 .. r0 + 31 of the tile.
  auto frag = [&](const unsigned char* t, bool strided, int r0, int ks, bool reorder) -> V {
    if (strided) {
      const int c = reorder ? ((s16 & 1) << 1) | ((s16 >> 1) & 1) : s16 & 3;
      const int col = r0 + 16 * (p16 & 1) + 4 * c;
      const int line = 16 * ks + 8 * (p16 >> 1) + (s16 >> 2);
      const unsigned char* panel = t + (col >> 6) * 8192 + (col & 4) * 2;
      const int piece = (col & 63) >> 3;
      const s16x4 lo = read_tr(panel + line * 128 + ((piece ^ piece_swizzle(line)) << 4));
      const s16x4 hi = read_tr(panel + (line + 4) * 128 + ((piece ^ piece_swizzle(line + 4)) << 4));
      return join_tr<T>(lo, hi);
    }
    const int line = r0 + (reorder ? tile_row(l32) : l32);
    return *reinterpret_cast<const V*>(t + line * 128 + (((2 * ks + g) ^ piece_swizzle(line)) << 4));
  };

  f32x16 acc[BM][BN];
#pragma unroll
  for (int i = 0; i < BM; ++i)
#pragma unroll
    for (int j = 0; j < BN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

#pragma unroll
  for (int s = 0; s < RING - 1; ++s)
    if (s_begin + s < s_end) load_stage();

  int buf = 0;
  for (int s = s_begin; s < s_end; ++s) {
    // this stage's loads are in; those of the next RING - 2 may still be under way
    if (RING > 2 && s + 1 < s_end)
      wait_vmcnt_lgkm0<(RING - 2) * (LM + LN)>();
    else
      wait_vmcnt_lgkm0<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (load_s < s_end) load_stage();  // into the buffer that every wave has left
    const unsigned char* tm = smem + buf * STAGE;
    const unsigned char* tn = tm + MBYTES;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      V fm[BM], fn[BN];
#pragma unroll
      for (int i = 0; i < BM; ++i) fm[i] = frag(tm, MS, (wm * BM + i) * 32, ks, false);
#pragma unroll
      for (int j = 0; j < BN; ++j) fn[j] = frag(tn, NS, (wn * BN + j) * 32, ks, true);
#pragma unroll
      for (int i = 0; i < BM; ++i)
#pragma unroll
        for (int j = 0; j < BN; ++j) acc[i][j] = Frag<T>::mfma(fn[j], fm[i], acc[i][j]);
    }
    buf = buf + 1 == RING ? 0 : buf + 1;
  }

  // Lane: row i of the output, 8 neighbouring columns a half of its accumulator.
#pragma unroll
  for (int i = 0; i < BM; ++i) {
    const int row = m0 + (wm * BM + i) * 32 + l32;
#pragma unroll
    for (int j = 0; j < BN; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = n0 + (wn * BN + j) * 32 + 16 * h + 8 * g;
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = acc[i][j][8 * h + e];
        if (row < a.m && col < a.n) {
          if (a.splits > 1) {
            float* p = a.partial + ((int64_t)blockIdx.y * a.m + row) * a.n + col;
            *reinterpret_cast<f32x4*>(p) = f32x4{z[0], z[1], z[2], z[3]};
            *reinterpret_cast<f32x4*>(p + 4) = f32x4{z[4], z[5], z[6], z[7]};
          } else {
            finish8<T>(a, row, col, z);
          }
        }
      }
  }
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
  finish8<T>(a, (int)i, j, z);
}

template <class T, int TM, int TN, int RING>
hipError_t launch_tiles(const GemmArgs& a, hipStream_t s) {
  const int tiles = ((a.m + TM - 1) / TM) * ((a.n + TN - 1) / TN);
  const dim3 grid((tiles + 7) / 8 * 8, a.splits), block(kBlock);
  if (a.m_strided && a.n_strided)
    hipLaunchKernelGGL((gemm_kernel<T, TM, TN, RING, true, true>), grid, block, 0, s, a);
  else if (a.n_strided)
    hipLaunchKernelGGL((gemm_kernel<T, TM, TN, RING, false, true>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((gemm_kernel<T, TM, TN, RING, false, false>), grid, block, 0, s, a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.splits > 1) {
    const int64_t threads = (int64_t)a.m * (a.n / 8);
    hipLaunchKernelGGL((gemm_join_kernel<T>), dim3((unsigned)((threads + kBlock - 1) / kBlock)), block, 0, s, a);
    e = hipGetLastError();
  }
  return e;
}

template <class T>
hipError_t launch_typed(const GemmArgs& a, const GemmPlan& p, hipStream_t s) {
  if (p.tm == 128) return launch_tiles<T, 128, 128, 2>(a, s);
  return launch_tiles<T, 64, 64, 3>(a, s);
}

// dz = dy act'(pre), 8 columns a thread, rows blockIdx.y, + gridDim.y, ...; column sums a part.
template <class T>
__global__ __launch_bounds__(kBlock) void act_grad_kernel(ActGradArgs a) {
  const int c = (blockIdx.x * kBlock + threadIdx.x) * 8;
  if (c >= a.n) return;
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  for (int64_t r = blockIdx.y; r < a.m; r += gridDim.y) {
    float g[8];
    load8((const T*)a.dy + r * a.dy_stride + c, g);
    if (a.act != kActNone) {
      float z[8];
      load8((const T*)a.pre + r * a.n + c, z);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] *= slope(z[e], a.act);
      store8((T*)a.dz + r * a.n + c, g);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += g[e];
  }
  if (a.partial != nullptr) {
    float* p = a.partial + (int64_t)blockIdx.y * a.n + c;
    *reinterpret_cast<f32x4*>(p) = f32x4{sum[0], sum[1], sum[2], sum[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{sum[4], sum[5], sum[6], sum[7]};
  }
}

}  // namespace

GemmPlan plan_gemm(int64_t m, int64_t n, int64_t k, bool m_strided, bool n_strided, int cus) {
  (void)m_strided, (void)n_strided;
  GemmPlan p;
  auto tiles = [&](int64_t t) { return ((m + t - 1) / t) * ((n + t - 1) / t); };
  p.tm = p.tn = tiles(128) >= cus ? 128 : 64;
  // a reduction long enough is split where the tiles leave CUs idle
  const int64_t t = tiles(p.tm), stages = (k + kDepth - 1) / kDepth;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(cus / std::max<int64_t>(t, 1), stages / 8));
  p.ws_bytes = p.splits > 1 ? (int64_t)p.splits * m * n * 4 : 0;
  return p;
}

hipError_t launch_gemm(const GemmArgs& a, const GemmPlan& p, hipStream_t s) {
  return a.type == kF16 ? launch_typed<_Float16>(a, p, s) : launch_typed<__bf16>(a, p, s);
}

int act_grad_parts(int64_t m, int64_t n, int cus) {
  const int64_t blocks = (n / 8 + kBlock - 1) / kBlock;
  return (int)std::max<int64_t>(1, std::min<int64_t>(m, 8 * cus / blocks));
}

hipError_t launch_act_grad(const ActGradArgs& a, hipStream_t s) {
  const dim3 grid((a.n / 8 + kBlock - 1) / kBlock, a.parts), block(kBlock);
  if (a.type == kF16)
    hipLaunchKernelGGL(act_grad_kernel<_Float16>, grid, block, 0, s, a);
  else
    hipLaunchKernelGGL(act_grad_kernel<__bf16>, grid, block, 0, s, a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.dbias != nullptr) e = launch_column_sums(a.partial, a.parts, a.n, a.n, a.type, a.dbias, s);
  return e;
}

}  // namespace cvs
