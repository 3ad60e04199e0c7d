// Attention, forward: out_i = sum_j softmax_j(scale q_i . k_j + bias(j - i)) v_j over the
// keys that row i sees, in one pass over the keys with a running maximum and sum.
//
// A workgroup has 128 query rows of a head, a wave 32 of them, and walks the keys
// in tiles of 64.  The scores are computed transposed (keys x queries), so that a
// lane's elements all belong to one query: the softmax's maximum and sum are sums
// within a lane and one exchange of the lane halves, and the probabilities, packed to
// 16 bits, are the B operand of out^T = V^T P^T as they stand.  V^T comes from LDS
// by transposing reads.  Probabilities are rounded to the inputs' type (as the matrix
// cores take them); scores, maxima, sums and the output's sum are fp32.
//
// A row that sees no key gets zeros, and -inf as its log sum.
#include <algorithm>

#include "cvs_attn_tile.h"

namespace cvs {

namespace {

constexpr int kKeys = 64;  // keys of a tile

template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(kBlock, 2) void attn_forward_kernel(AttnArgs a) {
  typedef typename Frag<T>::V V;
  constexpr int KS = DP / 16, DB = DP / 32, TILE = kKeys * DP * 2;
  __shared__ __attribute__((aligned(128))) unsigned char sk[2][TILE], sv[2][TILE];
  extern __shared__ float tab[];

  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = a.batch * a.heads;
  const int bh = blockIdx.x % heads, block = blockIdx.x / heads;
  const int b = bh / a.heads, h = bh % a.heads, hk = h / (a.heads / a.k_heads);
  const int nk = key_count(a, b), nq = query_count(a, b), off = query_offset(a, b);
  const int r0 = block * kAttnRows + wave * 32;
  const int i = r0 + l32;
  const unsigned char* qrow = (const unsigned char*)a.q + 2 * (b * a.qs[0] + i * a.qs[1] + h * a.qs[2]);
  const unsigned char* kbase = (const unsigned char*)a.k + 2 * (b * a.ks[0] + hk * a.ks[2]);
  const unsigned char* vbase = (const unsigned char*)a.v + 2 * (b * a.vs[0] + hk * a.vs[2]);

  V qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = global_frag<T>(qrow, s, a.d, i < nq);
  if (BIAS) load_diag(tab, a, h);

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = zero16();
  float m = -__builtin_inff(), sum = 0.f;
  const float c = a.scale * kLog2e;

  // this workgroup's keys: a part of those that some row of it sees
  const int last_row = min(block * kAttnRows + kAttnRows, nq) - 1;
  int end = last_row < block * kAttnRows ? 0 : nk;
  if (a.causal) end = min(end, max(last_row + off + 1, 0));
  const int tiles = (end + kKeys - 1) / kKeys;
  const int t0 = (int)((int64_t)tiles * blockIdx.y / a.splits), t1 = (int)((int64_t)tiles * (blockIdx.y + 1) / a.splits);

  TileLoad<DP, kKeys> lk, lv;
  if (t0 < t1) {
    lk.load(kbase, 2 * a.ks[1], t0 * kKeys, nk, a.d);
    lv.load(vbase, 2 * a.vs[1], t0 * kKeys, nk, a.d);
  }
  for (int t = t0; t < t1; ++t) {
    const int buf = t & 1;
    lk.store(sk[buf]);
    lv.store(sv[buf]);
    __syncthreads();
    if (t + 1 < t1) {
      lk.load(kbase, 2 * a.ks[1], (t + 1) * kKeys, nk, a.d);
      lv.load(vbase, 2 * a.vs[1], (t + 1) * kKeys, nk, a.d);
    }
    const int j0 = t * kKeys;
    f32x16 x[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      x[kb] = zero16();
#pragma unroll
      for (int s = 0; s < KS; ++s) x[kb] = Frag<T>::mfma(row_frag<T, DP>(sk[buf], kb * 32, s), qf[s], x[kb]);
    }
    const bool whole = j0 + kKeys <= nk && (!a.causal || j0 + kKeys - 1 <= r0 + off);
    float top = m;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = j0 + kb * 32 + elem_row(e, g);
        float v = x[kb][e] * c;
        if (BIAS) v += tab[min(max(j - i - off, -a.max_distance), a.max_distance) + a.max_distance];
        if (!whole && (j >= nk || (a.causal && j > i + off))) v = -__builtin_inff();
        x[kb][e] = v;
        top = fmaxf(top, v);
      }
    top = fmaxf(top, swap_halves(top));
    const float base = top == -__builtin_inff() ? 0.f : top;
    const float fade = __builtin_amdgcn_exp2f(m - base);
    m = top;
    float part = 0.f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[kb][e] = __builtin_amdgcn_exp2f(x[kb][e] - base);
        part += x[kb][e];
      }
    sum = sum * fade + part;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[d][e] *= fade;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const V p = pack8<T>(x[kb], s);
#pragma unroll
        for (int d = 0; d < DB; ++d)
          acc[d] = Frag<T>::mfma(col_frag<T, DP>(sv[buf], kb * 32 + 16 * s, d * 32), p, acc[d]);
      }
  }
  sum += swap_halves(sum);
  if (i >= a.lq) return;
  if (i >= nq) sum = 0.f, m = -__builtin_inff();
  const int64_t at = (int64_t)bh * a.lq + i;  // [batch, heads, lq]
  if (a.splits > 1) {
    const int64_t rows = (int64_t)heads * a.lq;
    if (g == 0) {
      a.part_ml[2 * (blockIdx.y * rows + at)] = m;
      a.part_ml[2 * (blockIdx.y * rows + at) + 1] = sum;
    }
    float* o = a.part_out + (blockIdx.y * rows + at) * a.d;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = d * 32 + 16 * (q >> 1) + 8 * g + 4 * (q & 1);
        if (col < a.d)
          *reinterpret_cast<f32x4*>(o + col) = f32x4{acc[d][4 * q], acc[d][4 * q + 1], acc[d][4 * q + 2], acc[d][4 * q + 3]};
      }
    return;
  }
  if (a.lse != nullptr && g == 0) a.lse[at] = sum == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(sum)) * kLn2;
  store_head_row<T, DP>((T*)a.out + ((int64_t)(b * (int64_t)a.lq + i) * a.heads + h) * a.d, acc,
                        sum == 0.f ? 0.f : 1.f / sum, a.d);
}

// Joins the parts of the keys: one wave a query row.
template <class T>
__global__ __launch_bounds__(kBlock) void attn_join_kernel(AttnArgs a) {
  const int64_t rows = (int64_t)a.batch * a.heads * a.lq;
  const int64_t at = (int64_t)blockIdx.x * (kBlock / kWave) + (threadIdx.x >> 6);
  if (at >= rows) return;
  const int lane = threadIdx.x & 63;
  float m = -__builtin_inff();
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[2 * (s * rows + at)]);
  const float base = m == -__builtin_inff() ? 0.f : m;
  float sum = 0.f, o0 = 0.f, o1 = 0.f;
  const int c = 2 * lane;
  for (int s = 0; s < a.splits; ++s) {
    const float* ml = a.part_ml + 2 * (s * rows + at);
    const float f = __builtin_amdgcn_exp2f(ml[0] - base);
    sum = fmaf(f, ml[1], sum);
    if (c < a.d) {
      const float* o = a.part_out + (s * rows + at) * a.d + c;
      o0 = fmaf(f, o[0], o0);
      o1 = fmaf(f, o[1], o1);
    }
  }
  const int i = (int)(at % a.lq);
  const int64_t bh = at / a.lq, b = bh / a.heads, h = bh % a.heads;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (c < a.d) {
    T* out = (T*)a.out + ((b * a.lq + i) * a.heads + h) * a.d + c;
    out[0] = (T)(o0 * inv);
    out[1] = (T)(o1 * inv);
  }
  if (a.lse != nullptr && lane == 0) a.lse[at] = sum == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <class T>
__global__ __launch_bounds__(kBlock) void attn_diag_kernel(AttnArgs a) {
  const int n = 2 * a.max_distance + 1;
  const int h = blockIdx.x;
  for (int t = threadIdx.x; t < n; t += kBlock) {
    const int rel = t - a.max_distance;
    const int dist = a.causal ? max(-rel, 0) : abs(rel);
    int u = 0;
    while (u + 1 < a.one_way && a.edges[u + 1] <= dist) ++u;
    const int bucket = !a.causal && rel > 0 ? a.one_way + u : u;
    a.diag[(int64_t)h * n + t] = (float)((const T*)a.table)[(int64_t)bucket * a.heads + h] * kLog2e;
  }
}

template <class T, int DP>
void launch_width(const AttnArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.lq + kAttnRows - 1) / kAttnRows * (int64_t)a.batch * a.heads), a.splits), block(kBlock);
  const size_t tab = a.table != nullptr ? (2 * a.max_distance + 1) * sizeof(float) : 0;
  if (a.table != nullptr)
    hipLaunchKernelGGL((attn_forward_kernel<T, DP, true>), grid, block, tab, s, a);
  else
    hipLaunchKernelGGL((attn_forward_kernel<T, DP, false>), grid, block, 0, s, a);
}

template <class T>
hipError_t forward(const AttnArgs& a, hipStream_t s) {
  if (a.d <= 32)
    launch_width<T, 32>(a, s);
  else if (a.d <= 64)
    launch_width<T, 64>(a, s);
  else
    launch_width<T, 128>(a, s);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.splits > 1) {
    const int64_t rows = (int64_t)a.batch * a.heads * a.lq;
    hipLaunchKernelGGL(attn_join_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(kBlock), 0, s, a);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace

int attn_splits(const AttnArgs& a, int cus) {
  const int64_t wgs = (a.lq + kAttnRows - 1) / kAttnRows * (int64_t)a.batch * a.heads;
  const int64_t tiles = (a.lk + kKeys - 1) / kKeys;
  return (int)std::max<int64_t>(1, std::min<int64_t>({2 * cus / std::max<int64_t>(wgs, 1), tiles / 4, (int64_t)64}));
}

hipError_t launch_attn_diag(const AttnArgs& a, hipStream_t s) {
  if (a.type == kF16)
    hipLaunchKernelGGL(attn_diag_kernel<_Float16>, dim3(a.heads), dim3(kBlock), 0, s, a);
  else
    hipLaunchKernelGGL(attn_diag_kernel<__bf16>, dim3(a.heads), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_attn_forward(const AttnArgs& a, hipStream_t s) {
  return a.type == kF16 ? forward<_Float16>(a, s) : forward<__bf16>(a, s);
}

}  // namespace cvs
