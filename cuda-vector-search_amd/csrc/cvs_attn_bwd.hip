// Attention, backward: the probabilities are computed again from q, k and the rows' log sums,
//   p_ij = exp(scale q_i . k_j + bias(j - i) - lse_i),   dv_j = sum_i p_ij dout_i,
//   ds_ij = p_ij (dout_i . v_j - delta_i), delta_i = dout_i . out_i,
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,
//   dtable[bucket, h] = sum of ds_ij over the pairs whose position falls in the bucket.
//
// Two kernels, each with sums that no other workgroup adds to: one walks the queries
// for 128 keys (dk, dv; the query heads that share a key head one after the other), one
// the keys for 128 queries (dq, dtable).  That computes the scores and dout . v twice
// (seven products instead of five), and needs neither atomics, whose order would
// change results, nor a pass that adds up partial dq.  As in the forward kernel, a block
// of scores is oriented so that, packed to 16 bits, it is an operand of the next
// product in registers.  Probabilities and ds are rounded to the inputs' type there;
// everything else is fp32.
//
// dtable: a lane group (half a wave) adds its ds to its own sums by relative
// position in LDS, where positions beyond the bias's range are registers instead;
// one position has one lane of the group at a time, so the order of the adds is fixed.
#include <algorithm>

#include "cvs_attn_tile.h"

namespace cvs {

namespace {

constexpr int kTile = 32;  // rows of a streamed tile
constexpr float kNever = __builtin_inff();

// delta: 8 lanes a row.
template <class T>
__global__ __launch_bounds__(kBlock) void attn_delta_kernel(AttnArgs a) {
  const int64_t row = (int64_t)blockIdx.x * (kBlock / 8) + threadIdx.x / 8;  // of [batch, lq, heads]
  if (row >= (int64_t)a.batch * a.lq * a.heads) return;
  const int h = (int)(row % a.heads);
  const int64_t bi = row / a.heads;
  const int i = (int)(bi % a.lq);
  const int64_t b = bi / a.lq;
  const T* o = (const T*)a.out + row * a.d;
  const T* g = (const T*)a.dout + b * a.dos[0] + i * a.dos[1] + h * a.dos[2];
  float s = 0.f;
  for (int c = threadIdx.x % 8 * 8; c < a.d; c += 64) {
    const auto x = *reinterpret_cast<const typename Frag<T>::V*>(o + c);
    const auto y = *reinterpret_cast<const typename Frag<T>::V*>(g + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf((float)x[j], (float)y[j], s);
  }
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) s += __shfl_xor(s, off);
  if (threadIdx.x % 8 == 0) a.delta[(b * a.heads + h) * a.lq + i] = s;
}

// dk and dv of 128 keys: wave w has keys 32 w .. of them as columns.
template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(kBlock, DP > 64 ? 1 : 2) void attn_backward_kv_kernel(AttnArgs a) {
  typedef typename Frag<T>::V V;
  constexpr int KS = DP / 16, DB = DP / 32, TILE = kTile * DP * 2;
  __shared__ __attribute__((aligned(128))) unsigned char sq[2][TILE], sg[2][TILE];
  __shared__ __attribute__((aligned(16))) float slse[2][kTile], sdelta[2][kTile];
  extern __shared__ float tab[];

  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kheads = a.batch * a.k_heads, group = a.heads / a.k_heads;
  const int bk = blockIdx.x % kheads, block = blockIdx.x / kheads;
  const int b = bk / a.k_heads, hk = bk % a.k_heads;
  const int nk = key_count(a, b), nq = query_count(a, b), off = query_offset(a, b);
  const int j0 = block * kAttnRows + wave * 32;
  const int j = j0 + l32;
  const unsigned char* krow = (const unsigned char*)a.k + 2 * (b * a.ks[0] + j * a.ks[1] + hk * a.ks[2]);
  const unsigned char* vrow = (const unsigned char*)a.v + 2 * (b * a.vs[0] + j * a.vs[1] + hk * a.vs[2]);
  V kf[KS], vf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    kf[s] = global_frag<T>(krow, s, a.d, j < nk);
    vf[s] = global_frag<T>(vrow, s, a.d, j < nk);
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dk[d] = dv[d] = zero16();
  const float c = a.scale * kLog2e;

  // queries that see a key of this workgroup
  int first = 0;
  if (a.causal) first = max(block * kAttnRows - off, 0);
  const int t0 = first / kTile, t1 = block * kAttnRows < nk ? (nq + kTile - 1) / kTile : 0;

  for (int hh = 0; hh < group; ++hh) {
    const int h = hk * group + hh;
    const unsigned char* qbase = (const unsigned char*)a.q + 2 * (b * a.qs[0] + h * a.qs[2]);
    const unsigned char* gbase = (const unsigned char*)a.dout + 2 * (b * a.dos[0] + h * a.dos[2]);
    const float* lse = a.lse + ((int64_t)b * a.heads + h) * a.lq;
    const float* delta = a.delta + ((int64_t)b * a.heads + h) * a.lq;
    __syncthreads();  // the last head's tiles and bias have been read
    if (BIAS) load_diag(tab, a, h);
    TileLoad<DP, kTile> lq, lg;
    float lrow = 0.f;  // lanes 0 .. 31: log2 sums, 32 .. 63: deltas of the rows
    auto load_rows = [&](int t) {
      const int i = t * kTile + (threadIdx.x & 31);
      if (threadIdx.x < 32) {
        lrow = i < nq ? lse[i] * kLog2e : kNever;
        if (lrow == -__builtin_inff()) lrow = kNever;  // a row that sees nothing
      } else if (threadIdx.x < 64) {
        lrow = i < nq ? delta[i] : 0.f;
      }
    };
    if (t0 < t1) {
      lq.load(qbase, 2 * a.qs[1], t0 * kTile, nq, a.d);
      lg.load(gbase, 2 * a.dos[1], t0 * kTile, nq, a.d);
      load_rows(t0);
    }
    for (int t = t0; t < t1; ++t) {
      const int buf = t & 1;
      lq.store(sq[buf]);
      lg.store(sg[buf]);
      if (threadIdx.x < 32)
        slse[buf][threadIdx.x] = lrow;
      else if (threadIdx.x < 64)
        sdelta[buf][threadIdx.x - 32] = lrow;
      __syncthreads();
      if (t + 1 < t1) {
        lq.load(qbase, 2 * a.qs[1], (t + 1) * kTile, nq, a.d);
        lg.load(gbase, 2 * a.dos[1], (t + 1) * kTile, nq, a.d);
        load_rows(t + 1);
      }
      const int i0 = t * kTile;
      f32x16 p = zero16(), ds = zero16();
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        p = Frag<T>::mfma(row_frag<T, DP>(sq[buf], 0, s), kf[s], p);
        ds = Frag<T>::mfma(row_frag<T, DP>(sg[buf], 0, s), vf[s], ds);
      }
      const bool whole = !a.causal || j0 + 31 <= i0 + off;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int r = elem_row(e, g), i = i0 + r;
        float x = p[e] * c;
        if (BIAS) x += tab[min(max(j - i - off, -a.max_distance), a.max_distance) + a.max_distance];
        float y = __builtin_amdgcn_exp2f(x - slse[buf][r]);
        if (!whole && j > i + off) y = 0.f;
        p[e] = y;
        ds[e] = y * (ds[e] - sdelta[buf][r]);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const V pf = pack8<T>(p, s), df = pack8<T>(ds, s);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          dv[d] = Frag<T>::mfma(col_frag<T, DP>(sg[buf], 16 * s, d * 32), pf, dv[d]);
          dk[d] = Frag<T>::mfma(col_frag<T, DP>(sq[buf], 16 * s, d * 32), df, dk[d]);
        }
      }
    }
  }
  if (j >= a.lk) return;
  const bool in = j < nk;
  if (!in) {
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[d] = dv[d] = zero16();
  }
  const int64_t at = (((int64_t)b * a.lk + j) * a.k_heads + hk) * a.d;
  store_head_row<T, DP>((T*)a.dk + at, dk, a.scale, a.d);
  store_head_row<T, DP>((T*)a.dv + at, dv, 1.f, a.d);
}

// dq of 128 queries (wave w: 32 of them as columns) and their sums for dtable.
template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(kBlock, DP > 64 ? 1 : 2) void attn_backward_q_kernel(AttnArgs a) {
  typedef typename Frag<T>::V V;
  constexpr int KS = DP / 16, DB = DP / 32, TILE = kTile * DP * 2;
  __shared__ __attribute__((aligned(128))) unsigned char sk[2][TILE], sv[2][TILE];
  extern __shared__ float tab[];  // bias by position, then 8 lane groups' sums by position

  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = a.batch * a.heads;
  const int bh = blockIdx.x % heads, block = blockIdx.x / heads;
  const int b = bh / a.heads, h = bh % a.heads, hk = h / (a.heads / a.k_heads);
  const int nk = key_count(a, b), nq = query_count(a, b), off = query_offset(a, b);
  const int r0 = block * kAttnRows + wave * 32;
  const int i = r0 + l32;
  const unsigned char* qrow = (const unsigned char*)a.q + 2 * (b * a.qs[0] + i * a.qs[1] + h * a.qs[2]);
  const unsigned char* grow = (const unsigned char*)a.dout + 2 * (b * a.dos[0] + i * a.dos[1] + h * a.dos[2]);
  const unsigned char* kbase = (const unsigned char*)a.k + 2 * (b * a.ks[0] + hk * a.ks[2]);
  const unsigned char* vbase = (const unsigned char*)a.v + 2 * (b * a.vs[0] + hk * a.vs[2]);
  V qf[KS], gf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    qf[s] = global_frag<T>(qrow, s, a.d, i < nq);
    gf[s] = global_frag<T>(grow, s, a.d, i < nq);
  }
  float lse = kNever, delta = 0.f;
  if (i < nq) {
    const int64_t at = (int64_t)bh * a.lq + i;
    lse = a.lse[at] * kLog2e;
    if (lse == -__builtin_inff()) lse = kNever;
    delta = a.delta[at];
  }
  // sums by position j - i - off = -reach .. reach; a tile with a position of the
  // bias's range reaches at most 62 beyond it
  const int reach = a.max_distance + 64, places = 2 * reach + 1;
  float* sums = tab + 2 * a.max_distance + 1;
  if (BIAS) {
    load_diag(tab, a, h);
    for (int t = threadIdx.x; t < 8 * places; t += kBlock) sums[t] = 0.f;
  }
  float* mine = sums + (wave * 2 + g) * places + reach;
  float before = 0.f, after = 0.f;  // positions all <= -max_distance, all >= max_distance

  f32x16 dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dq[d] = zero16();
  const float c = a.scale * kLog2e;
  const int last_row = min(block * kAttnRows + kAttnRows, nq) - 1;
  int end = last_row < block * kAttnRows ? 0 : nk;
  if (a.causal) end = min(end, max(last_row + off + 1, 0));
  const int tiles = (end + kTile - 1) / kTile;

  TileLoad<DP, kTile> lk, lv;
  if (tiles > 0) {
    lk.load(kbase, 2 * a.ks[1], 0, nk, a.d);
    lv.load(vbase, 2 * a.vs[1], 0, nk, a.d);
  }
  for (int t = 0; t < tiles; ++t) {
    const int buf = t & 1;
    lk.store(sk[buf]);
    lv.store(sv[buf]);
    __syncthreads();
    if (t + 1 < tiles) {
      lk.load(kbase, 2 * a.ks[1], (t + 1) * kTile, nk, a.d);
      lv.load(vbase, 2 * a.vs[1], (t + 1) * kTile, nk, a.d);
    }
    const int j0 = t * kTile;
    f32x16 p = zero16(), ds = zero16();
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      p = Frag<T>::mfma(row_frag<T, DP>(sk[buf], 0, s), qf[s], p);
      ds = Frag<T>::mfma(row_frag<T, DP>(sv[buf], 0, s), gf[s], ds);
    }
    const bool whole = j0 + kTile <= nk && (!a.causal || j0 + kTile - 1 <= r0 + off);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int j = j0 + elem_row(e, g);
      float x = p[e] * c;
      if (BIAS) x += tab[min(max(j - i - off, -a.max_distance), a.max_distance) + a.max_distance];
      float y = __builtin_amdgcn_exp2f(x - lse);
      if (!whole && (j >= nk || (a.causal && j > i + off))) y = 0.f;
      ds[e] = y * (ds[e] - delta);
    }
    if (BIAS) {
      const int lo = j0 - (r0 + 31) - off, hi = j0 + 31 - r0 - off;  // this wave's positions
      if (hi <= -a.max_distance) {
#pragma unroll
        for (int e = 0; e < 16; ++e) before += ds[e];
      } else if (lo >= a.max_distance) {
#pragma unroll
        for (int e = 0; e < 16; ++e) after += ds[e];
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          __hip_atomic_fetch_add(mine + (j0 + elem_row(e, g) - i - off), ds[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const V df = pack8<T>(ds, s);
#pragma unroll
      for (int d = 0; d < DB; ++d) dq[d] = Frag<T>::mfma(col_frag<T, DP>(sk[buf], 16 * s, d * 32), df, dq[d]);
    }
  }
  if (i < a.lq) {
    const int64_t at = (((int64_t)b * a.lq + i) * a.heads + h) * a.d;
    store_head_row<T, DP>((T*)a.dq + at, dq, a.scale, a.d);
  }
  if (BIAS) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      before += __shfl_xor(before, s);
      after += __shfl_xor(after, s);
    }
    __syncthreads();
    if (l32 == 0) {  // (the group's ends hold nothing of tiles in range)
      mine[-reach] += before;
      mine[reach] += after;
    }
    __syncthreads();
    // bucket of a direction: distances edges[u] .. edges[u + 1] - 1 (the last: all further ones)
    const int u = threadIdx.x % a.one_way, side = threadIdx.x / a.one_way;  // side 0: key at or before the query
    if (threadIdx.x < a.buckets) {
      float s = 0.f;
      const int d1 = u + 1 < a.one_way ? a.edges[u + 1] : reach + 1;
      for (int dist = a.edges[u]; dist < d1; ++dist) {
        if (side == 1 && dist == 0) continue;
        const float* at = sums + reach + (side == 1 ? dist : -dist);
#pragma unroll
        for (int w = 0; w < 8; ++w) s += at[w * places];
      }
      a.part_table[((int64_t)h * a.table_parts + (int64_t)b * (a.table_parts / a.batch) + block) * a.buckets + threadIdx.x] = s;
    }
  }
}

// dtable[bucket, h]: the workgroups' sums in order; 64 lanes a (bucket, head).
template <class T>
__global__ __launch_bounds__(64) void attn_table_kernel(AttnArgs a) {
  const int bucket = blockIdx.x % a.buckets, h = blockIdx.x / a.buckets;
  const float* p = a.part_table + (int64_t)h * a.table_parts * a.buckets + bucket;
  float s = 0.f;
  for (int t = threadIdx.x; t < a.table_parts; t += 64) s += p[(int64_t)t * a.buckets];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  if (threadIdx.x == 0) ((T*)a.dtable)[(int64_t)bucket * a.heads + h] = (T)s;
}

template <class T, int DP, bool BIAS>
hipError_t launch_width(const AttnArgs& a, hipStream_t s) {
  const int64_t qblocks = (a.lq + kAttnRows - 1) / kAttnRows, kblocks = (a.lk + kAttnRows - 1) / kAttnRows;
  const size_t tab = BIAS ? (2 * a.max_distance + 1) * sizeof(float) : 0;
  const size_t sums = BIAS ? 8 * (2 * (a.max_distance + 64) + 1) * sizeof(float) : 0;
  if (kblocks > 0)
    hipLaunchKernelGGL((attn_backward_kv_kernel<T, DP, BIAS>), dim3((unsigned)(kblocks * a.batch * a.k_heads)), dim3(kBlock),
                       tab, s, a);
  if (qblocks > 0)
    hipLaunchKernelGGL((attn_backward_q_kernel<T, DP, BIAS>), dim3((unsigned)(qblocks * a.batch * a.heads)), dim3(kBlock),
                       tab + sums, s, a);
  return hipGetLastError();
}

template <class T, bool BIAS>
hipError_t launch_bias(const AttnArgs& a, hipStream_t s) {
  if (a.d <= 32) return launch_width<T, 32, BIAS>(a, s);
  if (a.d <= 64) return launch_width<T, 64, BIAS>(a, s);
  return launch_width<T, 128, BIAS>(a, s);
}

template <class T>
hipError_t backward(const AttnArgs& a, hipStream_t s) {
  const int64_t rows = (int64_t)a.batch * a.lq * a.heads;
  if (rows > 0)
    hipLaunchKernelGGL(attn_delta_kernel<T>, dim3((unsigned)((rows + kBlock / 8 - 1) / (kBlock / 8))), dim3(kBlock), 0,
                       s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (a.table == nullptr) return launch_bias<T, false>(a, s);
  e = launch_bias<T, true>(a, s);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(attn_table_kernel<T>, dim3(a.buckets * a.heads), dim3(64), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attn_backward(const AttnArgs& a, hipStream_t s) {
  return a.type == kF16 ? backward<_Float16>(a, s) : backward<__bf16>(a, s);
}

}  // namespace cvs
