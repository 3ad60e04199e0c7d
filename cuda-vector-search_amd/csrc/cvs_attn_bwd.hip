// Attention, backward: the probabilities are computed again from q, k and the rows' log sums,
//   p_ij = exp(scale q_i . k_j + bias(j - i) - lse_i),   dv_j = sum_i p_ij dout_i,
//   ds_ij = p_ij (dout_i . v_j - delta_i), delta_i = dout_i . out_i,
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,
//   dtable[bucket, h] = sum of ds_ij over the pairs whose position falls in the bucket.
//
// Two kernels, each with sums that no other workgroup adds to: one walks the keys for 128
// queries (delta, dq, dtable), then one the queries for 128 keys (dk, dv; the query heads
// that share a key head one after the other).  That computes the scores and dout . v twice
// (seven products instead of five), and needs neither atomics, whose order would
// change results, nor a pass that adds up partial dq.  As in the forward kernel, a block
// of scores is oriented so that, packed to 16 bits, it is an operand of the next
// product in registers, and the products start from what is added to them: scores from
// the bias, dout . v from -delta.  Probabilities and ds are rounded to the inputs' type for
// those products; everything else is fp32.
//
// Rows that see nothing, and keys that no row sees, are not read, and have no gradient.
//
// Where all of a wave's rows see at most the first tile of keys (sequences of that many keys, the
// first rows of causal ones) they take delta from the probabilities themselves, normalised
// again: few keys leave ds small beside its terms, and the rounding of out would be most of
// it.  (The rows after them take it from out, with that rounding.)
#include <algorithm>

#include "cvs_attn_tile.h"

namespace cvs {

namespace {

constexpr float kNever = __builtin_inff();

// float16 holds ds of long rows and small gradients only as subnormals (p of 1 / 3000 times
// dout . v of 2^-12 has few digits left: dq off by 2%), so probabilities are taken times 2^10
// there, by their exponent, and sums divided at the end: what a ds then loses is 2^-35 at
// most, and 8192 of them, each against an operand of 1 and times a scale of 1/8, come to half the
// spacing of the result's own subnormals.  A ds past 2^5 takes less than 2^10: the q kernel
// lowers the exponent of a column (a query) when a tile brings one, and leaves each workgroup's
// largest for the kv kernel, which takes one factor for a key head from those.  (The pass
// of 32 sequences of up to 512, 12 heads of 64, bias, 112 us against 109 without any of this, causal
// 2 x 4096, 16 heads on 4 of 128, 579 both; with a column's own exponent in the kv kernel too 606.)
template <class T>
constexpr int kLift = 0;
template <>
constexpr int kLift<_Float16> = 10;
template <class T>
constexpr float kUnlift = 1.f / (1 << kLift<T>);
constexpr int kTop = 15;  // lifted values stay below 2^15, or the sums of a rounding more

// The exponent that brings values of at most `top` below 2^kTop.
__device__ __forceinline__ int room(float top) { return kTop - __builtin_amdgcn_frexp_expf(top); }

__device__ __forceinline__ float largest(const f32x16& v, float top) {
#pragma unroll
  for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(v[e]));
  return top;
}
template <int DB>
__device__ __forceinline__ void times(f32x16* sums, float factor) {
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) sums[d][e] *= factor;
}
// A column's state in the q kernel.
struct Lifted {
  float lift, unit = 1.f;  // its exponent; what a value times 2^kLift is of one times 2^lift
  float peak = 0.f;        // its largest value so far, times 2^lift
};

// Lowers the exponents of columns whose values, of which this lane's largest is `top`, pass 2^kTop,
// with these values and the sums so far.
template <int DB, int N>
__device__ __forceinline__ void fit_half(float top, Lifted& c, f32x16* sums, f32x16* ds) {
  c.peak = fmaxf(c.peak, top);
  if (__builtin_expect(__any(top > (float)(1 << kTop)), 0)) {
    const int past = max(-room(halves_max(top)), 0);
    const float change = ldexpf(1.f, -past);
    c.lift -= past;
    c.unit = ldexpf(c.unit, past);
    c.peak *= change;
    times<DB>(sums, change);
    times<N>(ds, change);
  }
}
// The wave's largest, in every lane: across its halves and quarters, then around each 16 lanes.
__device__ __forceinline__ float wave_max(float v) {
  v = halves_max(v);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xf, 0xf, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x124, 0xf, 0xf, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x122, 0xf, 0xf, false)));
  return fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x121, 0xf, 0xf, false)));
}

// Rows of a streamed tile: 64, or 32 of width 128 (two workgroups' tiles fit a CU's LDS).
template <int DP>
constexpr int kTile = DP > 64 ? 32 : 64;

// dtable's sums.  A block of ds, laid out by position (row j - i + 31, pitch 36 words: column
// writes and row reads without bank conflicts; places that no pair of the block has stay
// zero), is added along the rows, a position a lane, in a fixed order.  (LDS atomics
// instead took 192 cycles each: 281 us of 32 sequences of up to 512, 12 heads of 64.)
constexpr int kSkewPitch = 36, kSkew = 64 * kSkewPitch;

__device__ __forceinline__ void put_positions(float* skew, const f32x16& ds) {
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  float* to = skew + (8 * g - l32 + 31) * kSkewPitch + l32;
#pragma unroll
  for (int e = 0; e < 16; ++e) to[elem_row(e, 0) * kSkewPitch] = ds[e];
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
}
__device__ __forceinline__ void take_positions(const float* skew, float* sums) {
  const int lane = threadIdx.x & 63;
  const f32x4* from = reinterpret_cast<const f32x4*>(skew + lane * kSkewPitch);
  f32x4 s = from[0];
#pragma unroll
  for (int q = 1; q < 8; ++q) s += from[q];
  sums[lane] += (s[0] + s[1]) + (s[2] + s[3]);
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
}

// delta, dq of 128 queries (wave w: 32 of them as columns), and their sums for dtable.  The queries'
// rows stay in registers, tiles of keys and values come into two LDS buffers in turn, and two
// workgroups a CU fill each other's waits.  Bound by issue of the matrix and vector instructions
// of a block, one after the other in a wave (the softmax's exponentials, the packing; with a bias
// also the positions' sums): 2 x 4096, 16 heads of 128, causal 217 us, 0.95 PFLOP/s of its three
// products; 64 x 512, 12 heads of 64, 122 us, with a bias 156; at short sequences by a
// workgroup's start and end, some 7 us (32 sequences of up to 512, 12 heads of 64, bias: 58 us).
template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(kBlock, 2) void attn_backward_q_kernel(AttnArgs a) {
  typedef typename Frag<T>::V V;
  constexpr int KS = DP / 16, DB = DP / 32, ROWS = kTile<DP>, KB = ROWS / 32, TILE = ROWS * DP * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char sk[2][TILE], sv[2][TILE];
  __shared__ __attribute__((aligned(16))) float skew[BIAS ? 4 : 1][BIAS ? kSkew : 4];
  __shared__ float peaks[4];
  extern __shared__ float tab[];  // bias by position, then the waves' sums by position

  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = a.batch * a.heads;
  // the last rows first: those see most keys when causal, and are of the longest sequences
  const int block = (a.lq + kAttnRows - 1) / kAttnRows - 1 - blockIdx.x / heads;
  const int bh = blockIdx.x % heads;
  const int b = bh / a.heads, h = bh % a.heads, hk = h / (a.heads / a.k_heads);
  const int nk = key_count(a, b), nq = query_count(a, b), off = query_offset(a, b);
  const int r0 = block * kAttnRows + wave * 32;
  const int i = r0 + l32;
  const unsigned char* qrow = (const unsigned char*)a.q + 2 * (b * a.qs[0] + i * a.qs[1] + h * a.qs[2]);
  const unsigned char* grow = (const unsigned char*)a.dout + 2 * (b * a.dos[0] + i * a.dos[1] + h * a.dos[2]);
  const unsigned char* orow = (const unsigned char*)a.out + 2 * ((((int64_t)b * a.lq + i) * a.heads + h) * a.d);
  const unsigned char* kbase = (const unsigned char*)a.k + 2 * (b * a.ks[0] + hk * a.ks[2]);
  const unsigned char* vbase = (const unsigned char*)a.v + 2 * (b * a.vs[0] + hk * a.vs[2]);

  const int last_row = min(block * kAttnRows + kAttnRows, nq) - 1;
  int end = last_row < block * kAttnRows ? 0 : nk;
  if (a.causal) end = min(end, max(last_row + off + 1, 0));
  const int all = (end + ROWS - 1) / ROWS;
  // this wave's rows see keys of the first tile only
  const bool one = (a.causal ? min(nk, r0 + 32 + off) : nk) <= ROWS;
  // this workgroup's part of the tiles (fewer than 2^24, at most 64 parts); the first part writes
  // delta, or, where the wave's rows take it from the first tile, the part that has it
  int t0 = 0, tiles = all;
  if (a.q_parts > 1) {
    t0 = (int)((unsigned)all * blockIdx.y / (unsigned)a.q_parts);
    tiles = (int)((unsigned)all * (blockIdx.y + 1) / (unsigned)a.q_parts);
  }
  const bool writes_delta = one && all > 0 ? t0 == 0 && tiles > 0 : blockIdx.y == 0;
  BiasLoad<T> bias;
  if (BIAS) bias.buckets(a);
  const TileLoad<DP, ROWS> lk(2 * a.ks[1], a.d), lv(2 * a.vs[1], a.d);
  auto load = [&](int t) {
    lk.load(kbase, 2 * a.ks[1], t * ROWS, end, sk[t & 1]);
    lv.load(vbase, 2 * a.vs[1], t * ROWS, end, sv[t & 1]);
  };
  if (t0 < tiles) load(t0);

  // the first loads are all on their way before one is waited for: the keys' and values' tiles,
  // the bias, the rows, and under them shared memory is cleared
  V qf[KS], gf[KS], of[KS];
  const bool in = i >= first_row(a, off) && i < nq;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    qf[s] = global_frag<T>(qrow, s, a.d, in);
    gf[s] = global_frag<T>(grow, s, a.d, in);
    of[s] = global_frag<T>(orow, s, a.d, in);
  }
  const int64_t row_at = (int64_t)bh * a.lq + i;
  float lse = in ? a.lse[row_at] * kLog2e : kNever;
  if (BIAS) bias.values(a, h);
  const int reach = a.far + kReach, places = 2 * reach + 1;
  float* sums = tab + places + wave * places + reach;  // by position, this wave's
  float before = 0.f, after = 0.f;                     // positions all <= -far, all >= far
  if (BIAS) {
    for (int t = threadIdx.x; t < 4 * places; t += kBlock) tab[places + t] = 0.f;
    for (int t = threadIdx.x; t < kSkew; t += kBlock) reinterpret_cast<f32x4*>(&skew[0][0])[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    bias.store(a, tab);
  }
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) delta = fmaf((float)gf[s][j], (float)of[s][j], delta);
  delta = one ? 0.f : halves_sum(delta);
  const bool blind = !in || lse == -__builtin_inff();  // a row that sees nothing
  if (blind) lse = kNever;

  f32x16 dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dq[d] = zero16();
  const float c = a.scale * kLog2e;
  Lifted col = {kLift<T>};  // of this column's probabilities and ds

  // the tiles that a row of this wave sees a key of; through the others it only loads its share
  int mine = r0 < nq ? tiles : t0;
  if (a.causal) mine = max(t0, min(mine, (r0 + 32 + off + ROWS - 1) / ROWS));
  for (int t = t0; t < mine; ++t) {
    const int buf = t & 1;
    tile_barrier();
    if (t + 1 < tiles) load(t + 1);
    f32x16 ds[KB], p[KB];
    float base[KB];
    const int near0 = t * ROWS - r0 - off;  // position of the tile's first key and the wave's first row
    V krows[KB][KS], vrows[KB][KS], kcols[KB][2][DB];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) krows[kb][s] = row_frag<T, DP>(sk[buf], kb * 32, s);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int near = near0 + kb * 32;
      base[kb] = col.lift - lse;
      if (BIAS) {
        if (near - 31 >= a.far || near + 31 <= -a.far) {
          base[kb] += tab[near > 0 ? 2 * reach : 0] * c;
          p[kb] = zero16();
        } else {
          const float* at = tab + (near - l32 + 8 * g + reach);
#pragma unroll
          for (int e = 0; e < 16; ++e) p[kb][e] = at[elem_row(e, 0)];
        }
      } else {
        p[kb] = zero16();
      }
    }
    auto read_vrows = [&]() {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) vrows[kb][s] = row_frag<T, DP>(sv[buf], kb * 32, s);
    };
    auto read_kcols = [&]() {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int d = 0; d < DB; ++d) kcols[kb][s][d] = col_frag<T, DP>(sk[buf], kb * 32 + 16 * s, d * 32);
    };
    if (DP <= 64) {
      keep_order();
      read_vrows();
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) p[kb] = Frag<T>::mfma(krows[kb][s], qf[s], p[kb]);
    if (DP <= 64) {
      keep_order();
      read_kcols();
    } else {  // no registers to read ahead with
      read_vrows();
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) ds[kb] = splat16(-delta);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) ds[kb] = Frag<T>::mfma(vrows[kb][s], gf[s], ds[kb]);
    if (DP <= 64)
      keep_order();
    else
      read_kcols();
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int j0 = t * ROWS + kb * 32;
#pragma unroll
      for (int e = 0; e < 16; ++e) p[kb][e] = __builtin_amdgcn_exp2f(fmaf(p[kb][e], c, base[kb]));
      if (j0 + 32 > nk || (a.causal && near0 + kb * 32 + 31 > 0)) {
        const int seen = min(nk - 1, a.causal ? i + off : nk) - j0 - 8 * g;  // last key of the block that the row sees
#pragma unroll
        for (int e = 0; e < 16; ++e) p[kb][e] = elem_row(e, 0) > seen ? 0.f : p[kb][e];
      }
    }
    if (one) {
      float sp = 0.f, spd = 0.f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) sp += p[kb][e];
      sp = halves_sum(sp);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          p[kb][e] = sp == 0.f ? 0.f : p[kb][e] / sp;
          spd = fmaf(p[kb][e], ds[kb][e], spd);
          if (kLift<T> != 0) p[kb][e] *= __builtin_amdgcn_exp2f(col.lift);
        }
      delta = halves_sum(spd);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[kb][e] -= delta;
    }
    if constexpr (kLift<T> != 0) {
      float top = 0.f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[kb][e] *= p[kb][e];
        top = largest(ds[kb], top);
      }
      fit_half<DB, KB>(top, col, dq, ds);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int near = near0 + kb * 32;
      const bool in_range = near + 31 > -a.far && near - 31 < a.far;
      if constexpr (kLift<T> == 0) {
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[kb][e] *= p[kb][e];
      }
      if (BIAS) {
        if (in_range) {
          if (kLift<T> == 0 || !__any(col.unit != 1.f)) {
            put_positions(skew[wave], ds[kb]);
          } else {
            f32x16 alike = ds[kb];
            times<1>(&alike, col.unit);
            put_positions(skew[wave], alike);
          }
        } else {
          float s = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) s += ds[kb][e];
          if (kLift<T> != 0) s *= col.unit;
          if (near < 0)
            before += s;
          else
            after += s;
        }
        keep_order();  // (the sums' places settle in LDS under the products)
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const V df = pack8<T>(ds[kb], s);
#pragma unroll
        for (int d = 0; d < DB; ++d) dq[d] = Frag<T>::mfma(kcols[kb][s][d], df, dq[d]);
      }
      if (BIAS) {
        keep_order();
        if (in_range) take_positions(skew[wave], sums + near - 31);
      }
    }
  }
  for (int t = mine; t < tiles; ++t) {
    tile_barrier();
    if (t + 1 < tiles) load(t + 1);
  }
  if (blind) {  // (the sums may be NaN: 0 times a value that other rows see)
    delta = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) dq[d] = zero16();
  }
  if (i < a.lq) {
    const int64_t at = (((int64_t)b * a.lq + i) * a.heads + h) * a.d;
    const float undo = kUnlift<T> * col.unit;
    if (a.q_parts > 1) {
      if (kLift<T> != 0) times<DB>(dq, undo);
      store_part_row<DP>(a.part_q + (int64_t)blockIdx.y * a.batch * a.lq * a.heads * a.d + at, dq, a.d);
    } else {
      store_head_row<T, DP>((T*)a.dq + at, dq, a.scale * undo, a.d);
    }
    if (g == 0 && writes_delta) a.delta[row_at] = delta;
  }
  if constexpr (kLift<T> != 0) {
    const float top = wave_max(col.peak * col.unit * kUnlift<T>);
    if (lane == 0) peaks[wave] = top;
    __syncthreads();
    const int blocks = (a.lq + kAttnRows - 1) / kAttnRows;
    if (threadIdx.x == 0)
      a.part_peak[((int64_t)bh * a.q_parts + blockIdx.y) * blocks + block] = fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3]));
  }
  if (BIAS) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) {
      before += __shfl_xor(before, s);
      after += __shfl_xor(after, s);
    }
    __syncthreads();
    if (lane == 0) {  // (the ends hold nothing of blocks in range)
      sums[-reach] = before;
      sums[reach] = after;
    }
    __syncthreads();
    // bucket of a direction: distances edges[u] .. edges[u + 1] - 1 (the last: all further
    // ones), a power of two of lanes to a bucket
    int lanes = 2;
    while (2 * lanes * a.buckets <= kBlock) lanes *= 2;
    const int bucket = threadIdx.x / lanes, l = threadIdx.x % lanes;
    float s = 0.f;
    if (bucket < a.buckets) {
      const int u = bucket % a.one_way, side = bucket / a.one_way;  // side 0: key at or before the query
      const int d0 = max((int)a.edges[u], side), d1 = u + 1 < a.one_way ? (int)a.edges[u + 1] : reach + 1;
#pragma unroll 4
      for (int dist = d0 + l; dist < d1; dist += lanes) {
        const float* at = tab + places + reach + (side == 1 ? dist : -dist);
        s += (at[0] + at[places]) + (at[2 * places] + at[3 * places]);
      }
    }
    for (int o = lanes / 2; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (bucket < a.buckets && l == 0)
      a.part_table[((int64_t)h * a.table_parts + ((int64_t)b * a.q_parts + blockIdx.y) * ((a.lq + kAttnRows - 1) / kAttnRows) +
                    block) * a.buckets + bucket] = s * kUnlift<T>;
  }
}

// dtable[bucket, h]: the q kernel's workgroups' sums in order; a wave a (bucket, head).
template <class T>
__device__ __forceinline__ void add_table(const AttnArgs& a, int at) {
  if (at >= a.buckets * a.heads) return;
  const int bucket = at % a.buckets, h = at / a.buckets, lane = threadIdx.x & 63;
  const float* p = a.part_table + (int64_t)h * a.table_parts * a.buckets + bucket;
  float s = 0.f;
  for (int t = lane; t < a.table_parts; t += 64) s += p[(int64_t)t * a.buckets];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  if (lane == 0) ((T*)a.dtable)[(int64_t)bucket * a.heads + h] = (T)s;
}

// dk and dv of 128 keys (wave w: 32 of them as columns), over a part of the queries that see
// them.  Where there is a bias, the workgroups from `key_wgs` on add up its table's gradient.
// The keys' rows of both operands and both sums stay in registers, at width 128 some 420 of them:
// one wave a SIMD then, whose products (37% of the time), exponentials and packing follow one
// another.  2 x 4096, 16 heads on 4 of 128, causal: 329 us, 0.84 PFLOP/s of its four products;
// 64 x 512, 12 heads of 64, two workgroups a CU: 148 us, with a bias 156.
template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(kBlock, DP > 64 ? 1 : 2) void attn_backward_kv_kernel(AttnArgs a, int key_wgs) {
  typedef typename Frag<T>::V V;
  constexpr int KS = DP / 16, DB = DP / 32, ROWS = 64, QB = ROWS / 32, TILE = ROWS * DP * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char sq[2][TILE], sg[2][TILE];
  __shared__ __attribute__((aligned(16))) float slse[2][ROWS], sdelta[2][ROWS];  // kLift - log2 sums, -deltas
  extern __shared__ float tab[];

  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (BIAS && (int)blockIdx.x >= key_wgs) {
    if (blockIdx.y == 0) add_table<T>(a, ((int)blockIdx.x - key_wgs) * 4 + wave);
    return;
  }
  const int kheads = a.batch * a.k_heads, group = a.heads / a.k_heads;
  // keys of most queries first: the first ones when causal, else those of the longest sequences
  const int bk = blockIdx.x % kheads;
  const int block = a.causal ? blockIdx.x / kheads : (a.lk + kAttnRows - 1) / kAttnRows - 1 - blockIdx.x / kheads;
  const int b = bk / a.k_heads, hk = bk % a.k_heads;
  const int nk = key_count(a, b), nq = query_count(a, b), off = query_offset(a, b);
  const int j0 = block * kAttnRows + wave * 32;
  const int j = j0 + l32;
  const unsigned char* krow = (const unsigned char*)a.k + 2 * (b * a.ks[0] + j * a.ks[1] + hk * a.ks[2]);
  const unsigned char* vrow = (const unsigned char*)a.v + 2 * (b * a.vs[0] + j * a.vs[1] + hk * a.vs[2]);
  const int row0 = min(first_row(a, off), nq), seen_keys = seen_count(a, nk, nq, off);
  float shrink = 1.f;  // of this workgroup's ds, where they would not fit
  V kf[KS], vf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    kf[s] = global_frag<T>(krow, s, a.d, j < seen_keys);
    vf[s] = global_frag<T>(vrow, s, a.d, j < seen_keys);
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dk[d] = dv[d] = zero16();
  const float c = a.scale * kLog2e;
  const int reach = a.far + kReach;
  const bool one = nk <= ROWS;  // delta is made of dout . v's own sums: subtracted as they stand, so that one key leaves 0

  // tiles of queries that see a key of this workgroup, those of all heads in a row; this part's
  const int t0 = (a.causal ? max(block * kAttnRows - off, 0) : 0) / ROWS;
  const int nt = block * kAttnRows < seen_keys ? max((nq + ROWS - 1) / ROWS - t0, 0) : 0;
  int f0 = 0, f1 = nt * group;
  if (a.kv_parts > 1) {
    const int64_t all = f1;
    f0 = (int)(all * blockIdx.y / a.kv_parts);
    f1 = (int)(all * (blockIdx.y + 1) / a.kv_parts);
  }
  const TileLoad<DP, ROWS> lq(2 * a.qs[1], a.d), lg(2 * a.dos[1], a.d);
  BiasLoad<T> bias;
  if (BIAS) bias.buckets(a);
  while (f0 < f1) {
    const int hh = f0 / nt, h = hk * group + hh;
    const int first = t0 + f0 % nt, last = min(t0 + nt, first + f1 - f0);  // this head's
    f0 += last - first;
    const unsigned char* qbase = (const unsigned char*)a.q + 2 * (b * a.qs[0] + h * a.qs[2]);
    const unsigned char* gbase = (const unsigned char*)a.dout + 2 * (b * a.dos[0] + h * a.dos[2]);
    const float* lse = a.lse + ((int64_t)b * a.heads + h) * a.lq;
    const float* delta = a.delta + ((int64_t)b * a.heads + h) * a.lq;
    __syncthreads();  // the last head's tiles and bias have been read
    if (BIAS) bias.values(a, h);
    float stat = 0.f;  // threads 0 .. ROWS - 1: -log2 sum of a row, the next ROWS: -delta
    auto load = [&](int t) {
      lq.load(qbase, 2 * a.qs[1], t * ROWS, nq, sq[t & 1], row0);
      lg.load(gbase, 2 * a.dos[1], t * ROWS, nq, sg[t & 1], row0);
      const int i = t * ROWS + threadIdx.x % ROWS;
      if (threadIdx.x < ROWS) {
        stat = i >= row0 && i < nq ? -lse[i] * kLog2e : -kNever;
        if (stat == __builtin_inff()) stat = -kNever;  // a row that sees nothing
      } else if (threadIdx.x < 2 * ROWS) {
        stat = i >= row0 && i < nq ? -delta[i] : 0.f;
      }
    };
    auto turn = [&](int t) {
      if (threadIdx.x < ROWS)
        slse[t & 1][threadIdx.x] = stat + kLift<T>;
      else if (threadIdx.x < 2 * ROWS)
        sdelta[t & 1][threadIdx.x - ROWS] = stat;
      tile_barrier();
      if (t + 1 < last) load(t + 1);
    };
    load(first);
    if (BIAS) bias.store(a, tab);
    if constexpr (kLift<T> != 0) {  // (under the first tile's loads)
      const int64_t count = (int64_t)group * a.q_parts * ((a.lq + kAttnRows - 1) / kAttnRows);
      const float* from = a.part_peak + bk * count;
      float peak = 0.f;  // of the heads that share this one
      for (int64_t t = lane; t < count; t += 64) peak = fmaxf(peak, from[t]);
      const int past = __builtin_amdgcn_readfirstlane(kLift<T> - room(wave_max(peak)));
      shrink = ldexpf(1.f, -max(past, 0));
    }
    // tiles that no key of this wave is seen from come first: it only loads its share of them
    int mine = j0 < seen_keys ? first : last;
    if (a.causal) mine = min(last, max(mine, (j0 - off) / ROWS));
    for (int t = first; t < mine; ++t) turn(t);
    for (int t = mine; t < last; ++t) {
      const int buf = t & 1;
      turn(t);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const int i0 = t * ROWS + qb * 32;
        const int near = j0 - i0 - off;
        V qrows[KS], grows[KS], qcols[2][DB], gcols[2][DB];
        f32x16 p, ds, base;
        float shift = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) qrows[s] = row_frag<T, DP>(sq[buf], qb * 32, s);
        if (BIAS) {
          if (near - 31 >= a.far || near + 31 <= -a.far) {
            shift = tab[near > 0 ? 2 * reach : 0] * c;
            p = zero16();
          } else {
            const float* at = tab + (near + l32 - 8 * g + reach);
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = at[-elem_row(e, 0)];
          }
        } else {
          p = zero16();
        }
        keep_order();
#pragma unroll
        for (int s = 0; s < KS; ++s) grows[s] = row_frag<T, DP>(sg[buf], qb * 32, s);
        if (one) {
          ds = zero16();
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) ds[e] = sdelta[buf][qb * 32 + elem_row(e, g)];
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) p = Frag<T>::mfma(qrows[s], kf[s], p);
        keep_order();
#pragma unroll
        for (int e = 0; e < 16; ++e) base[e] = slse[buf][qb * 32 + elem_row(e, g)];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int d = 0; d < DB; ++d) gcols[s][d] = col_frag<T, DP>(sg[buf], qb * 32 + 16 * s, d * 32);
#pragma unroll
        for (int s = 0; s < KS; ++s) ds = Frag<T>::mfma(grows[s], vf[s], ds);
        keep_order();
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int d = 0; d < DB; ++d) qcols[s][d] = col_frag<T, DP>(sq[buf], qb * 32 + 16 * s, d * 32);
        if (one) {
#pragma unroll
          for (int e = 0; e < 16; ++e) ds[e] += sdelta[buf][qb * 32 + elem_row(e, g)];
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(p[e], c, BIAS ? base[e] + shift : base[e]));
        if (a.causal && near + 31 > 0) {
          const int seen = j - off - i0 - 8 * g;  // first row of the block that sees the key
#pragma unroll
          for (int e = 0; e < 16; ++e) p[e] = elem_row(e, 0) < seen ? 0.f : p[e];
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[e] *= p[e];
        if (kLift<T> != 0 && shrink != 1.f) times<1>(&ds, shrink);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const V pf = pack8<T>(p, s), df = pack8<T>(ds, s);
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            dv[d] = Frag<T>::mfma(gcols[s][d], pf, dv[d]);
            dk[d] = Frag<T>::mfma(qcols[s][d], df, dk[d]);
          }
        }
      }
    }
  }
  if (j >= a.lk) return;
  if (j >= seen_keys) {
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[d] = dv[d] = zero16();
  }
  const int64_t at = (((int64_t)b * a.lk + j) * a.k_heads + hk) * a.d;
  const float undo = kUnlift<T> / shrink;
  if (a.kv_parts > 1) {
    if (kLift<T> != 0) times<DB>(dk, undo), times<DB>(dv, kUnlift<T>);
    const int64_t all = (int64_t)a.batch * a.lk * a.k_heads * a.d;
    float* to = a.part_kv + 2 * blockIdx.y * all + at;
    store_part_row<DP>(to, dk, a.d);
    store_part_row<DP>(to + all, dv, a.d);
    return;
  }
  store_head_row<T, DP>((T*)a.dk + at, dk, a.scale * undo, a.d);
  store_head_row<T, DP>((T*)a.dv + at, dv, kUnlift<T>, a.d);
}

// Adds `parts` of n values, `stride` apart, in order: 8 a thread; blockIdx.y: the second of two sums
// beside each other.  dk and dv of 8192 x 4 heads of 128 in 2 parts, 67 MB read and 17 written: 12.9 us,
// 6.5 TB/s, more than memory's 5.1, so that part of the sums still comes from the cache.
template <class T>
__global__ __launch_bounds__(kBlock) void attn_join_grads_kernel(const float* part, int parts, int64_t stride, int64_t n, float scale0,
                                                                 T* out0, T* out1) {
  const int64_t at = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * 8;
  if (at >= n) return;
  f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
  for (int p = 0; p < parts; ++p) {
    const f32x4* from = reinterpret_cast<const f32x4*>(part + p * stride + blockIdx.y * n + at);
    lo += from[0];
    hi += from[1];
  }
  const float scale = blockIdx.y == 0 ? scale0 : 1.f;
  typename Frag<T>::V v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (T)(lo[e] * scale), v[4 + e] = (T)(hi[e] * scale);
  *reinterpret_cast<typename Frag<T>::V*>((blockIdx.y == 0 ? out0 : out1) + at) = v;
}

template <class T, int DP, bool BIAS>
hipError_t launch_width(const AttnArgs& a, hipStream_t s) {
  const int64_t qblocks = (a.lq + kAttnRows - 1) / kAttnRows, kblocks = (a.lk + kAttnRows - 1) / kAttnRows;
  const size_t tab = BIAS ? (2 * (a.far + kReach) + 1) * sizeof(float) : 0;
  if (qblocks > 0)
    hipLaunchKernelGGL((attn_backward_q_kernel<T, DP, BIAS>), dim3((unsigned)(qblocks * a.batch * a.heads), a.q_parts),
                       dim3(kBlock), 5 * tab, s, a);
  const int64_t key_wgs = kblocks * a.batch * a.k_heads, all_wgs = key_wgs + (BIAS ? (a.buckets * a.heads + 3) / 4 : 0);
  if (all_wgs > 0)
    hipLaunchKernelGGL((attn_backward_kv_kernel<T, DP, BIAS>), dim3((unsigned)all_wgs, a.kv_parts), dim3(kBlock), tab, s, a,
                       (int)key_wgs);
  auto join = [&](const float* part, int parts, int64_t n, int sums, float scale, void* out0, void* out1) {
    const dim3 grid((unsigned)((n / 8 + kBlock - 1) / kBlock), sums);
    hipLaunchKernelGGL(attn_join_grads_kernel<T>, grid, dim3(kBlock), 0, s, part, parts, sums * n, n, scale, (T*)out0, (T*)out1);
  };
  if (a.q_parts > 1) join(a.part_q, a.q_parts, (int64_t)a.batch * a.lq * a.heads * a.d, 1, a.scale, a.dq, nullptr);
  if (a.kv_parts > 1) join(a.part_kv, a.kv_parts, (int64_t)a.batch * a.lk * a.k_heads * a.d, 2, a.scale, a.dk, a.dv);
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
  return a.table == nullptr ? launch_bias<T, false>(a, s) : launch_bias<T, true>(a, s);
}

}  // namespace

// Parts of the keys for dq, and of the queries for dk and dv: enough workgroups for two of a CU,
// of at least 8 tiles each.  (dq of 128 rows over 8192 keys, 8 heads of 64: the backward pass 35 us,
// 141 with whole rows; dk and dv of 128 keys from 8192 rows: 39 us, 207 whole.  Causal, 2 x 4096 of
// 16 heads on 4 of 128, 256 workgroups of unequal work: the pass 563 us in 2 parts, 590 in 4, whose
// sums weigh more than their balance gains, 790 whole; not causal 1060 and 1094; 2000 rows, 12 heads
// of 64 81 and 85; but causal 8192 rows, 8 heads on 1 of 128 932 for two workgroups a CU and 874 for four.)
int attn_q_parts(const AttnArgs& a, int cus) {
  const int64_t wgs = (a.lq + kAttnRows - 1) / kAttnRows * (int64_t)a.batch * a.heads;
  return (int)std::max<int64_t>(1, std::min<int64_t>({2 * cus / wgs, a.lk / 512, (int64_t)64}));
}
int attn_kv_parts(const AttnArgs& a, int cus) {
  const int64_t wgs = (a.lk + kAttnRows - 1) / kAttnRows * (int64_t)a.batch * a.k_heads;
  const int64_t tiles = (a.lq + 63) / 64 * (int64_t)(a.heads / a.k_heads);
  return (int)std::max<int64_t>(1, std::min<int64_t>({2 * cus / wgs, tiles / 8, (int64_t)16}));
}

hipError_t launch_attn_backward(const AttnArgs& a, hipStream_t s) {
  return a.type == kF16 ? backward<_Float16>(a, s) : backward<__bf16>(a, s);
}

}  // namespace cvs
