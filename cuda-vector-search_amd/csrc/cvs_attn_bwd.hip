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

// A window's gradients round what the products take to 16 bits; dk's and dv's sums over many rows average those
// roundings.  Of few rows they do not: there the products take what was rounded off too.  (100 rows of 8192 keys, 12 heads
// of 64, 4 sequences: 76 us for 50, delta's pass among them; a row alone would be 1.9 times as far off as its rounding.)
__host__ __device__ __forceinline__ bool few_rows(const AttnArgs& a) { return (int64_t)a.lq * (a.heads / a.k_heads) < kAttnRows; }
// Whether a window's delta is attn_delta_kernel's: that of a sequence whose keys fill no more than a tile the q kernel
// makes from its own sums.
__host__ __device__ __forceinline__ bool exact_delta(const AttnArgs& a, bool bias, int nk, int rows) {
  return window_narrow(a) || ((bias || few_rows(a)) && nk > rows);
}

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

// delta of a window's rows: sum p dp / sum p of the sums that the gradients themselves are made of; in a narrow
// window peak + sum p (dp - peak) / sum p with the largest dp as peak: of one key it is dp itself, and ds is 0.
// dout . out has out's rounding in it, some 2^-9 of |dout| |out|, which is all that is left in sums of ds that cancel:
// the table's gradients, whose sum over a row's keys is 0 (of 2 heads, 166 keys back, an error of 3.1e-4 for 1.6e-4
// in fp16), and those of few rows.  128 rows of a workgroup, 32 of a wave as columns; a kernel of its own, so that the
// parts of dq do not each repeat it, with four workgroups' registers and LDS a CU.  Bound by vector instructions, and by start
// and end: 8 x up to 2048, 12 heads of 64, window 128, bias: 30 us (31 as a pass of the q kernel).
template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(kBlock, DP > 64 ? 2 : 4) void attn_delta_kernel(AttnArgs a) {
  typedef typename Frag<T>::V V;
  constexpr int KS = DP / 16, ROWS = kTile<DP>, KB = ROWS / 32, TILE = ROWS * DP * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char sk[2][TILE], sv[2][TILE];
  extern __shared__ float tab[];  // bias by position

  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = a.batch * a.heads;
  const int block = (a.lq + kAttnRows - 1) / kAttnRows - 1 - blockIdx.x / heads;  // (as the q kernel's)
  const int bh = blockIdx.x % heads;
  const int b = bh / a.heads, h = bh % a.heads, hk = h / (a.heads / a.k_heads);
  const int nk = key_count(a, b), nq = query_count(a, b), off = query_offset(a, b);
  if (!exact_delta(a, BIAS, nk, ROWS)) return;
  const int r0 = block * kAttnRows + wave * 32, i = r0 + l32;
  const unsigned char* qrow = (const unsigned char*)a.q + 2 * (b * a.qs[0] + i * a.qs[1] + h * a.qs[2]);
  const unsigned char* grow = (const unsigned char*)a.dout + 2 * (b * a.dos[0] + i * a.dos[1] + h * a.dos[2]);
  const unsigned char* kbase = (const unsigned char*)a.k + 2 * (b * a.ks[0] + hk * a.ks[2]);
  const unsigned char* vbase = (const unsigned char*)a.v + 2 * (b * a.vs[0] + hk * a.vs[2]);
  const int last_row = min(block * kAttnRows + kAttnRows, nq) - 1;
  const WindowTiles<ROWS> win(a, nk, block * kAttnRows + off, last_row + off);
  int row_first, row_end;  // the rows that see a key of a window
  window_rows(a, nk, nq, off, row_first, row_end);
  const TileLoad<DP, ROWS> lk(2 * a.ks[1], a.d), lv(2 * a.vs[1], a.d);
  auto load = [&](int t) {
    const int first = win.tile(t) * ROWS;
    lk.load_window(kbase, 2 * a.ks[1], first, win.end, sk[t & 1], win.low, win.head);
    lv.load_window(vbase, 2 * a.vs[1], first, win.end, sv[t & 1], win.low, win.head);
  };
  BiasLoad<T> bias;
  if (BIAS) bias.buckets(a);
  if (win.count > 0) load(0);
  V qf[KS], gf[KS];
  const bool in = i >= row_first && i < row_end;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    qf[s] = global_frag<T>(qrow, s, a.d, in);
    gf[s] = global_frag<T>(grow, s, a.d, in);
  }
  const int64_t row_at = (int64_t)bh * a.lq + i;
  float lse = in ? a.lse[row_at] * kLog2e : kNever;
  if (BIAS) {
    bias.values(a, h);
    bias.store(a, tab);
  }
  const int reach = a.far + kReach;
  const bool blind = !in || lse == -__builtin_inff();  // a row that sees nothing
  if (blind) lse = kNever;
  const float c = a.scale * kLog2e;
  const bool narrow = window_narrow(a);
  float sp = 0.f, spd = 0.f, peak = narrow ? -kNever : 0.f;
  for (int t = 0; t < win.count; ++t) {
    tile_barrier();
    if (t + 1 < win.count) load(t + 1);
    const int tile0 = win.tile(t) * ROWS;
    if (r0 >= nq) continue;
#pragma unroll 1
    for (int kb = 0; kb < KB; ++kb) {
      const int j0 = tile0 + kb * 32, near = j0 - r0 - off;
      if (!window_meets(a, j0, 32, r0 + off, min(r0 + 31, nq - 1) + off)) continue;
      V krows[KS], vrows[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) krows[s] = row_frag<T, DP>(sk[t & 1], kb * 32, s);
      f32x16 p = zero16(), dp = zero16();
      float base = -lse;
      if (BIAS) {
        if (near - 31 >= a.far || near + 31 <= -a.far) {
          base += tab[near > 0 ? 2 * reach : 0] * c;
        } else {
          const float* at = tab + (near - l32 + 8 * g + reach);
#pragma unroll
          for (int e = 0; e < 16; ++e) p[e] = at[elem_row(e, 0)];
        }
      }
      keep_order();
#pragma unroll
      for (int s = 0; s < KS; ++s) vrows[s] = row_frag<T, DP>(sv[t & 1], kb * 32, s);
#pragma unroll
      for (int s = 0; s < KS; ++s) p = Frag<T>::mfma(krows[s], qf[s], p);
      keep_order();
#pragma unroll
      for (int s = 0; s < KS; ++s) dp = Frag<T>::mfma(vrows[s], gf[s], dp);
#pragma unroll
      for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(p[e], c, base));
      if (j0 + 32 > nk || near + 31 > a.after || near < 31 - a.before) {
        WindowMask(a, nk, i + off, j0 + 8 * g).apply(p, 0, j0 < a.sinks, 0.f);
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = p[e] > 0.f ? dp[e] : peak;
      }
      if (narrow) {
        float top = -kNever;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = p[e] > 0.f ? fmaxf(top, dp[e]) : top;
        top = fmaxf(peak, halves_max(top));
        if (top > peak) {
          spd = peak == -kNever ? 0.f : fmaf(sp, peak - top, spd);
          peak = top;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = p[e] > 0.f ? dp[e] - peak : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        sp += p[e];
        spd = fmaf(p[e], dp[e], spd);
      }
    }
  }
  sp = halves_sum(sp), spd = halves_sum(spd);
  if (i < a.lq && g == 0) a.delta[row_at] = !blind && sp > 0.f ? (narrow ? peak + spd / sp : spd / sp) : 0.f;
}

// delta, dq of 128 queries (wave w: 32 of them as columns), and their sums for dtable.  The queries'
// rows stay in registers, tiles of keys and values come into two LDS buffers in turn, and two
// workgroups a CU fill each other's waits.  Bound by issue of the matrix and vector instructions
// of a block, one after the other in a wave (the softmax's exponentials, the packing; with a bias
// also the positions' sums): 2 x 4096, 16 heads of 128, causal 217 us, 0.95 PFLOP/s of its three
// products; 64 x 512, 12 heads of 64, 122 us, with a bias 156; at short sequences by a
// workgroup's start and end, some 7 us (32 sequences of up to 512, 12 heads of 64, bias: 58 us).
// Of a window dq's products take both 16-bit halves of ds: keys have much in common, and a row's ds cancel.  8 x up to
// 2048, 12 heads of 64, window 128, bias: 69 us (62 without the second halves); 8192 rows, 16 heads on 4 of 128, window
// 1024: 153 us, 0.85 PFLOP/s of its four products.
template <class T, int DP, bool BIAS, bool WIN>
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
  int all = (end + ROWS - 1) / ROWS;
  WindowTiles<ROWS> win;
  int row_first, row_end;  // the rows that see a key of a window
  const bool narrow = WIN && window_narrow(a);
  const bool exact = WIN && exact_delta(a, BIAS, nk, ROWS);  // attn_delta_kernel's
  // this wave's rows see keys of the first tile only
  bool one = (a.causal ? min(nk, r0 + 32 + off) : nk) <= ROWS;
  if constexpr (WIN) {
    win = WindowTiles<ROWS>(a, nk, block * kAttnRows + off, last_row + off);
    all = win.count;
    window_rows(a, nk, nq, off, row_first, row_end);
    one = !exact && (one || (!a.causal && min(nk, max(r0 + 32 + off + a.after, a.sinks)) <= ROWS));
  }
  // this workgroup's part of the tiles (fewer than 2^24, at most 64 parts); the first part writes
  // delta, or, where the wave's rows take it from the first tile, the part that has it
  int t0 = 0, tiles = all;
  if (a.q_parts > 1) {
    t0 = (int)((unsigned)all * blockIdx.y / (unsigned)a.q_parts);
    tiles = (int)((unsigned)all * (blockIdx.y + 1) / (unsigned)a.q_parts);
  }
  const bool writes_delta = exact ? false : one && all > 0 ? t0 == 0 && tiles > 0 : blockIdx.y == 0;
  BiasLoad<T> bias;
  if (BIAS) bias.buckets(a);
  const TileLoad<DP, ROWS> lk(2 * a.ks[1], a.d), lv(2 * a.vs[1], a.d);
  auto load = [&](int t) {
    if constexpr (WIN) {
      const int first = win.tile(t) * ROWS;
      lk.load_window(kbase, 2 * a.ks[1], first, win.end, sk[t & 1], win.low, win.head);
      lv.load_window(vbase, 2 * a.vs[1], first, win.end, sv[t & 1], win.low, win.head);
    } else {
      lk.load(kbase, 2 * a.ks[1], t * ROWS, end, sk[t & 1]);
      lv.load(vbase, 2 * a.vs[1], t * ROWS, end, sv[t & 1]);
    }
  };
  if (t0 < tiles) load(t0);

  // the first loads are all on their way before one is waited for: the keys' and values' tiles,
  // the bias, the rows, and under them shared memory is cleared
  V qf[KS], gf[KS], of[KS];
  const bool in = WIN ? i >= row_first && i < row_end : i >= first_row(a, off) && i < nq;
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
  if (WIN && exact) delta = in ? a.delta[row_at] : 0.f;
  const bool blind = !in || lse == -__builtin_inff();  // a row that sees nothing
  if (blind) lse = kNever;

  f32x16 dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dq[d] = zero16();
  const float c = a.scale * kLog2e;
  Lifted col = {kLift<T>};  // of this column's probabilities and ds
  float left = 0.f;         // sum of ds so far, of which delta's own rounding would leave nothing

  constexpr bool kPlaces = WIN && DP == 128;
  const uint32_t places_of[2] = {kPlaces ? wide_row_place() : 0, kPlaces ? wide_col_place() : 0};
  // the tiles that a row of this wave sees a key of; through the others it only loads its share
  int mine = r0 < nq ? tiles : t0;
  if (!WIN && a.causal) mine = max(t0, min(mine, (r0 + 32 + off + ROWS - 1) / ROWS));
  for (int t = t0; t < mine; ++t) {
    const int buf = t & 1;
    tile_barrier();
    if (t + 1 < tiles) load(t + 1);
    const int tile0 = (WIN ? win.tile(t) : t) * ROWS;
    if (WIN && !window_meets(a, tile0, ROWS, r0 + off, min(r0 + 31, nq - 1) + off)) continue;
    f32x16 ds[KB], p[KB];
    float base[KB];
    const int near0 = tile0 - r0 - off;  // position of the tile's first key and the wave's first row
    V krows[KB][KS], vrows[KB][KS], kcols[KB][2][DB];
    uint32_t row_place = 0, v_place = 0, col_place = 0;
    if constexpr (kPlaces) {
      row_place = lds_address(sk[buf]) + places_of[0], v_place = lds_address(sv[buf]) + places_of[0];
      col_place = lds_address(sk[buf]) + places_of[1];
      asm volatile("" : "+v"(row_place), "+v"(v_place), "+v"(col_place));
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) krows[kb][s] = kPlaces ? wide_row_frag<T>(row_place, s) : row_frag<T, DP>(sk[buf], kb * 32, s);
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
        for (int kb = 0; kb < KB; ++kb) vrows[kb][s] = kPlaces ? wide_row_frag<T>(v_place, s) : row_frag<T, DP>(sv[buf], kb * 32, s);
    };
    auto read_kcols = [&]() {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int d = 0; d < DB; ++d)
            kcols[kb][s][d] = kPlaces ? wide_col_frag<T>(col_place, 16 * s, d * 32) : col_frag<T, DP>(sk[buf], kb * 32 + 16 * s, d * 32);
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
    for (int kb = 0; kb < KB; ++kb) ds[kb] = splat16(WIN && narrow ? 0.f : -delta);
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
      const int j0 = tile0 + kb * 32;
#pragma unroll
      for (int e = 0; e < 16; ++e) p[kb][e] = __builtin_amdgcn_exp2f(fmaf(p[kb][e], c, base[kb]));
      if constexpr (WIN) {
        const int near = near0 + kb * 32;
        if (j0 + 32 > nk || near + 31 > a.after || near < 31 - a.before)
          WindowMask(a, nk, i + off, j0 + 8 * g).apply(p[kb], 0, j0 < a.sinks, 0.f);
      } else if (j0 + 32 > nk || (a.causal && near0 + kb * 32 + 31 > 0)) {
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
    if (WIN && narrow) {  // (delta is of these very sums: subtracted as they stand)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[kb][e] -= delta;
    }
    if constexpr (WIN) {  // past both branches: the compiler leaves an 8-pass product 11 wait states, which takes 12
      asm volatile("s_nop 0");
      keep_order();
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
      if constexpr (WIN && !BIAS) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) s += ds[kb][e];
        left = kLift<T> == 0 ? left + s : fmaf(s, col.unit, left);
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
        if constexpr (WIN) {
          const V rest = pack8_rest<T>(ds[kb], s, df);
#pragma unroll
          for (int d = 0; d < DB; ++d) dq[d] = Frag<T>::mfma(kcols[kb][s][d], rest, dq[d]);
        }
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
  // ds sums to 0 over a row's keys: what is left is delta's error, from the rounded `out`, times the probabilities'
  // sum of 1, and dk and dv are made without it (unless a NaN that other rows see is in it)
  if (WIN && !BIAS && !exact && !one && a.q_parts == 1) {
    left = halves_sum(left) * kUnlift<T>;
    delta += fabsf(left) < kNever ? left : 0.f;
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

// dk and dv of the first keys, which rows see from anywhere: 32 keys as columns, each wave walking row tiles of
// its own (32 rows, of all heads that share the key head, one after the other) through a buffer of its own, with
// no barrier; a tile's operands are in registers before the next one's loads go into its place, under the
// products.  The waves' sums are joined at the end; parts of the rows by attn_join_sinks_kernel.  Workgroup
// `id` of these is one of the kv kernel's launch, whose others hide its waits: its kernel of its own took 20 us of
// 8 sequences of up to 2048, 12 heads of 64, and as many of 8192 rows, 16 heads on 4 of 128.
// tq, tg: four tiles of 32 rows of q and of dout; slse, sdelta: of 32 values.
template <class T, int DP, bool BIAS, bool REST>
__device__ __forceinline__ void sink_gradients(const AttnArgs& a, int id, unsigned char* tq, unsigned char* tg, float* slse, float* sdelta) {
  typedef typename Frag<T>::V V;
  constexpr int KS = DP / 16, DB = DP / 32, TILE = 32 * DP * 2;
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kheads = a.batch * a.k_heads, group = a.heads / a.k_heads;
  const int bk = id % kheads, part = id / kheads % a.sink_parts, j0 = id / kheads / a.sink_parts * 32;
  const int b = bk / a.k_heads, hk = bk % a.k_heads;
  const int nk = key_count(a, b), nq = query_count(a, b), off = query_offset(a, b);
  const int j = j0 + l32;
  int row0, row1;
  window_rows(a, nk, nq, off, row0, row1);
  const int heads_seen = min(a.sinks, a.causal ? min(nk, max(row1 + off, 0)) : nk);  // keys of these that some row sees
  const bool seen = row0 < row1 && j < heads_seen;
  const unsigned char* krow = (const unsigned char*)a.k + 2 * (b * a.ks[0] + j * a.ks[1] + hk * a.ks[2]);
  const unsigned char* vrow = (const unsigned char*)a.v + 2 * (b * a.vs[0] + j * a.vs[1] + hk * a.vs[2]);
  unsigned char *sq = tq + wave * TILE, *sg = tg + wave * TILE;
  slse += wave * 32, sdelta += wave * 32;

  // row tiles of all heads in a row (fewer than 2^31: their results lie in memory); this part's, of which each wave takes every fourth
  const int t0 = (a.causal ? max(row0, j0 - off) : row0) / 32;
  const unsigned nt = row0 < row1 && j0 < heads_seen ? max((row1 + 31) / 32 - t0, 0) : 0;
  const unsigned all = nt * group, f0 = (uint64_t)all * part / a.sink_parts, f1 = (uint64_t)all * (part + 1) / a.sink_parts;
  const TileLoad<DP, 32, 1> lq(2 * a.qs[1], a.d), lg(2 * a.dos[1], a.d);
  float stat = 0.f;  // lanes 0 .. 31: -log2 sum of a row, the others: -delta
  auto load = [&](unsigned f) {
    const int h = hk * group + f / nt, t = t0 + f % nt;
    lq.load((const unsigned char*)a.q + 2 * (b * a.qs[0] + h * a.qs[2]), 2 * a.qs[1], t * 32, row1, sq, row0);
    lg.load((const unsigned char*)a.dout + 2 * (b * a.dos[0] + h * a.dos[2]), 2 * a.dos[1], t * 32, row1, sg, row0);
    const int i = t * 32 + l32;
    const int64_t at = ((int64_t)b * a.heads + h) * a.lq + i;
    const bool in = i >= row0 && i < row1;
    if (g == 0) {
      stat = in ? -a.lse[at] * kLog2e : -kNever;
      if (stat == __builtin_inff()) stat = -kNever;  // a row that sees nothing
    } else {
      stat = in ? -a.delta[at] : 0.f;
    }
  };
  unsigned f = f0 + wave;
  if (f < f1) load(f);
  V kf[KS], vf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    kf[s] = global_frag<T>(krow, s, a.d, seen);
    vf[s] = global_frag<T>(vrow, s, a.d, seen);
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dk[d] = dv[d] = zero16();
  const float c = a.scale * kLog2e;
  float shrink = 1.f;  // of ds, where they would not fit (as the other keys')
  if constexpr (kLift<T> != 0) {
    const int64_t count = (int64_t)group * a.q_parts * ((a.lq + kAttnRows - 1) / kAttnRows);
    const float* from = a.part_peak + bk * count;
    float peak = 0.f;
    for (int64_t t = lane; t < count; t += 64) peak = fmaxf(peak, from[t]);
    shrink = ldexpf(1.f, -max(__builtin_amdgcn_readfirstlane(kLift<T> - room(wave_max(peak))), 0));
  }
  for (; f < f1; f += 4) {
    wait_vmcnt_lgkm0<0>();
    asm volatile("" ::: "memory");
    (g == 0 ? slse : sdelta)[l32] = g == 0 ? stat + kLift<T> : stat;
    const int h = hk * group + f / nt, i0 = (t0 + f % nt) * 32;
    const int near = j0 - i0 - off;
    V qrows[KS], grows[KS], qcols[2][DB], gcols[2][DB];
#pragma unroll
    for (int s = 0; s < KS; ++s) qrows[s] = row_frag<T, DP>(sq, 0, s), grows[s] = row_frag<T, DP>(sg, 0, s);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int d = 0; d < DB; ++d) qcols[s][d] = col_frag<T, DP>(sq, 16 * s, d * 32), gcols[s][d] = col_frag<T, DP>(sg, 16 * s, d * 32);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    f32x16 lse, delta;
#pragma unroll
    for (int e = 0; e < 16; ++e) lse[e] = slse[elem_row(e, g)], delta[e] = sdelta[elem_row(e, g)];
    wait_vmcnt_lgkm0<63>();  // every read of the buffers
    asm volatile("" ::: "memory");
    keep_order();
    if (f + 4 < f1) load(f + 4);
    f32x16 p = zero16(), ds = zero16();  // (delta may be made of dout . v's own sums: subtracted as they stand)
    float shift = 0.f;
    if (BIAS) {
      const float unit = 1.f / a.scale;
      const T* table = (const T*)a.table + h;
      auto bias = [&](int rel) {
        int u = a.bucket_of[min(abs(rel), a.far)];
        if (rel > 0) u = a.causal ? 0 : u + a.one_way;
        return (float)table[(int64_t)u * a.heads] * unit;
      };
      if (near - 31 >= a.far || near + 31 <= -a.far) {
        shift = bias(near) * c;
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = bias(near + l32 - elem_row(e, g));
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) p = Frag<T>::mfma(qrows[s], kf[s], p);
#pragma unroll
    for (int s = 0; s < KS; ++s) ds = Frag<T>::mfma(grows[s], vf[s], ds);
#pragma unroll
    for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(p[e], c, lse[e] + shift));
    if (a.causal && near + 31 > 0) {
      const int first = j - off - i0 - 8 * g;  // first row of the block that sees the key
#pragma unroll
      for (int e = 0; e < 16; ++e) p[e] = elem_row(e, 0) < first ? 0.f : p[e];
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) ds[e] = (ds[e] + delta[e]) * p[e];
    if (kLift<T> != 0 && shrink != 1.f) times<1>(&ds, shrink);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const V pf = pack8<T>(p, s), df = pack8<T>(ds, s);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        dv[d] = Frag<T>::mfma(gcols[s][d], pf, dv[d]);
        dk[d] = Frag<T>::mfma(qcols[s][d], df, dk[d]);
      }
      if constexpr (REST) {
        const V pr = pack8_rest<T>(p, s, pf), dr = pack8_rest<T>(ds, s, df);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          dv[d] = Frag<T>::mfma(gcols[s][d], pr, dv[d]);
          dk[d] = Frag<T>::mfma(qcols[s][d], dr, dk[d]);
        }
      }
    }
  }
  // join the waves: dk, then dv, each wave's [32 columns][DP] in the place of two tiles, the pieces of 4 in an order by column
  wait_vmcnt_lgkm0<0>();
  auto sums_of = [&](int w) { return reinterpret_cast<float*>((w < 2 ? tq : tg) + (w & 1) * 2 * TILE); };
  const int64_t plane = (int64_t)a.batch * a.sinks * a.k_heads * a.d;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float* sums = sums_of(wave);
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16& acc = u == 0 ? dk[d] : dv[d];
        const int piece = (d * 32 + 16 * (q >> 1) + 8 * g + 4 * (q & 1)) / 4;
        *reinterpret_cast<f32x4*>(sums + l32 * DP + ((piece ^ (l32 & 7)) * 4)) =
            f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
      }
    __syncthreads();
    const float undo = u == 0 ? kUnlift<T> / shrink : kUnlift<T>;
    for (int t = threadIdx.x; t < 32 * (DP / 8); t += kBlock) {
      const int col = t / (DP / 8), c8 = t % (DP / 8) * 8;
      if (c8 >= a.d || j0 + col >= a.sinks) continue;
      float z[8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w)
          s += *reinterpret_cast<const f32x4*>(sums_of(w) + col * DP + (((c8 / 4 + half) ^ (col & 7)) * 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) z[4 * half + e] = j0 + col < heads_seen ? s[e] * undo : 0.f;
      }
      if (a.sink_parts > 1) {
        float* o = a.part_sinks + (2 * part + u) * plane + (((int64_t)b * a.sinks + j0 + col) * a.k_heads + hk) * a.d + c8;
        *reinterpret_cast<f32x4*>(o) = f32x4{z[0], z[1], z[2], z[3]};
        *reinterpret_cast<f32x4*>(o + 4) = f32x4{z[4], z[5], z[6], z[7]};
      } else {
        V v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T)(u == 0 ? z[e] * a.scale : z[e]);
        *reinterpret_cast<V*>((T*)(u == 0 ? a.dk : a.dv) + (((int64_t)b * a.lk + j0 + col) * a.k_heads + hk) * a.d + c8) = v;
      }
    }
  }
}

// dk and dv of 128 keys (wave w: 32 of them as columns), over a part of the queries that see
// them.  Where there is a bias, the workgroups from `key_wgs` on add up its table's gradient.
// The keys' rows of both operands and both sums stay in registers, at width 128 some 420 of them:
// one wave a SIMD then, whose products (37% of the time), exponentials and packing follow one
// another.  2 x 4096, 16 heads on 4 of 128, causal: 329 us, 0.84 PFLOP/s of its four products;
// 64 x 512, 12 heads of 64, two workgroups a CU: 148 us, with a bias 156.
// Of a window blocks of 32 rows that see none of a wave's keys are passed over; 8 x up to 2048, 12 heads of 64, window
// 128, bias: 59 us, 8192 rows, 16 heads on 4 of 128, window 1024: 208 us, 0.62 PFLOP/s.  REST, few rows: both halves of
// p and ds (a branch instead of the parameter spilled 49 registers at width 128).
template <class T, int DP, bool BIAS, bool WIN, bool REST>
__global__ __launch_bounds__(kBlock, DP > 64 ? 1 : 2) void attn_backward_kv_kernel(AttnArgs a, int key_wgs, int sink_wgs) {
  typedef typename Frag<T>::V V;
  constexpr int KS = DP / 16, DB = DP / 32, ROWS = 64, QB = ROWS / 32, TILE = ROWS * DP * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char sq[2][TILE], sg[2][TILE];
  __shared__ __attribute__((aligned(16))) float slse[2][ROWS], sdelta[2][ROWS];  // kLift - log2 sums, -deltas
  extern __shared__ float tab[];

  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if constexpr (WIN) {  // (after the others, whose CUs are free at different times)
    if ((int)blockIdx.x >= key_wgs && (int)blockIdx.x < key_wgs + sink_wgs) {
      if (blockIdx.y == 0) sink_gradients<T, DP, BIAS, REST>(a, (int)blockIdx.x - key_wgs, sq[0], sg[0], slse[0], sdelta[0]);
      return;
    }
  }
  if (BIAS && (int)blockIdx.x >= key_wgs) {
    if (blockIdx.y == 0) add_table<T>(a, ((int)blockIdx.x - key_wgs - (WIN ? sink_wgs : 0)) * 4 + wave);
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
  int row0 = min(first_row(a, off), nq), row1 = nq, seen_keys = seen_count(a, nk, nq, off);  // rows that see a key, keys that are seen
  if constexpr (WIN) {
    window_rows(a, nk, nq, off, row0, row1);
    seen_keys = row1 > row0 ? min(nk, max(row1 - 1 + off + a.after + 1, 0)) : 0;  // (by the window; from its first row's on)
  }
  const int seen_low = WIN ? row0 + off - a.before : 0;
  const bool seen = j < seen_keys && (!WIN || j >= seen_low);
  float shrink = 1.f;  // of this workgroup's ds, where they would not fit
  V kf[KS], vf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    kf[s] = global_frag<T>(krow, s, a.d, seen);
    vf[s] = global_frag<T>(vrow, s, a.d, seen);
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dk[d] = dv[d] = zero16();
  const float c = a.scale * kLog2e;
  const int reach = a.far + kReach;
  // delta is made of dout . v's own sums: subtracted as they stand, so that one key leaves 0
  const bool one = nk <= ROWS || (WIN && window_narrow(a));

  // tiles of queries that see a key of this workgroup, those of all heads in a row; this part's
  int t0 = (a.causal ? max(block * kAttnRows - off, 0) : 0) / ROWS;
  int nt = block * kAttnRows < seen_keys ? max((nq + ROWS - 1) / ROWS - t0, 0) : 0;
  if constexpr (WIN) {  // (the first keys' gradients are sink_gradients')
    const int lo = max(row0, block * kAttnRows - off - a.after), hi = min(row1, block * kAttnRows + kAttnRows - off + a.before);
    t0 = lo / ROWS;
    nt = block * kAttnRows < seen_keys && block * kAttnRows + kAttnRows > a.sinks && lo < hi ? (hi + ROWS - 1) / ROWS - t0 : 0;
  }
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
      lq.load(qbase, 2 * a.qs[1], t * ROWS, row1, sq[t & 1], row0);
      lg.load(gbase, 2 * a.dos[1], t * ROWS, row1, sg[t & 1], row0);
      const int i = t * ROWS + threadIdx.x % ROWS;
      if (threadIdx.x < ROWS) {
        stat = i >= row0 && i < row1 ? -lse[i] * kLog2e : -kNever;
        if (stat == __builtin_inff()) stat = -kNever;  // a row that sees nothing
      } else if (threadIdx.x < 2 * ROWS) {
        stat = i >= row0 && i < row1 ? -delta[i] : 0.f;
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
    if (!WIN && a.causal) mine = min(last, max(mine, (j0 - off) / ROWS));
    for (int t = first; t < mine; ++t) turn(t);
    for (int t = mine; t < last; ++t) {
      const int buf = t & 1;
      turn(t);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const int i0 = t * ROWS + qb * 32;
        const int near = j0 - i0 - off;
        if (WIN && (near + 31 < -a.before || near - 31 > a.after)) continue;
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
        if constexpr (WIN) {
          if (near + 31 > a.after || near < 31 - a.before) {
            const int low = j - off - a.after - i0 - 8 * g;  // first row of the block that sees the key
            const unsigned span = a.after + a.before;
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = (unsigned)(elem_row(e, 0) - low) <= span ? p[e] : 0.f;
          }
        } else if (a.causal && near + 31 > 0) {
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
          if constexpr (REST) {
            const V pr = pack8_rest<T>(p, s, pf), dr = pack8_rest<T>(ds, s, df);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
              dv[d] = Frag<T>::mfma(gcols[s][d], pr, dv[d]);
              dk[d] = Frag<T>::mfma(qcols[s][d], dr, dk[d]);
            }
          }
        }
      }
    }
  }
  if (j >= a.lk || (WIN && j < a.sinks)) return;
  if (!seen) {
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

// Adds the parts of the first keys' dk and dv: 8 values to 16 lanes, which take every 16th part and add their
// sums in a fixed order (a thread alone waited for 64 parts' loads in turn, 21 us).
template <class T>
__global__ __launch_bounds__(kBlock) void attn_join_sinks_kernel(AttnArgs a) {
  const int64_t row = (int64_t)a.sinks * a.k_heads * a.d, plane = a.batch * row;
  const int64_t at = ((int64_t)blockIdx.x * (kBlock / 16) + threadIdx.x / 16) * 8;
  if (at >= plane) return;
  const int lane = threadIdx.x % 16;
  float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int p = lane; p < a.sink_parts; p += 16) {
    const f32x4* from = reinterpret_cast<const f32x4*>(a.part_sinks + (2 * p + blockIdx.y) * plane + at);
    const f32x4 lo = from[0], hi = from[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] += lo[e], z[4 + e] += hi[e];
  }
#pragma unroll
  for (int s = 8; s > 0; s >>= 1)
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += __shfl_xor(z[e], s);
  if (lane != 0) return;
  const float scale = blockIdx.y == 0 ? a.scale : 1.f;
  typename Frag<T>::V v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (T)(z[e] * scale);
  *reinterpret_cast<typename Frag<T>::V*>((T*)(blockIdx.y == 0 ? a.dk : a.dv) + at / row * a.lk * a.k_heads * a.d + at % row) = v;
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

// Workgroups of dk's and dv's launch: of the keys, of the first keys, and of the table's sums after them.
int64_t key_workgroups(const AttnArgs& a) { return (a.lk + kAttnRows - 1) / kAttnRows * (int64_t)a.batch * a.k_heads; }
int64_t sink_workgroups(const AttnArgs& a) { return ((int64_t)a.sinks + 31) / 32 * a.batch * a.k_heads * a.sink_parts; }

template <class T, int DP, bool BIAS, bool WIN>
hipError_t launch_window(const AttnArgs& a, hipStream_t s) {
  const int64_t qblocks = (a.lq + kAttnRows - 1) / kAttnRows;
  const size_t tab = BIAS ? (2 * (a.far + kReach) + 1) * sizeof(float) : 0;
  // few rows, or dq in parts, none of which has a row's whole sum of ds to correct delta with
  const bool rests = WIN && (few_rows(a) || a.q_parts > 1);
  if (qblocks > 0) {
    const dim3 grid((unsigned)(qblocks * a.batch * a.heads), a.q_parts);
    if constexpr (WIN) {
      if (exact_delta(a, BIAS, a.lk, kTile<DP>))
        hipLaunchKernelGGL((attn_delta_kernel<T, DP, BIAS>), dim3(grid.x), dim3(kBlock), tab, s, a);
    }
    hipLaunchKernelGGL((attn_backward_q_kernel<T, DP, BIAS, WIN>), grid, dim3(kBlock), 5 * tab, s, a);
  }
  const int64_t sink_wgs = WIN ? sink_workgroups(a) : 0, key_wgs = key_workgroups(a), all_wgs = attn_key_workgroups(a);
  if (all_wgs > 0) {
    const dim3 grid((unsigned)all_wgs, a.kv_parts);
    if (rests)
      hipLaunchKernelGGL((attn_backward_kv_kernel<T, DP, BIAS, WIN, WIN>), grid, dim3(kBlock), tab, s, a, (int)key_wgs, (int)sink_wgs);
    else
      hipLaunchKernelGGL((attn_backward_kv_kernel<T, DP, BIAS, WIN, false>), grid, dim3(kBlock), tab, s, a, (int)key_wgs, (int)sink_wgs);
  }
  auto join = [&](const float* part, int parts, int64_t n, int sums, float scale, void* out0, void* out1) {
    const dim3 grid((unsigned)((n / 8 + kBlock - 1) / kBlock), sums);
    hipLaunchKernelGGL(attn_join_grads_kernel<T>, grid, dim3(kBlock), 0, s, part, parts, sums * n, n, scale, (T*)out0, (T*)out1);
  };
  if (a.q_parts > 1) join(a.part_q, a.q_parts, (int64_t)a.batch * a.lq * a.heads * a.d, 1, a.scale, a.dq, nullptr);
  if (a.kv_parts > 1) join(a.part_kv, a.kv_parts, (int64_t)a.batch * a.lk * a.k_heads * a.d, 2, a.scale, a.dk, a.dv);
  if (WIN && a.sink_parts > 1) {  // (after the join, which writes the first keys' places too)
    const int64_t plane = (int64_t)a.batch * a.sinks * a.k_heads * a.d;
    hipLaunchKernelGGL(attn_join_sinks_kernel<T>, dim3((unsigned)((plane / 8 + 15) / 16), 2), dim3(kBlock), 0, s, a);
  }
  return hipGetLastError();
}

template <class T, int DP, bool BIAS>
hipError_t launch_width(const AttnArgs& a, hipStream_t s) {
  return a.windowed ? launch_window<T, DP, BIAS, true>(a, s) : launch_window<T, DP, BIAS, false>(a, s);
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
  if (window_narrow(a)) return 1;
  int64_t keys = a.lk;  // that a workgroup walks
  if (a.windowed) keys = std::min(keys, (int64_t)a.sinks + a.before + a.after + std::min(a.lq, kAttnRows));
  return (int)std::max<int64_t>(1, std::min<int64_t>({2 * cus / wgs, keys / 512, (int64_t)64}));
}
int attn_kv_parts(const AttnArgs& a, int cus) {
  const int64_t wgs = (a.lk + kAttnRows - 1) / kAttnRows * (int64_t)a.batch * a.k_heads;
  int64_t rows = a.lq;  // that a workgroup walks of each head
  if (a.windowed) rows = std::min(rows, (int64_t)a.before + a.after + kAttnRows);
  const int64_t tiles = (rows + 63) / 64 * (int64_t)(a.heads / a.k_heads);
  // (one workgroup a CU, and all of them walk as many rows: 8192 rows, 16 heads on 4 of 128, the pass 352 us, 373 for two)
  if (a.windowed && a.d > 64) cus /= 2;
  return (int)std::max<int64_t>(1, std::min<int64_t>({2 * cus / wgs, tiles / 8, (int64_t)16}));
}

// Parts of the rows for the first keys' dk and dv, of at least 16 tiles of 32 rows, 4 a wave, so that these workgroups
// take no longer than the other keys' (8 x 2048, 12 heads of 64, 1 key: the pass 148 us, of 4 tiles 154, of 64 157; 8192
// rows, 16 heads on 4 of 128, 4 keys: 353, 355 and 366).  (Where there are parts of the others' rows too, their join
// overwrites what a single part writes: two at least.)
int attn_sink_parts(const AttnArgs& a, int kv_parts, int cus) {
  const int64_t wgs = (a.sinks + 31) / 32 * (int64_t)a.batch * a.k_heads;
  const int64_t tiles = (a.lq + 31) / 32 * (int64_t)(a.heads / a.k_heads);
  return (int)std::max<int64_t>(kv_parts > 1 ? 2 : 1, std::min<int64_t>({tiles / 16, 8 * cus / wgs, (int64_t)64}));
}

int64_t attn_key_workgroups(const AttnArgs& a) {
  return key_workgroups(a) + sink_workgroups(a) + (a.table != nullptr ? (a.buckets * a.heads + 3) / 4 : 0);
}

hipError_t launch_attn_backward(const AttnArgs& a, hipStream_t s) {
  return a.type == kF16 ? backward<_Float16>(a, s) : backward<__bf16>(a, s);
}

}  // namespace cvs
