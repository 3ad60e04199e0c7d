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
// A row that sees no key gets zeros, and -inf as its log sum.  Keys past the last one that a
// workgroup's rows see are not read (a cache's places not yet written), nor, with a window, those before the first
// one and after the first keys; a value that is not finite, of a key that some row of the workgroup sees, does
// reach its other rows, the earlier ones and those whose window has moved past the key, as 0 times it.
#include <algorithm>

#include "cvs_attn_tile.h"

namespace cvs {

namespace {

constexpr int kKeys = 64;  // keys of a tile

// Two LDS buffers of 64 keys and values, two or three workgroups a CU (which fill each other's
// exponentials and waits with products), queries and sums in registers.  Bound by the vector
// instructions between the products: 2 x 8192, 12 heads of 64, 469 us, 0.88 PFLOP/s; 2 x 4096, 16 heads
// of 128, 270 us, 1.02; at short sequences by a workgroup's start and end (64 x up to 512, 12 heads
// of 64, bias: 57 us).  With a window a workgroup walks the first keys' tiles and its rows' own: 8192 rows, 12 heads of 64,
// window 128, 4 first keys 23 us, five to seven tiles a workgroup: some 9 of start and end (windows of 0 to 1024 keys to either
// side, 13.5 to 86 us, are a line of 2.05 us a tile), under which nothing of another workgroup runs, all 768 having started at once.
template <class T, int DP, bool BIAS, bool WIN>
__global__ __launch_bounds__(kBlock, DP > 64 ? 2 : 3) void attn_forward_kernel(AttnArgs a) {
  typedef typename Frag<T>::V V;
  constexpr int KS = DP / 16, DB = DP / 32, TILE = kKeys * DP * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char sk[2][TILE], sv[2][TILE];
  extern __shared__ float tab[];

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
  const unsigned char* kbase = (const unsigned char*)a.k + 2 * (b * a.ks[0] + hk * a.ks[2]);
  const unsigned char* vbase = (const unsigned char*)a.v + 2 * (b * a.vs[0] + hk * a.vs[2]);

  // this workgroup's keys: a part of those that some row of it sees
  const int last_row = min(block * kAttnRows + kAttnRows, nq) - 1;
  int end = last_row < block * kAttnRows ? 0 : nk;
  if (a.causal) end = min(end, max(last_row + off + 1, 0));
  int tiles = (end + kKeys - 1) / kKeys;
  WindowTiles<kKeys> win;
  if constexpr (WIN) {
    win = WindowTiles<kKeys>(a, nk, block * kAttnRows + off, last_row + off);
    tiles = win.count;
  }
  int t0 = 0, t1 = tiles;
  if (a.splits > 1) {  // (fewer than 2^23 tiles, at most 64 parts)
    t0 = (int)((unsigned)tiles * blockIdx.y / (unsigned)a.splits);
    t1 = (int)((unsigned)tiles * (blockIdx.y + 1) / (unsigned)a.splits);
  }

  BiasLoad<T> bias;
  if (BIAS) bias.buckets(a);
  const TileLoad<DP, kKeys> lk(2 * a.ks[1], a.d), lv(2 * a.vs[1], a.d);
  auto load = [&](int t) {
    if constexpr (WIN) {
      const int first = win.tile(t) * kKeys;
      lk.load_window(kbase, 2 * a.ks[1], first, win.end, sk[t & 1], win.low, win.head);
      lv.load_window(vbase, 2 * a.vs[1], first, win.end, sv[t & 1], win.low, win.head);
    } else {
      lk.load(kbase, 2 * a.ks[1], t * kKeys, end, sk[t & 1]);
      lv.load(vbase, 2 * a.vs[1], t * kKeys, end, sv[t & 1]);
    }
  };
  if (t0 < t1) load(t0);
  V qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = global_frag<T>(qrow, s, a.d, i < nq);
  if (BIAS) {
    bias.values(a, h);
    bias.store(a, tab);
  }

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = zero16();
  // m: what the row's exponentials are relative to, in units of unscaled scores.  It follows
  // the maximum only once that is 2^8 past it: rescaling the sums is then rare, and
  // exponentials up to 2^8 lose nothing.
  float m = -__builtin_inff(), sum = 0.f;
  const float c = a.scale * kLog2e, slack = 8.f / c;

  // the tiles that a row of this wave sees a key of; through the others it only loads its share
  int mine = r0 < nq ? t1 : t0;
  if (!WIN && a.causal) mine = max(t0, min(mine, (r0 + 32 + off + kKeys - 1) / kKeys));
  for (int t = t0; t < mine; ++t) {
    const int buf = t & 1;
    tile_barrier();
    if (t + 1 < t1) load(t + 1);
    const int j0 = (WIN ? win.tile(t) : t) * kKeys;
    if (WIN && !window_meets(a, j0, kKeys, r0 + off, min(r0 + 31, nq - 1) + off)) continue;
    const int near = j0 - r0 - off;  // position of the tile's first key and the wave's first row
    V rows[2][KS];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) rows[kb][s] = row_frag<T, DP>(sk[buf], kb * 32, s);
    f32x16 x[2];
    float shift = 0.f;  // a bias that all of the tile has
    auto scores = [&]() {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) x[kb] = Frag<T>::mfma(rows[kb][s], qf[s], x[kb]);
    };
    const int reach = a.far + kReach;
    if (!BIAS || near - 31 >= a.far || near + kKeys - 1 <= -a.far) {
      if (BIAS) shift = tab[near > 0 ? 2 * reach : 0];
      keep_order();
      x[0] = x[1] = zero16();
      scores();
    } else {
      const float* at = tab + (near - l32 + 8 * g + reach);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[kb][e] = at[kb * 32 + elem_row(e, 0)];
      keep_order();
      scores();
    }
    V cols[2][2][DB];
    if constexpr (!WIN) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int d = 0; d < DB; ++d) cols[kb][s][d] = col_frag<T, DP>(sv[buf], kb * 32 + 16 * s, d * 32);
    }
    keep_order();
    if constexpr (WIN) {
      if (j0 + kKeys > nk || near + kKeys - 1 > a.after || near < 31 - a.before) {
        const WindowMask mask(a, nk, i + off, j0 + 8 * g);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) mask.apply(x[kb], kb * 32, j0 < a.sinks, -__builtin_inff());
      }
      // (before the mask, under the products, there are not the registers)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int d = 0; d < DB; ++d) cols[kb][s][d] = col_frag<T, DP>(sv[buf], kb * 32 + 16 * s, d * 32);
    } else if (j0 + kKeys > nk || (a.causal && near + kKeys - 1 > 0)) {
      const int seen = min(nk - 1, a.causal ? i + off : nk) - j0 - 8 * g;  // last key of the tile that the row sees
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[kb][e] = kb * 32 + elem_row(e, 0) > seen ? -__builtin_inff() : x[kb][e];
    }
    float top = x[0][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, x[kb][e]);
    top = halves_max(top) + shift;
    if (__any(top > m + slack)) {
      const float next = fmaxf(m, top);
      const float fade = next == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m - next) * c);
      m = next;
      sum *= fade;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] *= fade;
    }
    const float base = m == -__builtin_inff() ? shift * c : (shift - m) * c;  // (no score yet: all of them -inf, or the bias)
    float part[2] = {0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[kb][e] = __builtin_amdgcn_exp2f(fmaf(x[kb][e], c, base));
        part[kb] += x[kb][e];
      }
    sum += part[0] + part[1];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const V p = pack8<T>(x[kb], s);
#pragma unroll
        for (int d = 0; d < DB; ++d)
          acc[d] = Frag<T>::mfma(cols[kb][s][d], p, acc[d]);
      }
  }
  for (int t = max(mine, t0); t < t1; ++t) {
    tile_barrier();
    if (t + 1 < t1) load(t + 1);
  }
  sum = halves_sum(sum);
  if (i >= a.lq) return;
  if (i >= nq) sum = 0.f, m = -__builtin_inff();
  m *= c;  // to base-2 logarithms
  const int64_t at = (int64_t)bh * a.lq + i;  // [batch, heads, lq]
  if (a.splits > 1) {
    const int64_t rows = (int64_t)heads * a.lq;
    if (g == 0) {
      a.part_ml[2 * (blockIdx.y * rows + at)] = m;
      a.part_ml[2 * (blockIdx.y * rows + at) + 1] = sum;
    }
    store_part_row<DP>(a.part_out + (blockIdx.y * rows + at) * a.d, acc, a.d);
    return;
  }
  if (sum == 0.f) {  // (the sums may be NaN: 0 times a value that other rows see)
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = zero16();
  }
  if (a.lse != nullptr && g == 0) a.lse[at] = sum == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(sum)) * kLn2;
  store_head_row<T, DP>((T*)a.out + ((int64_t)(b * (int64_t)a.lq + i) * a.heads + h) * a.d, acc,
                        sum == 0.f ? 0.f : 1.f / sum, a.d);
}

// Few query rows (single tokens, a pooling query) over many keys, bound by reading the keys.
// The rows of the query heads that share a key head (of one head where there is a
// bias) are the columns of one block, at most 32.  Each wave walks key tiles of its own, 32
// keys, through buffers of its own, with no barrier, its next tile's loads under way (64 KiB a
// CU); the waves' sums are joined at the end.  (8 x 12 heads of 64, one row over up to 8191 keys:
// 23 us, 5.4 TB/s of keys and values; 36 us in the kernel above, where three of four waves had no
// rows.  One sequence of 23, 12 heads of 32, with a bias: 5.2 us, the latency of the bias's two
// dependent loads, the keys' tile and a launch.)
template <class T, int DP, bool BIAS, bool WIN>
__global__ __launch_bounds__(kBlock, DP > 64 ? 1 : 2) void attn_rows_kernel(AttnArgs a) {
  typedef typename Frag<T>::V V;
  constexpr int KS = DP / 16, DB = DP / 32, TILE = 32 * DP * 2, LOADS = TILE / 1024;
  // per wave: two tiles of keys and of values; at the end its sums
  __shared__ __attribute__((aligned(1024))) unsigned char smem[4][2][2][TILE];
  __shared__ float stat[4][2][32];
  extern __shared__ float tab[];

  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = a.heads / a.k_heads, gcols = BIAS ? 1 : group;  // query heads of a block
  const int blocks = a.heads / gcols;
  const int b = blockIdx.x / blocks, h0 = blockIdx.x % blocks * gcols, hk = h0 / group;
  const int nk = key_count(a, b), nq = query_count(a, b), off = query_offset(a, b);
  const int i = l32 % a.lq, h = h0 + l32 / a.lq;
  const bool row = l32 < a.lq * gcols;  // this lane's column is a row of a head
  const unsigned char* kbase = (const unsigned char*)a.k + 2 * (b * a.ks[0] + hk * a.ks[2]);
  const unsigned char* vbase = (const unsigned char*)a.v + 2 * (b * a.vs[0] + hk * a.vs[2]);

  int end = nq > 0 ? nk : 0;
  if (a.causal) end = min(end, max(nq + off, 0));
  int tiles = (end + 31) / 32;
  WindowTiles<32> win;
  if constexpr (WIN) {
    win = WindowTiles<32>(a, nk, off, nq - 1 + off);
    tiles = win.count;
  }
  int t0 = 0, t1 = tiles;
  if (a.splits > 1) {
    t0 = (int)((unsigned)tiles * blockIdx.y / (unsigned)a.splits);
    t1 = (int)((unsigned)tiles * (blockIdx.y + 1) / (unsigned)a.splits);
  }
  BiasLoad<T> bias;
  if (BIAS) bias.buckets(a);
  const TileLoad<DP, 32, 1> lk(2 * a.ks[1], a.d), lv(2 * a.vs[1], a.d);
  auto load = [&](int t, int buf) {
    if constexpr (WIN) {
      const int first = win.tile(t) * 32;
      lk.load_window(kbase, 2 * a.ks[1], first, win.end, smem[wave][buf][0], win.low, win.head);
      lv.load_window(vbase, 2 * a.vs[1], first, win.end, smem[wave][buf][1], win.low, win.head);
    } else {
      lk.load(kbase, 2 * a.ks[1], t * 32, end, smem[wave][buf][0]);
      lv.load(vbase, 2 * a.vs[1], t * 32, end, smem[wave][buf][1]);
    }
  };
  int t = t0 + wave, buf = 0;
  if (t < t1) load(t, 0);
  V qf[KS];
  const unsigned char* qrow = (const unsigned char*)a.q + 2 * (b * a.qs[0] + i * a.qs[1] + h * a.qs[2]);
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = global_frag<T>(qrow, s, a.d, row && i < nq);
  if (BIAS) {
    bias.values(a, h0);
    bias.store(a, tab);
    __syncthreads();
  }

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = zero16();
  float m = -__builtin_inff(), sum = 0.f;
  const float c = a.scale * kLog2e, slack = 8.f / c;
  const int reach = a.far + kReach;
  wait_vmcnt_lgkm0<0>();
  for (; t < t1; t += 4, buf ^= 1) {
    wait_vmcnt_lgkm0<63>();  // the reads of the buffer to be loaded next
    asm volatile("" ::: "memory");
    if (t + 4 < t1) {
      load(t + 4, buf ^ 1);
      wait_vmcnt_lgkm0<2 * LOADS>();
    } else {
      wait_vmcnt_lgkm0<0>();
    }
    asm volatile("" ::: "memory");
    const unsigned char* sk = smem[wave][buf][0];
    const unsigned char* sv = smem[wave][buf][1];
    const int j0 = (WIN ? win.tile(t) : t) * 32, near = j0 - off;
    V rows[KS], cols[2][DB];
#pragma unroll
    for (int s = 0; s < KS; ++s) rows[s] = row_frag<T, DP>(sk, 0, s);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int d = 0; d < DB; ++d) cols[s][d] = col_frag<T, DP>(sv, 16 * s, d * 32);
    f32x16 x = zero16();
    float shift = 0.f;
    if (BIAS) {
      if (near - 31 >= a.far || near + 31 <= -a.far) {
        shift = tab[near > 0 ? 2 * reach : 0];
      } else {
        const float* at = tab + (near - l32 + 8 * g + reach);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = at[elem_row(e, 0)];
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) x = Frag<T>::mfma(rows[s], qf[s], x);
    if constexpr (WIN) {
      if (j0 + 32 > nk || near + 31 > a.after || near < nq - 1 - a.before)
        WindowMask(a, nk, i + off, j0 + 8 * g).apply(x, 0, j0 < a.sinks, -__builtin_inff());
    } else if (j0 + 32 > nk || (a.causal && near + 31 > 0)) {
      const int seen = min(nk - 1, a.causal ? i + off : nk) - j0 - 8 * g;
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = elem_row(e, 0) > seen ? -__builtin_inff() : x[e];
    }
    float top = x[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
    top = halves_max(top) + shift;
    if (__any(top > m + slack)) {
      const float next = fmaxf(m, top);
      const float fade = next == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m - next) * c);
      m = next;
      sum *= fade;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] *= fade;
    }
    const float base = m == -__builtin_inff() ? shift * c : (shift - m) * c;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], c, base));
      sum += x[e];
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const V p = pack8<T>(x, s);
#pragma unroll
      for (int d = 0; d < DB; ++d) acc[d] = Frag<T>::mfma(cols[s][d], p, acc[d]);
      if constexpr (WIN) {  // (of one row, p's rounding does not average out; hidden behind the keys' loads)
        const V rest = pack8_rest<T>(x, s, p);
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = Frag<T>::mfma(cols[s][d], rest, acc[d]);
      }
    }
  }
  // join the waves: sums relative to the largest of their m, column by column
  sum = halves_sum(sum);
  if (g == 0) stat[wave][0][l32] = m, stat[wave][1][l32] = sum;
  wait_vmcnt_lgkm0<0>();
  __syncthreads();  // (every wave is done with the tiles, too)
  float top = -__builtin_inff();
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][0][l32]);
  const float base = top == -__builtin_inff() ? 0.f : top;
  const float fade = __builtin_amdgcn_exp2f((m - base) * c);
  float* sums = reinterpret_cast<float*>(smem[wave]);  // [32 columns][DP], the pieces of 4 in an order by column
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int piece = (d * 32 + 16 * (q >> 1) + 8 * g + 4 * (q & 1)) / 4;
      *reinterpret_cast<f32x4*>(sums + l32 * DP + ((piece ^ (l32 & 7)) * 4)) =
          f32x4{acc[d][4 * q], acc[d][4 * q + 1], acc[d][4 * q + 2], acc[d][4 * q + 3]} * fade;
    }
  __syncthreads();
  const int64_t rows = (int64_t)a.batch * a.heads * a.lq;
  for (int u = threadIdx.x; u < a.lq * gcols * (DP / 8); u += kBlock) {
    const int col = u / (DP / 8), c8 = u % (DP / 8) * 8;
    if (c8 >= a.d) continue;
    const int ci = col % a.lq, ch = h0 + col / a.lq;
    const int64_t at = ((int64_t)b * a.heads + ch) * a.lq + ci;
    float ct = -__builtin_inff(), cs = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) ct = fmaxf(ct, stat[w][0][col]);
    const float cb = ct == -__builtin_inff() ? 0.f : ct;
#pragma unroll
    for (int w = 0; w < 4; ++w) cs += stat[w][1][col] * __builtin_amdgcn_exp2f((stat[w][0][col] - cb) * c);
    if (ci >= nq) ct = -__builtin_inff(), cs = 0.f;
    float z[8];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w)
        s += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(smem[w]) + col * DP + (((c8 / 4 + half) ^ (col & 7)) * 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) z[4 * half + e] = s[e];
    }
    if (a.splits > 1) {
      float* o = a.part_out + (blockIdx.y * rows + at) * a.d + c8;
      *reinterpret_cast<f32x4*>(o) = f32x4{z[0], z[1], z[2], z[3]};
      *reinterpret_cast<f32x4*>(o + 4) = f32x4{z[4], z[5], z[6], z[7]};
      if (c8 == 0) {
        a.part_ml[2 * (blockIdx.y * rows + at)] = ct * c;
        a.part_ml[2 * (blockIdx.y * rows + at) + 1] = cs;
      }
    } else {
      const float inv = cs == 0.f ? 0.f : 1.f / cs;
      V v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)(cs == 0.f ? 0.f : z[e] * inv);
      *reinterpret_cast<V*>((T*)a.out + (((int64_t)b * a.lq + ci) * a.heads + ch) * a.d + c8) = v;
      if (c8 == 0 && a.lse != nullptr) a.lse[at] = cs == 0.f ? -__builtin_inff() : (ct * c + __builtin_amdgcn_logf(cs)) * kLn2;
    }
  }
}

// Joins the parts of the keys: one wave a query row (96 rows of 64 in 5 parts: 5 us, latency).
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
    const bool seen = ml[1] != 0.f;  // (where nothing was, the sums may be NaN; a select, so that the loads go together)
    const float f = __builtin_amdgcn_exp2f(ml[0] - base);
    sum = fmaf(f, ml[1], sum);
    if (c < a.d) {
      const float* o = a.part_out + (s * rows + at) * a.d + c;
      o0 = fmaf(f, seen ? o[0] : 0.f, o0);
      o1 = fmaf(f, seen ? o[1] : 0.f, o1);
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

// Whether the rows of a block of heads are few enough for one block's columns.
bool few_rows(const AttnArgs& a) { return (int64_t)a.lq * (a.table != nullptr ? 1 : a.heads / a.k_heads) <= 32; }

int64_t workgroups(const AttnArgs& a) {
  if (few_rows(a)) return (int64_t)a.batch * (a.table != nullptr ? a.heads : a.k_heads);
  return (a.lq + kAttnRows - 1) / kAttnRows * (int64_t)a.batch * a.heads;
}

template <class T, int DP, bool WIN>
void launch_window(const AttnArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)workgroups(a), a.splits), block(kBlock);
  const size_t tab = (2 * (a.far + kReach) + 1) * sizeof(float);
  if (few_rows(a) && a.table != nullptr)
    hipLaunchKernelGGL((attn_rows_kernel<T, DP, true, WIN>), grid, block, tab, s, a);
  else if (few_rows(a))
    hipLaunchKernelGGL((attn_rows_kernel<T, DP, false, WIN>), grid, block, 0, s, a);
  else if (a.table != nullptr)
    hipLaunchKernelGGL((attn_forward_kernel<T, DP, true, WIN>), grid, block, tab, s, a);
  else
    hipLaunchKernelGGL((attn_forward_kernel<T, DP, false, WIN>), grid, block, 0, s, a);
}

template <class T, int DP>
void launch_width(const AttnArgs& a, hipStream_t s) {
  if (a.windowed)
    launch_window<T, DP, true>(a, s);
  else
    launch_window<T, DP, false>(a, s);
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

// Parts of the keys: enough for two workgroups a CU, of at least 4 tiles of 64 (or 4 a wave
// of 32) each.  (128 rows over 8192 keys, 8 heads of 64: 37 us, 100 whole; one row over 8 x
// up to 8191 keys, 12 heads of 64: 23 us and 5 for the join, 40 whole.)
int attn_splits(const AttnArgs& a, int cus) {
  const int64_t least = few_rows(a) ? 4 * 4 * 32 : 4 * kKeys;
  int64_t keys = a.lk;  // that a workgroup walks
  if (a.windowed) keys = std::min(keys, (int64_t)a.sinks + a.before + a.after + std::min(a.lq, kAttnRows));
  return (int)std::max<int64_t>(1, std::min<int64_t>({2 * cus / std::max<int64_t>(workgroups(a), 1), keys / least, (int64_t)64}));
}

hipError_t launch_attn_forward(const AttnArgs& a, hipStream_t s) {
  return a.type == kF16 ? forward<_Float16>(a, s) : forward<__bf16>(a, s);
}

}  // namespace cvs
