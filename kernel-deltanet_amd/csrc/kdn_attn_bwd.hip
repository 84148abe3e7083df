// Causal attention over packed sequences: the backward.
//
//   p_ij = exp(scale q_i.k_j - lse_i),  delta_i = dy_i . y_i,  ds_ij = p_ij (dy_i.v_j - delta_i),
//   dv_j = sum_i p_ij dy_i,  dk_j = scale sum_i ds_ij q_i,  dq_i = scale sum_j ds_ij k_j,
// with the sums over i of a key head running over all query heads that share it.
//
// Delta first; then dk and dv, a workgroup per 128 keys of a key head walking the query rows that see them, and dq, a
// workgroup per 128 query rows of a head walking its keys.  The scores are formed twice (seven products for the five that
// one pass with atomic sums of dq would take; eight with 128 features, see Dkdv): every sum then has one owner and one order,
// so that the gradients are the same bits every time.  As in the forward a product's accumulator is the next one's B
// operand in registers: in bf16 p and ds are rounded to its eight bits there, and dq and dk come 1.40 to 1.46 times as far from 64 bits
// as sums in fp32 of unrounded ones, rounded once, do; in two parts each, three of the eight products would be six.
//   What bounds it: as in the forward, products and exponentials that overlap in part.  One sequence of 8192 rows, 32 heads
// of 128 over 8, bf16: the forward 0.56 ms, the gradients 2.1 to 2.4 (2.20 TFLOP in eight products: 0.9 to 1.0 PFLOP/s; five of
// them, those that the formulas need, 0.6), at 1.7 to 1.9 GHz.  fp32, 4096 rows, 32 heads of 128: 5.0 ms, matrix cores busy 71 %
// at 2.2 GHz.
#include <algorithm>
#include "kdn_attn_tile.hpp"
#include "kdn_io.hpp"

namespace kdn {

// Minus delta, and minus lse / scale: what dkdv's products start from.  Sixteen lanes a row, eight values each; 8192 rows of
// 32 heads, 128 features, bf16: 35 us, 5.7 TB/s of y, its low part and dy.
template <class P>
__global__ void __launch_bounds__(256) attn_delta_kernel(AttnParams p, float* stat, float* delta, int64_t first) {
  typedef typename P::elem E;
  const int64_t at = first + (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);  // (row, head), heads fastest
  const int j = threadIdx.x & 15;
  if (at >= p.total_q * p.H) return;
  const int64_t row = at / p.H, h = at % p.H;
  const E* y = reinterpret_cast<const E*>(p.y) + row * p.ys[0] + h * p.ys[1];
  const E* dy = reinterpret_cast<const E*>(p.dy) + row * p.dys[0] + h * p.dys[1];
  float sum = 0.f;
  if (8 * j < P::D) {
    const typename P::frag a = P::load(y + 8 * j), b = P::load(dy + 8 * j);
    float x[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) x[s] = (float)a[s];
    if (sizeof(E) == 2 && p.low) {
      const typename P::frag rest = P::load(reinterpret_cast<const E*>(p.low) + row * p.lows[0] + h * p.lows[1] + 8 * j);
#pragma unroll
      for (int s = 0; s < 8; ++s) x[s] += (float)rest[s];
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) sum = __builtin_fmaf(x[s], (float)b[s], sum);
  }
  sum += xor_shuffle<1>(sum);
  sum += xor_shuffle<2>(sum);
  sum += xor_shuffle<4>(sum);
  sum += xor_shuffle<8>(sum);
  if (j == 0) {
    delta[h * p.total_q + row] = -sum;
    stat[h * p.total_q + row] = -p.lse[h * p.total_q + row] / p.scale;
  }
}

// The launch's first argument, read anew: what a part of attn_grads_kernel does not use is not loaded before it (with all of it
// in scalar registers from the start, 30 to 70 of them spilled).
__device__ __forceinline__ const AttnParams& params_here() {
  typedef const __attribute__((address_space(4))) AttnParams* Args;
  Args a = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return *(const AttnParams*)a;
}

// Under a window (WIN) the rows that see a tile of keys end `window` behind it, but for the first `sinks` keys, which all later
// rows see: one workgroup that walked them all would run on when the others are done (a sequence of 65536 rows and a window of
// 1024: fifty times as long).  So those rows are cut into segments of FAR_ROWS, a workgroup each and 32 sinks, whose waves share the
// rows (one wave with all of them: the gradients of 16384 rows in a window of 1024, four sinks, 32 heads of 128 over 8, bf16, 1 % more).  Their sums of the sinks' dk and dv come to lie apart in fp32, as the near rows' do a second time; attn_sinks_kernel adds them
// in a fixed order.
//   Of their 1430 to 1500 us by card dv takes a quarter, dk and dq a third each, the far rows a twentieth; matrix cores busy 39 %, at 2.0 GHz.  With the
// products that the formulas need, 0.45 to 0.47 PFLOP/s: eight are formed for five, and a tile of 128 keys walks 1152 rows for 1024.
constexpr int FAR_ROWS = 1024;
constexpr int FAR_SINKS = 256;  // with more, their tiles are many themselves, and walked by one workgroup each: no segments
// The query rows [from, to) of a sequence that see keys of the tile row0 .. row0 + keys - 1 for nearness, in whole tiles of `rows`.
// Those from `to` on see of it the sinks alone.
struct NearRows {
  int from, to;
  __device__ __forceinline__ NearRows(int row0, int off, int lenq, int window, int keys, int rows) {
    from = max(row0 - off, 0) / rows * rows;
    const int end = min(lenq, max(row0 + keys - 1 - off + window, 0));
    to = from < end ? from + (end - from + rows - 1) / rows * rows : from;
  }
};

// dk and dv of 128 / SPLIT keys: a wave owns 32 keys (a lane one), their K and V fragments and the transposed sums in
// registers.  The query rows pass in tiles with their lse and delta; S = Q K^T and dP = dY V^T have the queries in
// registers, so that P and dS are the B operands of dV^T += dY^T P and dK^T += Q^T dS.
//   With 128 features both sums and the operands do not fit the registers of two waves a SIMD, and one wave, whose softmax
// nothing overlaps, takes 2.13 ms at 8192 rows, 32 heads, where dv and dk apart (DV, DK), S formed in both, take 1.79.
template <class P, int SPLIT>
struct Dkdv {
  static constexpr int KEYS = 128 / SPLIT, ROWS = SPLIT == 4 ? 128 : 64, BLOCKS = ROWS / 32 / SPLIT;
  static constexpr int TILE = ROWS * P::ROW, SLOT = 2 * TILE + 2 * ROWS * 4, BUFS = 2 * SLOT <= 160 * 1024 ? 2 : 1;
  static constexpr int JOIN = 4 * (P::D / 32) * 4096;
  static constexpr int LDS = BUFS * SLOT > JOIN ? BUFS * SLOT : JOIN;
};

template <class P, int SPLIT, bool DV, bool DK, bool WIN>
__device__ __forceinline__ void dkdv(int id, int slots, int far, unsigned char* lds) {
  const AttnParams& p = params_here();
  typedef typename P::elem E;
  typedef Dkdv<P, SPLIT> S;
  constexpr int KS = P::D / 16, CT = P::D / 32, TILE = S::TILE, ROWS = S::ROWS;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = w % SPLIT;
  const int e = id % p.KV, sub = id / p.KV % p.subsets, heads = p.G / p.subsets;
  SeqTile t;  // the keys' tile
  int64_t qlo;
  int lenq, far_slot = -1, segment = 0;
  if (WIN && id < far) {
    const int tiles = (p.sinks + 31) / 32, u = id / p.KV / p.subsets;
    far_slot = u / tiles;
    const SeqTile rows = find_tile<FAR_ROWS>(p.cu_q, p.nseq, p.total_q, far_slot, lane);
    if (rows.row0 < 0) return;
    qlo = rows.lo, lenq = rows.len, segment = rows.row0;
    t.row0 = u % tiles * 32;
    other_rows(p.cu_k, p.nseq, p.total_k, rows.seq, t.lo, t.len);
    if (t.row0 >= t.len) return;
  } else {
    t = find_heavy<S::KEYS, true>(p.cu_k, p.nseq, p.total_k, (WIN ? id - far : id) / p.KV / p.subsets, slots, lane);
    if (t.row0 < 0) return;
    other_rows(p.cu_q, p.nseq, p.total_q, t.seq, qlo, lenq);
  }
  const int lenk = t.len;
  const int off = lenk - lenq;
  const bool is_far = WIN && far_slot >= 0;
  const int first_key = t.row0 + (is_far ? 0 : 32 * (w / SPLIT)), key = first_key + (lane & 31);
  const bool live = key < lenk;
  typename P::frag k[KS], v[DK ? KS : 1];
  {
    const int64_t at = t.lo + min(key, lenk - 1);
    const E* ksrc = reinterpret_cast<const E*>(p.k) + at * p.ks[0] + (int64_t)e * p.ks[1];
    const E* vsrc = reinterpret_cast<const E*>(p.v) + at * p.vs[0] + (int64_t)e * p.vs[1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      k[ks] = P::load(ksrc + 16 * ks + 8 * half);
      if constexpr (DK) v[ks] = P::load(vsrc + 16 * ks + 8 * half);
    }
  }
  f32x16 dk[DK ? CT : 1], dv[DV ? CT : 1];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if constexpr (DK) dk[ct] = zero16();
    if constexpr (DV) dv[ct] = zero16();
  }
  const float c = p.scale * LOG2E;

  // the query tiles that see key row0: rows from row0 - off on, of each head of the subset
  int q0 = max(t.row0 - off, 0) / ROWS * ROWS, q1 = lenq;
  if constexpr (WIN) {
    const NearRows near(t.row0 / S::KEYS * S::KEYS, off, lenq, p.window, S::KEYS, ROWS);
    if (p.far_slots > 0 || t.row0 >= p.sinks) q1 = min(near.to, lenq);
    if (is_far) {
      q0 = max(near.to, segment);
      q1 = min(lenq, segment + FAR_ROWS);
      if (q0 >= q1) return;
    }
  }
  const int per = q0 < q1 ? (q1 - q0 + ROWS - 1) / ROWS : 0;
  const int ntiles = per * heads;
  // the end of the rows that see the lane's key; from which first row on a block of 32 is past some of the wave's keys, and past all
  const int last_row = !WIN || key < p.sinks ? lenq : min(lenq, key - off + p.window);
  const int cut_from = WIN && first_key + 31 >= p.sinks ? first_key - 31 - off + p.window : INT32_MAX;
  const int hidden_from = WIN && first_key >= p.sinks ? first_key + 31 - off + p.window : INT32_MAX;
  const Stager<P, ROWS, 4> stage_q(p.qs[0], w, lane), stage_y(p.dys[0], w, lane);
  const AttnParams& first = p;
  auto stage = [&](int j, unsigned char* to) {
    // at 128 features two waves a row and a window: read where they are used, or scalar registers are spilled to memory
    const AttnParams& p = WIN && P::D == 128 && SPLIT == 2 ? params_here() : first;
    const int h = e * p.G + sub * heads + j / per, r0 = q0 + j % per * ROWS, last = min(lenq - 1 - r0, ROWS - 1);
    stage_q(reinterpret_cast<const E*>(p.q) + (qlo + r0) * p.qs[0] + (int64_t)h * p.qs[1], last, to);
    stage_y(reinterpret_cast<const E*>(p.dy) + (qlo + r0) * p.dys[0] + (int64_t)h * p.dys[1], last, to + TILE);
    if (64 * w < 2 * ROWS) {  // lse of the rows, then delta, 64 a wave
      const float* src = (64 * w < ROWS ? p.stat : p.delta) + (int64_t)h * p.total_q + qlo + r0;
      copy4_to_lds(buffer_at(src), 4 * min(64 * w % ROWS + lane, last), to + 2 * TILE + 256 * w);
    }
  };
  // as in the forward: the next tile's copies and this one's reads do not overlap
  auto step = [&](int j, const unsigned char* __restrict qt, unsigned char* __restrict next) {
    if (S::BUFS == 2 && j + 1 < ntiles) stage(j + 1, next);
    const unsigned char *yt = qt + TILE, *stat = qt + 2 * TILE;
#pragma unroll sizeof(E) == 2 ? S::BLOCKS : 1
    for (int u = 0; u < S::BLOCKS; ++u) {
      const int tr = 32 * (S::BLOCKS * part + u), i0 = q0 + j % per * ROWS + tr;  // the wave's rows of the tile: i0 .. i0 + 31
      if (i0 >= lenq || i0 + 31 + off < first_key) continue;                      // none of them sees a key of this wave
      if (WIN && (i0 >= hidden_from || (is_far && ((j * (ROWS / 32) + tr / 32) & 3) != w))) continue;
      // bf16: the sums start at minus lse / scale and minus delta of their rows.  fp32 adds these last: a sum that starts at
      // 100 rounds each of its products at that size.
      constexpr bool START = sizeof(E) == 2;
      f32x16 s = zero16(), dp = zero16();
      auto add_stat = [&]() {
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(stat + 4 * (tr + 8 * a + 4 * half));
          const f32x4 de = DK ? *reinterpret_cast<const f32x4*>(stat + 4 * (ROWS + tr + 8 * a + 4 * half)) : zero4();
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            s[4 * a + x] = START ? ls[x] : s[4 * a + x] + ls[x];
            dp[4 * a + x] = START ? de[x] : dp[4 * a + x] + de[x];
          }
        }
      };
      if constexpr (START) {
        add_stat();
        __builtin_amdgcn_sched_group_barrier(0x100, DK ? 8 : 4, 0);
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = P::mma(s, P::row_frag(qt, tr + (lane & 31), ks, half), k[ks]);
      if constexpr (!DK) sched_products<P, KS, P::ROW_READS>();
      if constexpr (DK) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) dp = P::mma(dp, P::row_frag(yt, tr + (lane & 31), ks, half), v[ks]);
        sched_products<P, 2 * KS, P::ROW_READS>();
      }
      if constexpr (!START) add_stat();
      const bool whole = i0 + off >= first_key + 31 && i0 + 32 <= lenq &&
                         !(WIN && i0 >= cut_from);
      const int lo = max(key - off, 0) - i0, hi = (WIN ? last_row : lenq) - i0;  // rows lo .. hi - 1 of the block see the key
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = rho(half, i);
        float pr = __builtin_amdgcn_exp2f(s[i] * c);
        float d = pr * dp[i];
        if (!whole) {
          const bool sees = r >= lo && r < hi;
          pr = sees ? pr : 0.f;
          d = sees ? d : 0.f;
        }
        s[i] = pr;
        dp[i] = d;
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const typename P::frag pf = P::from_acc(s, m), df = P::from_acc(dp, m);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          if constexpr (DV) dv[ct] = P::mma(dv[ct], P::col_frag(yt, tr + 16 * m, ct, lane), pf);
          if constexpr (DK) dk[ct] = P::mma(dk[ct], P::col_frag(qt, tr + 16 * m, ct, lane), df);
        }
      }
      sched_products<P, 2 * CT * (DV + DK), P::COL_READS>();
    }
  };
  if (S::BUFS == 2 && ntiles > 0) stage(0, lds);
  for (int j = 0; j < ntiles; ++j) {
    if (S::BUFS == 1) {
      staged_barrier();
      stage(j, lds);
    }
    staged_barrier();
    step(j, lds + (S::BUFS == 2 ? (j & 1) * S::SLOT : 0), lds + (S::BUFS == 2 ? (~j & 1) * S::SLOT : 0));
  }
  const AttnParams& out = params_here();
  const int64_t at = t.lo + key, part_at = (((int64_t)sub * out.total_k + at) * out.KV + e) * P::D;
  const int64_t far_at = ((((int64_t)(far_slot >= 0 ? far_slot : out.far_slots + t.seq) * out.subsets + sub) * out.sinks + key) * out.KV + e) * P::D;
  const bool sinks = out.far_slots > 0 && t.row0 < out.sinks && (is_far || (t.seq >= 0 && t.seq < out.nseq));  // (keys outside the offsets have none)
  auto store_k = [&](int ct, const f32x16& x, float f) {
    if (WIN && sinks) store_row32(out.far_dk + far_at + 32 * ct, x, f, half, live && key < out.sinks);
    if (is_far) return;
    if (out.subsets > 1) store_row32(out.part_dk + part_at + 32 * ct, x, f, half, live);
    else store_row32(reinterpret_cast<E*>(out.dk) + at * out.dks[0] + (int64_t)e * out.dks[1] + 32 * ct, x, f, half, live);
  };
  auto store_v = [&](int ct, const f32x16& x) {
    if (WIN && sinks) store_row32(out.far_dv + far_at + 32 * ct, x, 1.f, half, live && key < out.sinks);
    if (is_far) return;
    if (out.subsets > 1) store_row32(out.part_dv + part_at + 32 * ct, x, 1.f, half, live);
    else store_row32(reinterpret_cast<E*>(out.dv) + at * out.dvs[0] + (int64_t)e * out.dvs[1] + 32 * ct, x, 1.f, half, live);
  };
  if (WIN && SPLIT < 4 && is_far) {
    staged_barrier();
    if constexpr (DK) join_sums<4>(dk, out.scale, lds, w, lane, [&](int ct, const f32x16& x) { store_k(ct, x, 1.f); });
    if constexpr (DV) join_sums<4>(dv, 1.f, lds, w, lane, store_v);
  } else if constexpr (SPLIT == 1) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if constexpr (DK) store_k(ct, dk[ct], out.scale);
      if constexpr (DV) store_v(ct, dv[ct]);
    }
  } else {
    staged_barrier();
    if constexpr (DK) join_sums<SPLIT>(dk, out.scale, lds, w, lane, [&](int ct, const f32x16& x) { store_k(ct, x, 1.f); });
    if constexpr (DV) join_sums<SPLIT>(dv, 1.f, lds, w, lane, store_v);
  }
}

// The subsets' sums added in order and rounded: four values of dk and of dv a lane.
template <class P>
__global__ void __launch_bounds__(256) attn_subsets_kernel(AttnParams p) {
  typedef typename P::elem E;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = p.total_k * p.KV * (P::D / 4);
  if (i >= n) return;
  const int64_t row = i / (P::D / 4), d = 4 * (i % (P::D / 4)), at = row / p.KV, e = row % p.KV;
  f32x4 dk = zero4(), dv = zero4();
  for (int s = 0; s < p.subsets; ++s) {
    dk += reinterpret_cast<const f32x4*>(p.part_dk)[s * n + i];
    dv += reinterpret_cast<const f32x4*>(p.part_dv)[s * n + i];
  }
  const float x[4] = {dk[0], dk[1], dk[2], dk[3]}, y[4] = {dv[0], dv[1], dv[2], dv[3]};
  store4(reinterpret_cast<E*>(p.dk) + at * p.dks[0] + e * p.dks[1] + d, x);
  store4(reinterpret_cast<E*>(p.dv) + at * p.dvs[0] + e * p.dvs[1] + d, y);
}

// The sinks' dk and dv: the sums of the near rows, then of the far ones' segments in order, of each the subsets in turn.  A thread
// has four values of one sink of one sequence and key head; `keys` and `rows` are Dkdv's.
template <class P>
__global__ void __launch_bounds__(256) attn_sinks_kernel(AttnParams p, int keys, int rows) {
  typedef typename P::elem E;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, each = (int64_t)p.sinks * p.KV * (P::D / 4);
  const int64_t b = i / each;
  if (b >= p.nseq) return;
  const int64_t in = i % each, d = 4 * (in % (P::D / 4)), e = in / (P::D / 4) % p.KV;
  const int key = (int)(in / (P::D / 4) / p.KV);
  int64_t klo, qlo;
  int lenk, lenq;
  other_rows(p.cu_k, p.nseq, p.total_k, (int)b, klo, lenk);
  other_rows(p.cu_q, p.nseq, p.total_q, (int)b, qlo, lenq);
  if (key >= lenk) return;
  f32x4 dk = zero4(), dv = zero4();
  const int64_t step = (int64_t)p.sinks * p.KV * P::D, at = ((int64_t)key * p.KV + e) * P::D + d;
  auto add = [&](int64_t slot, int64_t slots) {  // of consecutive slots
    const float *k = p.far_dk + slot * p.subsets * step + at, *v = p.far_dv + slot * p.subsets * step + at;
    const int64_t n = slots * p.subsets;
    for (int64_t i0 = 0; i0 < n; i0 += 8) {  // eight on their way at a time
      f32x4 x[8], y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = *reinterpret_cast<const f32x4*>(k + min(i0 + i, n - 1) * step);
        y[i] = *reinterpret_cast<const f32x4*>(v + min(i0 + i, n - 1) * step);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < n) dk += x[i], dv += y[i];
    }
  };
  add(p.far_slots + b, 1);
  const NearRows near(key / keys * keys, lenk - lenq, lenq, p.window, keys, rows);
  const int64_t first = qlo / FAR_ROWS + b + 1, end = near.to < lenq ? (lenq + FAR_ROWS - 1) / FAR_ROWS : 0;
  add(first + near.to / FAR_ROWS, end - near.to / FAR_ROWS);
  const float x[4] = {dk[0], dk[1], dk[2], dk[3]}, y[4] = {dv[0], dv[1], dv[2], dv[3]};
  store4(reinterpret_cast<E*>(p.dk) + (klo + key) * p.dks[0] + e * p.dks[1] + d, x);
  store4(reinterpret_cast<E*>(p.dv) + (klo + key) * p.dvs[0] + e * p.dvs[1] + d, y);
}

// dq of 128 / SPLIT query rows of a head: the forward's walk over the keys with S^T = K Q^T and dP^T = V dY^T, and
// dQ^T += K^T dS^T.
template <class P, int SPLIT>
struct Dq {
  static constexpr int ROWS = 128 / SPLIT, KEYS = SPLIT == 4 ? 128 : 64, BLOCKS = KEYS / 32 / SPLIT;
  static constexpr int TILE = KEYS * P::ROW, BUFS = 4 * TILE <= 128 * 1024 ? 2 : 1;
  static constexpr int JOIN = SPLIT > 1 ? 4 * (P::D / 32) * 4096 : 0;
  static constexpr int LDS = 2 * BUFS * TILE > JOIN ? 2 * BUFS * TILE : JOIN;
};

template <class P, int SPLIT, bool WIN>
__device__ __forceinline__ void dq(int id, int slots, unsigned char* lds) {
  const AttnParams& p = params_here();
  typedef typename P::elem E;
  typedef Dq<P, SPLIT> S;
  constexpr int KS = P::D / 16, CT = P::D / 32, KEYS = S::KEYS, TILE = S::TILE;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = w % SPLIT;
  int h;
  if (p.H % 8 == 0) {
    const int per = p.H / 8;
    h = id % 8 * per + id / 8 % per;
  } else {
    h = id % p.H;
  }
  const SeqTile t = find_heavy<S::ROWS, false>(p.cu_q, p.nseq, p.total_q, id / p.H, slots, lane);
  if (t.row0 < 0) return;
  const int lenq = t.len;
  int64_t klo;
  int lenk;
  other_rows(p.cu_k, p.nseq, p.total_k, t.seq, klo, lenk);
  const int off = lenk - lenq;
  const int first_row = t.row0 + 32 * (w / SPLIT), row = first_row + (lane & 31);
  const bool live = row < lenq;
  const int64_t at = t.lo + min(row, lenq - 1);
  const E* kb = reinterpret_cast<const E*>(p.k) + klo * p.ks[0] + (int64_t)(h / p.G) * p.ks[1];
  const E* vb = reinterpret_cast<const E*>(p.v) + klo * p.vs[0] + (int64_t)(h / p.G) * p.vs[1];
  typename P::frag q[KS], dy[KS];
  {
    const E* qsrc = reinterpret_cast<const E*>(p.q) + at * p.qs[0] + (int64_t)h * p.qs[1];
    const E* ysrc = reinterpret_cast<const E*>(p.dy) + at * p.dys[0] + (int64_t)h * p.dys[1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      q[ks] = P::load(qsrc + 16 * ks + 8 * half);
      dy[ks] = P::load(ysrc + 16 * ks + 8 * half);
    }
  }
  const float c = p.scale * LOG2E;
  const float ls = p.stat[(int64_t)h * p.total_q + at] * c, de = p.delta[(int64_t)h * p.total_q + at];
  f32x16 sum[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) sum[ct] = zero16();

  const int sees = min(lenk, t.row0 + S::ROWS + off);
  const KeyWalk walk(t.row0 + off, sees, WIN ? p.window : (int)NO_WINDOW, WIN ? p.sinks : 0, KEYS);
  const int ntiles = WIN ? walk.tiles : sees > 0 ? (sees + KEYS - 1) / KEYS : 0;
  auto tile = [&](int j) { return WIN ? walk.at(j) : j; };
  const int wfirst = first_row + off, wlast = wfirst + 31;
  const Stager<P, KEYS, 4> stage_k(p.ks[0], w, lane), stage_v(p.vs[0], w, lane);
  auto stage = [&](int j, unsigned char* to) {
    const int k0 = tile(j) * KEYS, last = min(lenk - 1 - k0, KEYS - 1);
    stage_k(kb + k0 * p.ks[0], last, to);
    stage_v(vb + k0 * p.vs[0], last, to + TILE);
  };
  auto step = [&](int j, const unsigned char* __restrict kt, unsigned char* __restrict next) {
    if (S::BUFS == 2 && j + 1 < ntiles) stage(j + 1, next);
    const unsigned char* vt = kt + TILE;
#pragma unroll
    for (int u = 0; u < S::BLOCKS; ++u) {
      const int r0 = 32 * (S::BLOCKS * part + u), j0 = tile(j) * KEYS + r0;  // the wave's keys of the tile
      if (j0 > wlast || j0 >= lenk) continue;
      if (WIN && window_hides(wfirst, j0, j0 + 31, p.window, p.sinks)) continue;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = P::mma(s, P::row_frag(kt, r0 + (lane & 31), ks, half), q[ks]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) dp = P::mma(dp, P::row_frag(vt, r0 + (lane & 31), ks, half), dy[ks]);
      sched_products<P, 2 * KS, P::ROW_READS>();
      const bool whole = j0 + 31 <= wfirst && !(WIN && window_cuts(wlast, j0, j0 + 31, p.window, p.sinks));
      const int limit = row + off - j0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float d = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, ls)) * (dp[i] + de);
        if (!whole) d = rho(half, i) <= limit && (!WIN || rho(half, i) > limit - p.window || rho(half, i) < p.sinks - j0) ? d : 0.f;
        dp[i] = d;
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const typename P::frag df = P::from_acc(dp, m);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) sum[ct] = P::mma(sum[ct], P::col_frag(kt, r0 + 16 * m, ct, lane), df);
      }
      sched_products<P, 2 * CT, P::COL_READS>();
    }
  };
  if (S::BUFS == 2 && ntiles > 0) stage(0, lds);
  for (int j = 0; j < ntiles; ++j) {
    if (S::BUFS == 1) {
      staged_barrier();
      stage(j, lds);
    }
    staged_barrier();
    step(j, lds + (S::BUFS == 2 ? (j & 1) * 2 * TILE : 0), lds + (S::BUFS == 2 ? (~j & 1) * 2 * TILE : 0));
  }
  E* dst = reinterpret_cast<E*>(p.dq) + (t.lo + row) * p.dqs[0] + (int64_t)h * p.dqs[1];
  if constexpr (SPLIT == 1) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) store_row32(dst + 32 * ct, sum[ct], p.scale, half, live);
  } else {
    staged_barrier();
    join_sums<SPLIT>(sum, p.scale, lds, w, lane, [&](int ct, const f32x16& x) { store_row32(dst + 32 * ct, x, 1.f, half, live); });
  }
}

// All of a backward's sums in one launch: dk's and dv's workgroups first (of 128 features dv's, then dk's), then dq's.  None
// waits for another, and the last of one kind leave no CU idle.  Three sequences of 101 to 1024 rows, 4 heads, fp32: 53 us,
// as two launches 51 and 38; 8192 rows, 32 heads, bf16: within 1 % of what the three launches took.
template <class P, int SPLIT, bool WIN>
__global__ void __launch_bounds__(256, sizeof(typename P::elem) == 2 ? 2 : 1)
    attn_grads_kernel(AttnParams p, int slots_k, int slots_q, int part, int nk, int far) {
  constexpr int LDS = Dkdv<P, SPLIT>::LDS > Dq<P, SPLIT>::LDS ? Dkdv<P, SPLIT>::LDS : Dq<P, SPLIT>::LDS;
  __shared__ __attribute__((aligned(256))) unsigned char lds[LDS];
  constexpr int PARTS = P::D == 64 ? 1 : 2;
  const int id = blockIdx.x;
  if (id >= PARTS * part) return dq<P, SPLIT, WIN>(id - PARTS * part, slots_q, lds);
  if constexpr (PARTS == 1) {
    if (id < nk) dkdv<P, SPLIT, true, true, WIN>(id, slots_k, far, lds);
  } else if (id < part) {
    if (id < nk) dkdv<P, SPLIT, true, false, WIN>(id, slots_k, far, lds);
  } else if (id - part < nk) {
    dkdv<P, SPLIT, false, true, WIN>(id - part, slots_k, far, lds);
  }
}

template <class P>
static int launch_delta(const AttnParams& p, hipStream_t st) {
  const int64_t blocks = (p.total_q * p.H + 15) / 16, most = max_groups(256);
  int rc = KDN_OK;
  for (int64_t first = 0; first < blocks && rc == KDN_OK; first += most) {  // 8 million rows of 32 heads are more than one grid
    hipLaunchKernelGGL(attn_delta_kernel<P>, dim3((unsigned)std::min(most, blocks - first)), dim3(256), 0, st, p, const_cast<float*>(p.stat), const_cast<float*>(p.delta),
                       16 * first);
    rc = launch_status();
  }
  return rc;
}

template <class P, int SPLIT, bool WIN>
static int launch_grads(const AttnParams& p, hipStream_t st) {
  const int64_t slots_k = p.total_k > 0 ? tile_slots(p.total_k, Dkdv<P, SPLIT>::KEYS, p.nseq) : 0;
  const int64_t slots_q = p.total_q > 0 ? tile_slots(p.total_q, Dq<P, SPLIT>::ROWS, p.nseq) : 0;
  const int64_t far = WIN && p.total_q > 0 ? p.far_slots * ((p.sinks + 31) / 32) * p.KV * p.subsets : 0;
  const int64_t far_blocks = far > 0 ? (p.nseq * p.sinks * p.KV * (P::D / 4) + 255) / 256 : 0;
  const int64_t nk = slots_k * p.KV * p.subsets + far, part = (nk + 7) / 8 * 8;  // a workgroup's number mod 8 is its XCD
  const int64_t grid = part * (P::D == 64 ? 1 : 2) + slots_q * p.H;
  const int64_t blocks = p.subsets > 1 && p.total_k > 0 ? (p.total_k * p.KV * (P::D / 4) + 255) / 256 : 0;
  if (std::max({grid, far_blocks, blocks}) > max_groups(256)) return KDN_ERR_UNSUPPORTED;
  int rc = launch_delta<P>(p, st);
  if (rc != KDN_OK) return rc;
  hipLaunchKernelGGL((attn_grads_kernel<P, SPLIT, WIN>), dim3((unsigned)grid), dim3(256), 0, st, p, (int)slots_k, (int)slots_q, (int)part, (int)nk,
                     (int)far);
  rc = launch_status();
  if (rc == KDN_OK && blocks > 0) {
    hipLaunchKernelGGL(attn_subsets_kernel<P>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    rc = launch_status();
  }
  if (rc == KDN_OK && far_blocks > 0) {
    hipLaunchKernelGGL(attn_sinks_kernel<P>, dim3((unsigned)far_blocks), dim3(256), 0, st, p, Dkdv<P, SPLIT>::KEYS, Dkdv<P, SPLIT>::ROWS);
    rc = launch_status();
  }
  return rc;
}

template <class P, bool WIN>
static int launch_grads(const AttnParams& p, hipStream_t st) {
  // one split for both walks, that of the one with fewer tiles (with as many keys as queries they agree: bwd_subsets; few rows
  // over many keys split the keys' walk as well, which has not been measured)
  auto rule = [](int64_t rows, int64_t heads) {
    return WIN ? window_split(rows, heads, WINDOW_FOUR<P>) : attn_split(rows, heads);
  };
  const int split = std::max(rule(p.total_k, (int64_t)p.KV * p.subsets), rule(p.total_q, p.H));
  if constexpr (!WIN || WINDOW_FOUR<P>)
    if (split == 4) return launch_grads<P, 4, WIN>(p, st);
  return split == 2 ? launch_grads<P, 2, WIN>(p, st) : launch_grads<P, 1, WIN>(p, st);
}

template <class P>
static int launch_bwd(const AttnParams& p, hipStream_t st) {
  return p.window < NO_WINDOW ? launch_grads<P, true>(p, st) : launch_grads<P, false>(p, st);
}

// Subsets of the query heads that share a key head whose dk and dv are summed apart: as many as it takes to have eight
// workgroups of 128 keys for each CU (two run there at a time, and the first keys have twice the average's work).  8192 rows,
// 32 heads over 8: four subsets 2900 us a training step, two 2935.
// Under a window all tiles have about the same work, and four workgroups for each CU are enough: 16384 rows in a window of 1024, one
// subset 1951 us a step, two (and their sums' launch) 2062.
static int bwd_subsets(const kdn_attn_args* f, bool window) {
  const int G = (int)(f->H / f->H_kv);
  const int64_t tiles = f->total_k / 128 * f->H_kv;
  int n = 1;
  while (n < G && (tiles * n < (window ? 1024 : 2048) || G % n != 0)) ++n;
  return n;
}
static size_t bwd_row_bytes(const kdn_attn_args* f) { return ((size_t)f->H * (size_t)f->total_q * 4 + 255) / 256 * 256 + 256; }
static size_t bwd_part_bytes(const kdn_attn_args* f) { return (size_t)f->total_k * (size_t)f->H_kv * (size_t)f->d * 4; }
// Slots of the far rows' segments, `sinks` after attn_window.
static int64_t bwd_far_slots(const kdn_attn_args* f, int64_t sinks) {
  return sinks > 0 && sinks <= FAR_SINKS ? tile_slots(f->total_q, FAR_ROWS, f->num_seqs) : 0;
}
// Of those and the near rows of each sequence.
static size_t bwd_far_bytes(const kdn_attn_args* f, int subsets, int64_t sinks) {
  const int64_t slots = bwd_far_slots(f, sinks);
  if (slots == 0) return 0;
  const size_t each = (size_t)subsets * (size_t)sinks * (size_t)f->H_kv * (size_t)f->d * 4;
  size_t all;
  return __builtin_mul_overflow((size_t)(slots + f->num_seqs), each, &all) || all > ((size_t)1 << 48) ? (size_t)1 << 48 : all;
}

}  // namespace kdn

using namespace kdn;

static size_t bwd_workspace_bytes(const kdn_attn_bwd_args* a, int64_t window, int64_t sinks) {
  if (!a || attn_check(a->fwd) != KDN_OK || window < 1 || sinks < 0) return 0;
  AttnParams p = attn_params(a->fwd);
  attn_window(p, window, sinks);
  const int subsets = bwd_subsets(a->fwd, p.window < NO_WINDOW);
  return 2 * bwd_row_bytes(a->fwd) + (subsets > 1 ? 2 * subsets * bwd_part_bytes(a->fwd) : 0) +
         2 * bwd_far_bytes(a->fwd, subsets, p.sinks);
}

static int attn_bwd(const kdn_attn_bwd_args* a, int64_t window, int64_t sinks, void* stream) {
  if (!a) return KDN_ERR_INVALID_ARGUMENT;
  const kdn_attn_args* f = a->fwd;
  int rc = attn_check(f);
  if (rc != KDN_OK) return rc;
  if (f->total_q == 0 && f->total_k == 0) return KDN_OK;
  if (f->total_q > 0) {
    if ((rc = attn_check_tensors(f)) != KDN_OK) return rc;
    if (!f->lse || !a->dy || !a->dq) return KDN_ERR_INVALID_ARGUMENT;
  }
  if (!f->cu_q || (f->total_k > 0 && (!f->k || !f->v || !a->dk || !a->dv))) return KDN_ERR_INVALID_ARGUMENT;
  if (!aligned(a->dy, 16) || !aligned(a->dq, 16) || !aligned(a->dk, 16) || !aligned(a->dv, 16) || !aligned(a->workspace, 16) ||
      !attn_strides_ok(a->dy_stride, f->dtype) || !attn_strides_ok(a->dq_stride, f->dtype) ||
      !attn_strides_ok(a->dk_stride, f->dtype) || !attn_strides_ok(a->dv_stride, f->dtype) ||
      !attn_strides_ok(f->k_stride, f->dtype) || !attn_strides_ok(f->v_stride, f->dtype) || !aligned(f->k, 16) || !aligned(f->v, 16))
    return KDN_ERR_MISALIGNED;
  if (!stage_reach(a->dy_stride[0], f->dtype)) return KDN_ERR_UNSUPPORTED;
  if (!a->workspace || a->workspace_bytes < bwd_workspace_bytes(a, window, sinks)) return KDN_ERR_WORKSPACE_TOO_SMALL;
  AttnParams p = attn_params(f);
  p.dy = a->dy; p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
  float *stat = reinterpret_cast<float*>(a->workspace), *delta = stat + bwd_row_bytes(f) / 4;
  p.stat = stat;
  p.delta = delta;
  attn_window(p, window, sinks);
  p.subsets = bwd_subsets(f, p.window < NO_WINDOW);
  p.part_dk = reinterpret_cast<float*>((unsigned char*)a->workspace + 2 * bwd_row_bytes(f));
  p.part_dv = p.part_dk + (size_t)p.subsets * bwd_part_bytes(f) / 4;
  p.far_slots = bwd_far_slots(f, p.sinks);
  p.far_dk = p.subsets > 1 ? p.part_dv + (size_t)p.subsets * bwd_part_bytes(f) / 4 : p.part_dk;
  p.far_dv = p.far_dk + bwd_far_bytes(f, p.subsets, p.sinks) / 4;
  for (int i = 0; i < 2; ++i) {
    p.dys[i] = a->dy_stride[i]; p.dqs[i] = a->dq_stride[i]; p.dks[i] = a->dk_stride[i]; p.dvs[i] = a->dv_stride[i];
  }
  hipStream_t st = as_stream(stream);
  if (f->dtype == KDN_DTYPE_BF16)
    return f->d == 64 ? launch_bwd<AttnBF16<64>>(p, st) : launch_bwd<AttnBF16<128>>(p, st);
  return f->d == 64 ? launch_bwd<AttnF32<64>>(p, st) : launch_bwd<AttnF32<128>>(p, st);
}

extern "C" size_t kdn_attn_bwd_workspace_bytes(const kdn_attn_bwd_args* a) { return bwd_workspace_bytes(a, NO_WINDOW, 0); }
extern "C" int kdn_attn_bwd(const kdn_attn_bwd_args* a, void* stream) { return attn_bwd(a, NO_WINDOW, 0, stream); }

extern "C" size_t kdn_attn_window_bwd_workspace_bytes(const kdn_attn_bwd_args* a, int64_t window, int64_t sinks) {
  return bwd_workspace_bytes(a, window, sinks);
}
extern "C" int kdn_attn_window_bwd(const kdn_attn_bwd_args* a, int64_t window, int64_t sinks, void* stream) {
  if (window < 1 || sinks < 0) return KDN_ERR_INVALID_ARGUMENT;
  return attn_bwd(a, window, sinks, stream);
}
