// The attention weight that each key of a packed batch got: w_ej = sum over the rows i that see key j and the query heads h that share
// key head e of exp(scale q_ih.k_je - lse_hi), the column sums of the softmax, for a cache that keeps the keys of largest weight.
//
// As dk's and dv's walk without their products (kdn_attn_bwd.hip): a wave owns 32 keys, or two times 32, with their K fragments in
// registers, and the query rows of the heads pass through LDS in tiles of 64 or 128; S = Q K^T has a key a lane and its rows in the lane's
// registers, so that a column's sum is register arithmetic and one exchange between the halves of the wave.
//   What bounds it: the exponential of each pair and the multiplication and the addition around it, at 64 features more than the
// products.  Three prompts of 1000 to 8192 rows, 16 heads of 64 over 4, bf16: 116 to 128 us by card, of which the join 5, 0.65 to 0.72 PFLOP/s; 14.6 vector
// instructions for each of the matrix cores' (12 are the arithmetic's), which are busy 30 %.  With 32 keys a wave it was 150,
// with the comparisons of the cut tiles formed for every block 150 too, with 64 rows a tile 133.  The products of one block beside the
// exponentials of the one before, in one wave, took 147 for 128 (230 registers).
#include <algorithm>
#include <cmath>
#include "kdn_attn_tile.hpp"

namespace kdn {

struct WeightsParams {
  AttnParams a;        // q, k, their strides, lse, offsets, heads, scale, window
  float* weights;      // [slot][key head], places next to one another
  int64_t weights_stride[2], places, num_slots;
  const int32_t* slots;
  float* part;         // [part][key head][total_k], or NULL: the sums go to their places at once
  float* far_part;     // [far][sequence][key head][sink]: of the rows behind a window, which see the sinks alone
  int parts, far, far_tiles, add;  // shares of a tile's rows; of the far ones', and tiles of the keys that have some
  int long_rows;       // few rows: a sequence with more has its tiles dealt out; INT_MAX where none has
};

template <class P>
struct WeightsTile {
  static constexpr int BLOCKS = P::ROW <= 256 ? 2 : 1;  // of 32 keys to a wave: as many as leave the registers of two waves a SIMD
  static constexpr int KEYS = 128 * BLOCKS, ROWS = P::ROW <= 128 ? 128 : 64, TILE = ROWS * P::ROW, SLOT = TILE + ROWS * 4;
};

// exp(scale q.k - lse) of 32 rows from i0 on and a wave's keys, added to the keys' sums: `rows` the tile in LDS, r0 the first row in it,
// `bits` their -lse in bits.
struct WeightsMask {
  int off, lenq, window, sinks;
};
template <class P, int BLOCKS, bool WIN>
__device__ __forceinline__ void add_weights(float (&sum)[BLOCKS], const typename P::frag (&k)[BLOCKS][P::D / 16], const unsigned char* rows, int r0,
                                            const float* bits, int i0, int first_key, int lane, float c, const WeightsMask& m) {
  constexpr int KS = P::D / 16, AHEAD = KS < P::AHEAD ? KS : P::AHEAD;
  const int half = lane >> 5;
  float l[16];
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(bits + 8 * a + 4 * half);
#pragma unroll
    for (int y = 0; y < 4; ++y) l[4 * a + y] = x[y];
  }
  f32x16 s[BLOCKS];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) s[b] = zero16();
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const typename P::frag a = P::row_frag(rows, r0 + (lane & 31), ks, half);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) s[b] = P::mma(s[b], a, k[b][ks]);
  }
  // as sched_products, an operand for BLOCKS products; the rows' bits first
  __builtin_amdgcn_sched_group_barrier(0x100, 4 + AHEAD * P::ROW_READS, 0);
#pragma unroll
  for (int i = 0; i < KS - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, P::MFMAS * BLOCKS, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, P::ROW_READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * P::MFMAS * BLOCKS, 0);
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    const int fk = first_key + 32 * b, kk = fk + (lane & 31);
    const bool whole = i0 + m.off >= fk + 31 && i0 + 32 <= m.lenq && !(WIN && window_cuts(i0 + 31 + m.off, fk, fk + 31, m.window, m.sinks));
    float part = 0.f;  // of a block, then of the walk: a long column's terms are added to few large sums
    if (whole) {
#pragma unroll
      for (int i = 0; i < 16; ++i) part += __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], c, l[i]));
    } else {
      int lo = max(kk - m.off, 0) - i0, hi = (WIN && kk >= m.sinks ? min(m.lenq, kk - m.off + m.window) : m.lenq) - i0;
      asm volatile("" : "+v"(lo), "+v"(hi));  // the comparisons stay here: formed for every block they were an eighth of the vector instructions
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = rho(half, i);
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], c, l[i]));
        part += r >= lo && r < hi ? x : 0.f;
      }
    }
    sum[b] += part;
  }
}

// A key's sum to its place: those before the sequence's first row are added to if the call says so, others are set.
__device__ __forceinline__ void put_weight(const WeightsParams& p, int seq, int e, int key, int off, float sum) {
  if (seq < 0 || seq >= p.a.nseq || key >= p.places) return;
  const int64_t slot = p.slots ? p.slots[seq] : seq;
  if (slot < 0 || slot >= p.num_slots) return;
  float* w = p.weights + slot * p.weights_stride[0] + e * p.weights_stride[1] + key;
  *w = p.add && key < off ? *w + sum : sum;
}

// `parts` workgroups share the tiles of query rows of a tile of keys evenly, each the next stretch of them.  (Fewer for the later
// keys, which fewer rows see: three prompts of 1000 to 8192 rows 131 us and more, for 127.)
//   WIN: the rows that see a tile of keys end `window` behind it, but for the sinks'.  Where prompts are long the rows behind are shared
// by `far` workgroups more for each tile with sinks: one that walked them all would run on when the others are done (one prompt of 8000
// rows in a window of 300, 32 heads of 128 over 8, as many shares for all tiles: 109 us with 16, 178 with eight).
template <class P, bool WIN>
__global__ void __launch_bounds__(256, sizeof(typename P::elem) == 2 ? 2 : 1) attn_weights_kernel(WeightsParams wp, int64_t slots) {
  typedef typename P::elem E;
  typedef WeightsTile<P> S;
  constexpr int KS = P::D / 16, BLOCKS = S::BLOCKS, ROWS = S::ROWS;
  __shared__ __attribute__((aligned(256))) unsigned char lds[2 * S::SLOT];
  const AttnParams& p = wp.a;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e = blockIdx.x % p.KV;
  const int64_t u = blockIdx.x / p.KV, nfar = WIN ? p.nseq * wp.far_tiles * wp.far : 0;
  const bool is_far = WIN && u < nfar;
  const int parts = is_far ? wp.far : wp.parts, part = (int)((is_far ? u : u - nfar) % parts);
  SeqTile t;
  if (is_far) {
    t.seq = (int)(u / parts / wp.far_tiles);
    t.row0 = (int)(u / parts % wp.far_tiles) * S::KEYS;
    other_rows(p.cu_k, p.nseq, p.total_k, t.seq, t.lo, t.len);
    if (t.row0 >= t.len) return;
  } else {
    t = find_heavy<S::KEYS, true>(p.cu_k, p.nseq, p.total_k, (u - nfar) / parts, slots, lane);
    if (t.row0 < 0) return;
  }
  const int lenk = t.len;
  int64_t qlo;
  int lenq;
  other_rows(p.cu_q, p.nseq, p.total_q, t.seq, qlo, lenq);
  const int off = lenk - lenq;
  const int first_key = t.row0 + 32 * BLOCKS * w, key = first_key + (lane & 31);
  // the rows that see a key of the tile, in whole tiles; past the window only the sinks are seen
  int q0 = max(t.row0 - off, 0) / ROWS * ROWS, q1 = lenq;
  if (WIN && (wp.far > 0 || t.row0 >= p.sinks)) {
    const int end = min(lenq, max(t.row0 + S::KEYS - 1 - off + p.window, 0));
    const int to = q0 < end ? q0 + (end - q0 + ROWS - 1) / ROWS * ROWS : q0;  // whole tiles: the far rows begin behind them
    if (is_far) q0 = to;
    else q1 = min(to, lenq);
  }
  const int per = q0 < q1 ? (q1 - q0 + ROWS - 1) / ROWS : 0;
  const int64_t all = (int64_t)per * p.G, j0 = all * part / parts;
  const int tiles = (int)(all * (part + 1) / parts - j0);
  typename P::frag k[BLOCKS][KS];
  float sum[BLOCKS];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    sum[b] = 0.f;
    if (tiles == 0) continue;  // (behind a window most keys have no rows here)
    const E* src = reinterpret_cast<const E*>(p.k) + (t.lo + min(key + 32 * b, lenk - 1)) * p.ks[0] + (int64_t)e * p.ks[1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k[b][ks] = P::load(src + 16 * ks + 8 * half);
  }
  const float c = p.scale * LOG2E;
  const Stager<P, ROWS, 4> stage_q(p.qs[0], w, lane);
  float lse = 0.f;  // of the tile that is on its way, 64 rows a wave
  int head = e * p.G, row = q0;  // of that tile
  if (per > 0) head += (int)(j0 / per), row += (int)(j0 % per) * ROWS;
  auto stage = [&](unsigned char* to) {
    const int last = min(lenq - 1 - row, ROWS - 1);
    stage_q(reinterpret_cast<const E*>(p.q) + (qlo + row) * p.qs[0] + (int64_t)head * p.qs[1], last, to);
    if (64 * w < ROWS) lse = p.lse[(int64_t)head * p.total_q + qlo + row + min(64 * w + lane, last)];
  };
  auto step = [&](int j, const unsigned char* __restrict qt, unsigned char* __restrict next) {
    const int r0 = row;
    row += ROWS;
    if (row >= q0 + per * ROWS) row = q0, ++head;
    if (j + 1 < tiles) stage(next);
#pragma unroll
    for (int u = 0; u < ROWS / 32; ++u) {
      const int i0 = r0 + 32 * u;  // the rows i0 .. i0 + 31
      if (i0 >= lenq || i0 + 31 + off < first_key) continue;
      if (WIN && window_hides(i0 + off, first_key, first_key + 32 * BLOCKS - 1, p.window, p.sinks)) continue;
      add_weights<P, BLOCKS, WIN>(sum, k, qt, 32 * u, reinterpret_cast<const float*>(qt + S::TILE) + 32 * u, i0, first_key, lane, c,
                                  {off, lenq, p.window, p.sinks});
    }
  };
  if (tiles > 0) stage(lds);
  for (int j = 0; j < tiles; ++j) {
    unsigned char* slot = lds + (j & 1) * S::SLOT;
    if (64 * w < ROWS) reinterpret_cast<float*>(slot + S::TILE)[64 * w + lane] = lse * -LOG2E;  // (read last two tiles ago)
    staged_barrier();
    step(j, slot, lds + (~j & 1) * S::SLOT);
  }
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    const int kk = key + 32 * b;
    const float x = half_sum(sum[b]);
    if (half != 0 || kk >= lenk) continue;
    if (is_far) {
      if (kk < p.sinks) wp.far_part[(((int64_t)part * p.nseq + t.seq) * p.KV + e) * p.sinks + kk] = x;
    } else if (wp.part) wp.part[((int64_t)part * p.KV + e) * p.total_k + t.lo + kk] = x;
    else put_weight(wp, t.seq, e, kk, off, x);
  }
}

// Few rows over many keys (the last rows of prompts): a sequence's rows of all heads of a key head stay in LDS while the workgroup
// goes along the keys, `per` tiles of them one after another, 32 keys a wave.  What is read is K, once.  More rows than LDS holds come in
// batches, for each tile of keys anew.  Four waves a SIMD have each other's loads, products and exponentials to wait beside: the last 64
// rows of five prompts of up to 32768 keys, 32 heads of 128 over 8, bf16: 64 us, 0.19 GB at 2.9 TB/s, 0.36 PFLOP/s; with 64 keys a wave,
// the next ones loaded ahead and two waves a SIMD 71.  Without the products 35 (5.4 TB/s), of which half is what starts and ends it;
// by the kernel above, whose workgroups stage the rows anew for every 256 keys, 88.
template <class P>
struct WeightsFew {
  static constexpr int WAVES = 8, BLOCKS = 1, KEYS = 32 * WAVES * BLOCKS, ROWS = 64, TILE = ROWS * P::ROW;
  static constexpr int TILES = 65536 / TILE, LDS = TILES * (TILE + ROWS * 4);  // two workgroups a CU
};

// The host knows the sequences' rows together, not apart: a prompt's piece beside decoding streams has many, and the tiles of its keys would be
// the walks of a few workgroups.  LONG: the tiles of the sequences that have more than long_rows, dealt out one by one; without it
// those are left out.  128 features, 32 heads over 8, 63 streams with one row and one with 4096, 4096 keys each: 3350 us, so 470; with
// 256 rows 369, so 173 (one launch for both, with dealt workgroups first, 357 and 178, and its registers cost even batches a tenth).
//
// The i-th tile of keys of those sequences, in order; past their last one a negative first row.
template <int KEYS>
__device__ __forceinline__ SeqTile long_tile(const WeightsParams& wp, int64_t i, int lane) {
  const AttnParams& p = wp.a;
  SeqTile t;
  t.row0 = -1;
  for (int64_t b0 = 0; b0 < p.nseq; b0 += 64) {
    int64_t lo, from;
    int len, rows;
    const int b = (int)min(b0 + lane, p.nseq);  // (the number past the last has no rows)
    other_rows(p.cu_k, p.nseq, p.total_k, b, lo, len);
    other_rows(p.cu_q, p.nseq, p.total_q, b, from, rows);
    const int n = rows > wp.long_rows ? (len + KEYS - 1) / KEYS : 0;
    int upto = n;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const int x = __shfl_up(upto, s);
      if (lane >= s) upto += x;
    }
    const int all = __builtin_amdgcn_readlane(upto, 63);
    if (i >= all) {
      i -= all;
      continue;
    }
    const int at = __builtin_amdgcn_readfirstlane(__popcll(__ballot(upto <= i)));
    t.seq = (int)b0 + at;
    t.lo = (int64_t)__builtin_amdgcn_readlane((int)(lo >> 32), at) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)lo, at);
    t.len = __builtin_amdgcn_readlane(len, at);
    t.row0 = ((int)i - __builtin_amdgcn_readlane(upto - n, at)) * KEYS;
    return t;
  }
  return t;
}

template <class P, bool LONG>
__global__ void __launch_bounds__(64 * WeightsFew<P>::WAVES, 4) attn_weights_few_kernel(WeightsParams wp, int64_t slots, int64_t per) {
  typedef typename P::elem E;
  typedef WeightsFew<P> S;
  constexpr int KS = P::D / 16, BLOCKS = S::BLOCKS, KEYS = S::KEYS, ROWS = S::ROWS, TILES = S::TILES;
  __shared__ __attribute__((aligned(256))) unsigned char lds[S::LDS];
  const AttnParams& p = wp.a;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // A workgroup's number mod 8 is its XCD, and an XCD has all heads of its keys: whole rows of them come through its cache (1 % less time
  // than with a head to an XCD).
  const int e = blockIdx.x / 8 % p.KV;
  const int64_t group = (int64_t)(blockIdx.x / 8 / p.KV) * 8 + blockIdx.x % 8;
  int64_t slot = (LONG ? group : group * per) - (LONG ? gridDim.x / p.KV : 1);
  const int64_t end = min(slot + 1 + per, slots);
  SeqTile now;
  now.row0 = -1;
  now.len = 0;
  // the tile after `t`, one with keys, or with a negative first row the end
  auto after = [&](SeqTile t) {
    if constexpr (LONG) return long_tile<KEYS>(wp, slot += gridDim.x / p.KV, lane);
    while (++slot < end) {
      if (t.row0 >= 0 && t.row0 + KEYS < t.len) {
        t.row0 += KEYS;
        return t;
      }
      t = find_tile<KEYS>(p.cu_k, p.nseq, p.total_k, slot, lane);
      if (t.row0 >= 0) return t;
    }
    t.row0 = -1;
    return t;
  };
  typename P::frag k[BLOCKS][KS];
  auto load = [&](const SeqTile& t) {
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const int64_t key = t.lo + min(t.row0 + 32 * (BLOCKS * w + b) + (lane & 31), t.len - 1);
      const E* src = reinterpret_cast<const E*>(p.k) + key * p.ks[0] + (int64_t)e * p.ks[1];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) k[b][ks] = P::load(src + 16 * ks + 8 * half);
    }
    asm volatile("" ::: "memory");  // they are issued here, not where they are used
  };
  const float c = p.scale * LOG2E;
  const Stager<P, ROWS, S::WAVES> stage_q(p.qs[0], w, lane);
  now = after(now);
  if (now.row0 < 0) return;
  load(now);
  int staged = -2, known = -2;  // the sequences whose rows are in LDS, all of them, and whose offsets are here
  int64_t qlo = 0;
  int lenq = 0;
  while (now.row0 >= 0) {
    const SeqTile then = after(now);
    if (known != now.seq) other_rows(p.cu_q, p.nseq, p.total_q, now.seq, qlo, lenq);
    known = now.seq;
    const int off = now.len - lenq, first_key = now.row0 + 32 * BLOCKS * w;
    const int each = (lenq + ROWS - 1) / ROWS;
    const bool others = !LONG && lenq > wp.long_rows;  // the other launch's
    const int64_t tiles = others ? 0 : (int64_t)each * p.G;
    float sum[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) sum[b] = 0.f;
    for (int64_t j0 = 0; j0 < tiles; j0 += TILES) {
      const int n = (int)min((int64_t)TILES, tiles - j0);
      int r0 = (int)(j0 % each) * ROWS;  // the batch's first tile's first row
      if (staged != now.seq || tiles > TILES) {
        __syncthreads();  // the rows before are read
        int h = e * p.G + (int)(j0 / each), r = r0;
        for (int j = 0; j < n; ++j) {
          const int last = min(lenq - 1 - r, ROWS - 1);
          stage_q(reinterpret_cast<const E*>(p.q) + (qlo + r) * p.qs[0] + (int64_t)h * p.qs[1], last, lds + j * S::TILE);
          if (w == j % S::WAVES) reinterpret_cast<float*>(lds + TILES * S::TILE)[j * ROWS + lane] = p.lse[(int64_t)h * p.total_q + qlo + r + min(lane, last)] * -LOG2E;
          r += ROWS;
          if (r >= lenq) r = 0, ++h;
        }
        staged_barrier();
        staged = now.seq;
      }
      for (int j = 0; j < n; ++j) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i0 = r0 + 32 * u;
          if (i0 >= lenq || i0 + 31 + off < first_key) continue;
          add_weights<P, BLOCKS, false>(sum, k, lds + j * S::TILE, 32 * u, reinterpret_cast<const float*>(lds + TILES * S::TILE) + j * ROWS + 32 * u, i0,
                                      first_key, lane, c, {off, lenq, 0, 0});
        }
        r0 += ROWS;
        if (r0 >= lenq) r0 = 0;
      }
    }
    if (then.row0 >= 0) load(then);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const int key = first_key + 32 * b + (lane & 31);
      const float x = half_sum(sum[b]);
      if (half == 0 && key < now.len && !others) put_weight(wp, now.seq, e, key, off, x);
    }
    now = then;
  }
}

// The parts' sums in order, a thread a key.
__global__ void __launch_bounds__(256) attn_weights_join_kernel(WeightsParams wp) {
  const AttnParams& p = wp.a;
  const int e = blockIdx.x % p.KV;
  const SeqTile t = find_tile<256>(p.cu_k, p.nseq, p.total_k, blockIdx.x / p.KV, threadIdx.x & 63);
  if (t.row0 < 0) return;
  const int key = t.row0 + (int)threadIdx.x;
  if (key >= t.len) return;
  int64_t qlo;
  int lenq;
  other_rows(p.cu_q, p.nseq, p.total_q, t.seq, qlo, lenq);
  float sum = 0.f;
  for (int i = 0; i < wp.parts; ++i) sum += wp.part[((int64_t)i * p.KV + e) * p.total_k + t.lo + key];
  if (wp.far > 0 && key < p.sinks && t.seq >= 0 && t.seq < p.nseq) {
    const float* from = wp.far_part + ((int64_t)t.seq * p.KV + e) * p.sinks + key;
    const int64_t step = p.nseq * p.KV * p.sinks;
    for (int i0 = 0; i0 < wp.far; i0 += 8) {  // eight on their way at a time
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = from[min(i0 + i, wp.far - 1) * step];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += i0 + i < wp.far ? x[i] : 0.f;
    }
  }
  put_weight(wp, t.seq, e, key, t.len - lenq, sum);
}

static int weights_check(const kdn_attn_weights_args* a) {
  if (!a || a->num_seqs < 0 || a->total_q < 0 || a->total_k < 0 || a->H <= 0 || a->H_kv <= 0 || a->H > (1 << 20) || a->H % a->H_kv != 0 ||
      !valid_dtype(a->dtype) || !(a->scale > 0.f) || !std::isfinite(a->scale) || a->window < 0 || a->sinks < 0 || a->places < 0 || a->num_slots < 0)
    return KDN_ERR_INVALID_ARGUMENT;
  if ((a->d != 64 && a->d != 128) || a->total_q > (1 << 30) || a->total_k > (1 << 30) || a->num_seqs > (1 << 30) || a->num_slots > INT32_MAX)
    return KDN_ERR_UNSUPPORTED;
  if ((!a->cu_k && a->total_k != a->total_q) || (!a->slots && a->num_slots < a->num_seqs)) return KDN_ERR_INVALID_ARGUMENT;
  return KDN_OK;
}

// How a call is shared out: by the kernel of few rows or by the other one, there by how many workgroups to a tile of keys, and by how
// many more to a tile with sinks.
struct WeightsPlan {
  bool few;
  int parts, far, far_tiles, long_rows;
  int window, sinks;
  explicit WeightsPlan(const kdn_attn_weights_args* a) : parts(1), far(0), far_tiles(0), long_rows(INT32_MAX) {
    AttnParams p = {};
    p.total_k = a->total_k;
    attn_window(p, a->window > 0 ? a->window : NO_WINDOW, a->sinks);
    window = p.window, sinks = p.sinks;
    const bool win = window < NO_WINDOW, bf16 = a->dtype == KDN_DTYPE_BF16;
    const int row = a->d * (int)dtype_size(a->dtype), keys = row <= 256 ? 256 : 128, rows = row <= 128 ? 128 : 64;
    const int64_t tiles = tile_slots(a->total_k, keys, a->num_seqs) * a->H_kv, G = a->H / a->H_kv;
    const int64_t each = a->total_q / std::max<int64_t>(a->num_seqs, 1);  // an average sequence's rows
    // Few rows: as long as reading K, not the products, is most of it, and there are tiles for half the CUs.  bf16, us by that kernel and
    // the other: 128 features, four heads to a key head, four prompts of 16000, their last 1, 64, 256, 512 rows 35 (54), 47 (62), 157 (163),
    // 300 (293); 64 features 18 (23), 20 (27), 59 (60).  One prompt of 8000, 64 features, 64 rows: 9 (12).  One of 500, 256 rows: 28 (13).
    // Never fp32, which waits for its products (four prompts of 16000, 64 rows 49 and 54, the other 48 and 52), and no window, which
    // leaves most keys fewer rows.
    few = bf16 && !win && tiles >= 128 && (each + 63) / 64 * G <= (a->d == 64 ? 8 : 16);
    if (few) {  // twice the average's tiles of rows
      long_rows = (int)std::min<int64_t>(128 * ((std::max<int64_t>(each, 1) + 63) / 64), INT32_MAX);
      return;
    }
    // Parts: a part costs a workgroup's start, and all of them a launch, so that there are as many as fill the CUs once, twice if each
    // has two tiles of rows left, eight times if eight (and an eighth more);
    // in bf16 a tile of a few rows is too little.  One prompt of 8000, 16 heads of 64 over 4, with 1, 4 and 16 parts: 1 row 11, 12,
    // 25; 256 rows 28, 18, 30; all rows 538, 159, 103.  Nine of 3000, 32 heads of 128 over 8: 256 rows 90, 105, 206; all rows 431, 417, 551.
    const int64_t walk = ((win ? std::min<int64_t>(each, window + keys) : each) + rows - 1) / rows * G;
    const int64_t st = (sinks + keys - 1) / keys;
    // tiles that have rows
    const int64_t busy = win ? (int64_t)std::min((double)tiles, (double)((each + window) / keys + 2 + st) * (double)a->num_seqs * (double)a->H_kv) : tiles;
    for (int n = 2; n <= 16 && each >= (bf16 ? 32 : 1); ++n)
      if ((busy * n <= 288 && walk >= (tiles * n <= 2304 ? n : 4 * n)) || (busy * n <= 576 && walk >= 2 * n) || (busy * n <= 2048 && walk >= 8 * n)) parts = n;
    if (win && sinks > 0 && each > (int64_t)window + 2 * keys && st <= 512 && a->num_seqs <= 512 && a->H_kv <= 512 && st * a->num_seqs * a->H_kv <= 512) {
      far_tiles = (int)st;
      far = (int)std::max<int64_t>(1, std::min<int64_t>({1024 / (st * a->num_seqs * a->H_kv), each / rows * G / 2, 64}));
    }
  }
};

template <class P>
static int launch_weights_few(WeightsParams p, hipStream_t st) {
  // as many workgroups as there is room for at a time, each as many tiles (twice or four times as many: 84 and 83 us for 81)
  const int64_t slots = tile_slots(p.a.total_k, WeightsFew<P>::KEYS, p.a.nseq), groups = std::max<int64_t>(1, 512 / p.a.KV);
  const int64_t per = (slots + groups - 1) / groups;
  const int64_t grid = ((slots + per - 1) / per + 7) / 8 * 8 * p.a.KV;
  const int64_t dealt = (groups + 7) / 8 * 8 * p.a.KV;
  if (std::max(grid, dealt) > max_groups(64 * WeightsFew<P>::WAVES)) return KDN_ERR_UNSUPPORTED;
  // A launch of the long sequences' own takes 2.7 us where there are none; without it the longest walk is that of a stretch whose rows
  // are all the call's, about a microsecond for each of its tiles of rows.
  const bool deal = p.a.total_q > p.long_rows && per * ((p.a.total_q + 63) / 64 * p.a.G) > 128;
  if (deal) hipLaunchKernelGGL((attn_weights_few_kernel<P, true>), dim3((unsigned)dealt), dim3(64 * WeightsFew<P>::WAVES), 0, st, p, slots, per);
  else p.long_rows = INT32_MAX;
  hipLaunchKernelGGL((attn_weights_few_kernel<P, false>), dim3((unsigned)grid), dim3(64 * WeightsFew<P>::WAVES), 0, st, p, slots, per);
  return launch_status();
}

template <class P>
static int launch_weights(const WeightsParams& p, bool few, hipStream_t st) {
  if constexpr (sizeof(typename P::elem) == 2)
    if (few) return launch_weights_few<P>(p, st);
  const int64_t slots = tile_slots(p.a.total_k, WeightsTile<P>::KEYS, p.a.nseq);
  const int64_t grid = (slots * p.parts + (p.far > 0 ? p.a.nseq * p.far_tiles * p.far : 0)) * p.a.KV;
  const int64_t joins = p.part ? tile_slots(p.a.total_k, 256, p.a.nseq) * p.a.KV : 0;
  if (std::max(grid, joins) > max_groups(256)) return KDN_ERR_UNSUPPORTED;
  if (p.a.window < NO_WINDOW) hipLaunchKernelGGL((attn_weights_kernel<P, true>), dim3((unsigned)grid), dim3(256), 0, st, p, slots);
  else hipLaunchKernelGGL((attn_weights_kernel<P, false>), dim3((unsigned)grid), dim3(256), 0, st, p, slots);
  if (joins > 0) hipLaunchKernelGGL(attn_weights_join_kernel, dim3((unsigned)joins), dim3(256), 0, st, p);
  return launch_status();
}

}  // namespace kdn

using namespace kdn;

extern "C" size_t kdn_attn_weights_workspace_bytes(const kdn_attn_weights_args* a) {
  if (weights_check(a) != KDN_OK) return 0;
  const WeightsPlan plan(a);
  if (plan.parts == 1 && plan.far == 0) return 4;
  return ((size_t)plan.parts * (size_t)a->total_k + (size_t)plan.far * (size_t)a->num_seqs * (size_t)plan.sinks) * (size_t)a->H_kv * 4;
}

extern "C" int kdn_attn_weights(const kdn_attn_weights_args* a, void* stream) {
  int rc = weights_check(a);
  if (rc != KDN_OK) return rc;
  if (a->total_k == 0 || a->num_seqs == 0) return KDN_OK;
  if (!a->cu_q || !a->k || (a->total_q > 0 && (!a->q || !a->lse)) || (a->num_slots > 0 && a->places > 0 && !a->weights)) return KDN_ERR_INVALID_ARGUMENT;
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->lse, 4) || !aligned(a->weights, 4) || !aligned(a->slots, 4) ||
      !aligned(a->workspace, 4) || !attn_strides_ok(a->q_stride, a->dtype) || !attn_strides_ok(a->k_stride, a->dtype))
    return KDN_ERR_MISALIGNED;
  if (!stage_reach(a->q_stride[0], a->dtype)) return KDN_ERR_UNSUPPORTED;
  WeightsParams p = {};
  const WeightsPlan plan(a);
  p.parts = plan.parts, p.far = plan.far, p.far_tiles = plan.far_tiles, p.long_rows = plan.long_rows;
  const bool join = plan.parts > 1 || plan.far > 0;
  if (join && (!a->workspace || a->workspace_bytes < kdn_attn_weights_workspace_bytes(a))) return KDN_ERR_WORKSPACE_TOO_SMALL;
  p.a.q = a->q; p.a.k = a->k;
  for (int i = 0; i < 2; ++i) {
    p.a.qs[i] = a->q_stride[i]; p.a.ks[i] = a->k_stride[i]; p.weights_stride[i] = a->weights_stride[i];
  }
  p.a.lse = const_cast<float*>(a->lse);
  p.a.cu_q = a->cu_q;
  p.a.cu_k = a->cu_k ? a->cu_k : a->cu_q;
  p.a.nseq = a->num_seqs; p.a.total_q = a->total_q; p.a.total_k = a->total_k;
  p.a.H = (int)a->H; p.a.KV = (int)a->H_kv; p.a.G = (int)(a->H / a->H_kv);
  p.a.scale = a->scale;
  p.a.window = plan.window, p.a.sinks = plan.sinks;
  p.weights = a->weights; p.places = a->places; p.num_slots = a->num_slots; p.slots = a->slots;
  p.part = join ? reinterpret_cast<float*>(a->workspace) : nullptr;
  p.far_part = plan.far > 0 ? p.part + (size_t)plan.parts * (size_t)a->H_kv * (size_t)a->total_k : nullptr;
  p.add = a->add != 0;
  hipStream_t st = as_stream(stream);
  const bool few = plan.few;
  if (a->dtype == KDN_DTYPE_BF16) return a->d == 64 ? launch_weights<AttnBF16<64>>(p, few, st) : launch_weights<AttnBF16<128>>(p, few, st);
  return a->d == 64 ? launch_weights<AttnF32<64>>(p, few, st) : launch_weights<AttnF32<128>>(p, few, st);
}
