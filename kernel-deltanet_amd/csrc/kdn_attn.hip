// Causal attention over packed sequences with grouped heads: the forward.
//
//   y_i = sum_j p_ij v_j / l_i,  p_ij = exp(scale q_i.k_j - m_i),  m_i = max_j, l_i = sum_j p_ij,  j <= i + len_k - len_q.
//
// One pass over the keys with a running maximum and sum.  A workgroup owns 128 query rows of one head, a wave 32 of them;
// tiles of 64 keys pass through LDS (two slots, copied by the load unit while the other is used).  The products are
// transposed, S^T = K Q^T and Y^T = V^T P^T: a query is a lane, its scores are 32 of the lane's registers, so the row
// maximum and sum are register arithmetic and one exchange between the halves of the wave, and P^T is the B operand of
// the second product as it lies (kdn_attn_tile.hpp).
#include <cmath>
#include "kdn_attn_tile.hpp"

namespace kdn {

// What bounds it: a block of 32 rows and 32 keys at 128 features is 512 cycles of products and about 450 of softmax, and two
// waves a SIMD overlap them in part.  One sequence of 16384 rows, 32 heads of 128 in bf16: 1.97 to 2.08 ms by card, 1.06 to
// 1.12 PFLOP/s, where a product of 16384-wide matrices reaches 1.35; the matrix cores are busy in 55 % of the cycles, at 1.6 GHz,
// which the load holds the clock to (2.4 at most); no LDS bank conflicts.  Seven prompts of 33 to 2048 rows, 16 heads of 64:
// 32 us.  fp32, 4096 rows, 32 heads of 128: 1.2 to 1.3 ms, 105 to 114 TFLOP/s of 150; matrix cores busy 72 %.
//   The walk over the keys is one chain, so that a batch with few rows takes the time of its longest row, however idle the
// GPU: then SPLIT waves share 32 rows and take every SPLIT-th block of 32 keys of a tile each, and their sums meet at the end
// (attn_split has the rule).
template <class P, int SPLIT>
struct Fwd {
  static constexpr int ROWS = 128 / SPLIT, KEYS = SPLIT == 4 ? 128 : 64, BLOCKS = KEYS / 32 / SPLIT;
  static constexpr int TILE = KEYS * P::ROW, BUFS = 4 * TILE <= 128 * 1024 ? 2 : 1;
  static constexpr int JOIN = SPLIT > 1 ? 4 * (P::D / 32) * 4096 + 4 * 64 * 8 : 0;
  static constexpr int LDS = 2 * BUFS * TILE > JOIN ? 2 * BUFS * TILE : JOIN;
};

template <class P, int SPLIT>
__global__ void __launch_bounds__(256, sizeof(typename P::elem) == 2 ? 2 : 1) attn_fwd_kernel(AttnParams p, int64_t slots) {
  typedef typename P::elem E;
  typedef Fwd<P, SPLIT> S;
  constexpr int KS = P::D / 16, CT = P::D / 32, KEYS = S::KEYS, TILE = S::TILE;
  __shared__ __attribute__((aligned(256))) unsigned char lds[S::LDS];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = w % SPLIT;
  // an XCD's heads next to one another, so that its L2 holds their keys
  int64_t id = blockIdx.x;
  int h;
  if (p.H % 8 == 0) {
    const int per = p.H / 8;
    h = (int)(id % 8) * per + (int)(id / 8 % per);
  } else {
    h = (int)(id % p.H);
  }
  const SeqTile t = find_heavy<S::ROWS, false>(p.cu_q, p.nseq, p.total_q, id / p.H, slots, lane);
  if (t.row0 < 0) return;
  const int lenq = t.len;
  int64_t klo;
  int lenk;
  other_rows(p.cu_k, p.nseq, p.total_k, t.seq, klo, lenk);
  const int off = lenk - lenq;  // query i sees keys 0 .. i + off
  const int first_row = t.row0 + 32 * (w / SPLIT), row = first_row + (lane & 31);
  const bool live = row < lenq;
  const E* kb = reinterpret_cast<const E*>(p.k) + klo * p.ks[0] + (int64_t)(h / p.G) * p.ks[1];
  const E* vb = reinterpret_cast<const E*>(p.v) + klo * p.vs[0] + (int64_t)(h / p.G) * p.vs[1];

  typename P::frag q[KS];
  {
    const E* src = reinterpret_cast<const E*>(p.q) + (t.lo + min(row, lenq - 1)) * p.qs[0] + (int64_t)h * p.qs[1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = P::load(src + 16 * ks + 8 * half);
  }
  f32x16 o[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) o[ct] = zero16();
  float m = -INFINITY, l = 0.f;
  const float c = p.scale * LOG2E;

  const int sees = min(lenk, t.row0 + S::ROWS + off);  // keys that any row of the workgroup sees
  const int ntiles = sees > 0 ? (sees + KEYS - 1) / KEYS : 0;
  const int wfirst = first_row + off, wlast = wfirst + 31;  // last key the wave's first / last row sees
  const Stager<P, KEYS, 4> stage_k(p.ks[0], w, lane), stage_v(p.vs[0], w, lane);
  auto stage = [&](int j, unsigned char* to) {
    const int k0 = j * KEYS, last = min(lenk - 1 - k0, KEYS - 1);
    stage_k(kb + k0 * p.ks[0], last, to);
    stage_v(vb + k0 * p.vs[0], last, to + TILE);
  };
  // One tile, read from `kt`, while the next one's copies go to `next`.  That the two do not overlap is said to the compiler
  // (__restrict): it would wait for the copies before it reads V otherwise.
  auto step = [&](int j, const unsigned char* __restrict kt, unsigned char* __restrict next) {
    if (S::BUFS == 2 && j + 1 < ntiles) stage(j + 1, next);
    const int r0 = 32 * S::BLOCKS * part, k0 = j * KEYS + r0;  // the wave's keys of the tile
    if (k0 > wlast) return;  // nothing of this tile is visible to the wave
    const unsigned char* vt = kt + TILE;
    f32x16 s[S::BLOCKS];
#pragma unroll
    for (int b = 0; b < S::BLOCKS; ++b) s[b] = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int b = 0; b < S::BLOCKS; ++b) s[b] = P::mma(s[b], P::row_frag(kt, r0 + 32 * b + (lane & 31), ks, half), q[ks]);
    sched_products<P, KS * S::BLOCKS, P::ROW_READS>();
    if (k0 + 32 * S::BLOCKS - 1 > wfirst) {
      const int limit = row + off - k0;
#pragma unroll
      for (int b = 0; b < S::BLOCKS; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = 32 * b + rho(half, i) <= limit ? s[b][i] : -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < S::BLOCKS; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    top = half_max(top);
    // the maximum moves only where it grows by more than 2^6 (the sums stay far inside fp32): most tiles rescale nothing
    if (__any((top - m) * c > 6.f || (m == -INFINITY && top > m))) {
      const float next_m = fmaxf(m, top);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - next_m) * c);
      m = next_m;
      l *= f;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[ct][i] *= f;
    }
    const float mc = m == -INFINITY ? 0.f : m * c;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < S::BLOCKS; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], c, -mc));
        sum += s[b][i];
      }
    l += sum;
#pragma unroll
    for (int kk = 0; kk < 2 * S::BLOCKS; ++kk) {
      const typename P::frag pf = P::from_acc(s[kk >> 1], kk & 1);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[ct] = P::mma(o[ct], P::col_frag(vt, r0 + 16 * kk, ct, lane), pf);
    }
    sched_products<P, 2 * S::BLOCKS * CT, P::COL_READS>();
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
  // A weight of zero times an infinity or NaN is no number: a tile that a row sees in part would give it what a key that it
  // does not see holds.  Where the sums are not all numbers, the workgroup goes over its tiles once more, slowly and with
  // the maxima known: V's numbers alone, weighted; then for each sum a count of the infinities, minus infinities and NaNs of
  // seen keys.  (Selecting V's values in the loop itself costs its registers: 237 for 164 at 64 features, two waves for three.)
  bool odd = false;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int i = 0; i < 16; ++i) odd |= !(__builtin_fabsf(o[ct][i]) < INFINITY);
  __syncthreads();
  int* flag = reinterpret_cast<int*>(lds);
  if (lane == 0) flag[w] = 0;
  if (live && odd) flag[w] = 1;  // (a wave's LDS accesses are in order)
  __syncthreads();
  const bool again = __builtin_amdgcn_readfirstlane(flag[0] | flag[1] | flag[2] | flag[3]);
  if (again) {
    const float mc = m == -INFINITY ? 0.f : m * c;
    const E* src = reinterpret_cast<const E*>(p.q) + (t.lo + min(row, lenq - 1)) * p.qs[0] + (int64_t)h * p.qs[1];
    f32x16 sum[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] = zero16();
#pragma unroll 1
    for (int kind = 0; kind <= 3; ++kind) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) sum[ct] = zero16();
#pragma unroll 1
      for (int j = 0; j < ntiles; ++j) {
        __syncthreads();
        stage(j, lds);
        staged_barrier();
#pragma unroll 1
        for (int b = 0; b < S::BLOCKS; ++b) {
          const int r0 = 32 * (S::BLOCKS * part + b), limit = row + off - (j * KEYS + r0);  // keys of the block that the row sees
          f32x16 x = zero16();
#pragma unroll 1
          for (int ks = 0; ks < KS; ++ks) x = P::mma(x, P::row_frag(lds, r0 + (lane & 31), ks, half), P::load(src + 16 * ks + 8 * half));
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const bool sees = rho(half, i) <= limit;
            x[i] = !sees ? 0.f : kind == 0 ? __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c, -mc)) : 1.f;
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const typename P::frag xf = P::from_acc(x, u);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
              const typename P::frag v = P::col_frag(lds + TILE, r0 + 16 * u, ct, lane);
              typename P::frag is;
#pragma unroll
              for (int e = 0; e < 8; ++e) is[e] = P::is_kind(v, e, kind) ? (kind == 0 ? v[e] : (E)1.f) : (E)0.f;
              sum[ct] = P::mma(sum[ct], is, xf);
            }
          }
        }
      }
      const float value = kind == 1 ? INFINITY : kind == 2 ? -INFINITY : NAN;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[ct][i] += kind == 0 ? sum[ct][i] : sum[ct][i] > 0.f ? value : 0.f;
    }
  }
  l = half_sum(l);
  E* dst = reinterpret_cast<E*>(p.out) + (t.lo + row) * p.ys[0] + (int64_t)h * p.ys[1];
  E* low = p.low ? reinterpret_cast<E*>(p.low) + (t.lo + row) * p.lows[0] + (int64_t)h * p.lows[1] : nullptr;
  auto ends = [&](int ct, const f32x16& v, float f) {
    store_row32(dst + 32 * ct, v, f, half, live);
    if (sizeof(E) == 2 && low) {
      f32x16 rest;
#pragma unroll
      for (int i = 0; i < 16; ++i) rest[i] = v[i] * f - (float)(E)(v[i] * f);
      store_row32(low + 32 * ct, rest, 1.f, half, live);
    }
  };
  if constexpr (SPLIT == 1) {
    const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) ends(ct, o[ct], f);
  } else {
    float* stat = reinterpret_cast<float*>(lds + 4 * CT * 4096);  // each wave's maxima and sums
    __syncthreads();
    stat[w * 64 + lane] = m;
    stat[256 + w * 64 + lane] = l;
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int x = 0; x < SPLIT; ++x) top = fmaxf(top, stat[(w - part + x) * 64 + lane]);
#pragma unroll
    for (int x = 0; x < SPLIT; ++x) {
      const float mx = stat[(w - part + x) * 64 + lane];
      sum += mx == -INFINITY ? 0.f : stat[256 + (w - part + x) * 64 + lane] * __builtin_amdgcn_exp2f((mx - top) * c);
    }
    const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - top) * c), f = sum == 0.f ? 0.f : 1.f / sum;
    join_sums<SPLIT>(o, mine, lds, w, lane, [&](int ct, const f32x16& v) { ends(ct, v, f); });
    m = top;
    l = sum;
  }
  if (p.lse && live && half == 0 && part == 0) p.lse[(int64_t)h * p.total_q + t.lo + row] = l == 0.f ? -INFINITY : m * p.scale + logf(l);
}

bool attn_strides_ok(const int64_t s[2], int dtype) {
  const int64_t per = 16 / (int64_t)dtype_size(dtype);
  return s[0] % per == 0 && s[1] % per == 0 && s[0] >= 0 && s[1] >= 0;
}

int attn_check(const kdn_attn_args* a) {
  if (!a || a->num_seqs < 0 || a->total_q < 0 || a->total_k < 0 || a->H <= 0 || a->H_kv <= 0 || a->H > (1 << 20) ||
      a->H % a->H_kv != 0 || !valid_dtype(a->dtype) || !(a->scale > 0.f) || !std::isfinite(a->scale))
    return KDN_ERR_INVALID_ARGUMENT;
  if (a->d != 64 && a->d != 128) return KDN_ERR_UNSUPPORTED;
  if (a->total_q > (1 << 30) || a->total_k > (1 << 30) || a->num_seqs > (1 << 30)) return KDN_ERR_UNSUPPORTED;
  if (!a->cu_k && a->total_k != a->total_q) return KDN_ERR_INVALID_ARGUMENT;
  return KDN_OK;
}

int attn_check_tensors(const kdn_attn_args* a) {
  if (!a->cu_q || !a->q || !a->y) return KDN_ERR_INVALID_ARGUMENT;
  if (a->total_k > 0 && (!a->k || !a->v)) return KDN_ERR_INVALID_ARGUMENT;
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->y, 16) || !aligned(a->y_low, 16) || !aligned(a->lse, 4) ||
      !attn_strides_ok(a->q_stride, a->dtype) || !attn_strides_ok(a->k_stride, a->dtype) ||
      !attn_strides_ok(a->v_stride, a->dtype) || !attn_strides_ok(a->y_stride, a->dtype) ||
      (a->y_low && !attn_strides_ok(a->y_low_stride, a->dtype)))
    return KDN_ERR_MISALIGNED;
  if (!stage_reach(a->q_stride[0], a->dtype) || !stage_reach(a->k_stride[0], a->dtype) || !stage_reach(a->v_stride[0], a->dtype))
    return KDN_ERR_UNSUPPORTED;
  return KDN_OK;
}

// Two workgroups on each of the 256 CUs: fewer tiles of 128 rows than that leave CUs idle, twice that are two rounds.  Two is
// what bf16 has with one or two waves to a row; with four at 128 features, and in fp32, registers or LDS allow one (fp32 of 64
// features with two waves, forward: two), and the rule has not been measured for them between 128 and 2048 tiles.
// Measured, four / two / one wave to a row: three sequences of 101 to 1024 rows, 4 heads, fp32, gradients 53 / - / 158 us;
// seven of 33 to 2048, 16 heads, bf16 56 / 33 / 39 us; one of 16384, 32 heads 5880 / 2560 / 2106 us.
int attn_split(int64_t rows, int64_t heads) {
  const int64_t tiles = rows / 128 * heads;
  return tiles < 512 ? 4 : tiles < 1024 ? 2 : 1;
}

AttnParams attn_params(const kdn_attn_args* a) {
  AttnParams p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.y = a->y; p.out = a->y;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; p.ys[i] = a->y_stride[i];
  }
  p.low = a->y_low;
  for (int i = 0; i < 2; ++i) p.lows[i] = a->y_low_stride[i];
  p.lse = a->lse;
  p.cu_q = a->cu_q;
  p.cu_k = a->cu_k ? a->cu_k : a->cu_q;
  p.nseq = a->num_seqs; p.total_q = a->total_q; p.total_k = a->total_k;
  p.H = (int)a->H; p.KV = (int)a->H_kv; p.G = (int)(a->H / a->H_kv);
  p.scale = a->scale;
  return p;
}

}  // namespace kdn

using namespace kdn;

extern "C" int kdn_anchor_version(void) { return 1 << 16; }

template <class P, int SPLIT>
static int launch_fwd(const AttnParams& p, hipStream_t st) {
  const int64_t slots = tile_slots(p.total_q, Fwd<P, SPLIT>::ROWS, p.nseq), grid = slots * p.H;
  if (grid > INT32_MAX) return KDN_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((attn_fwd_kernel<P, SPLIT>), dim3((unsigned)grid), dim3(256), 0, st, p, slots);
  return launch_status();
}

template <class P>
static int launch_fwd(const AttnParams& p, hipStream_t st) {
  switch (attn_split(p.total_q, p.H)) {
    case 4: return launch_fwd<P, 4>(p, st);
    case 2: return launch_fwd<P, 2>(p, st);
    default: return launch_fwd<P, 1>(p, st);
  }
}

extern "C" int kdn_attn_fwd(const kdn_attn_args* a, void* stream) {
  int rc = attn_check(a);
  if (rc != KDN_OK) return rc;
  if (a->total_q == 0) return KDN_OK;
  if ((rc = attn_check_tensors(a)) != KDN_OK) return rc;
  const AttnParams p = attn_params(a);
  hipStream_t st = as_stream(stream);
  if (a->dtype == KDN_DTYPE_BF16) return a->d == 64 ? launch_fwd<AttnBF16<64>>(p, st) : launch_fwd<AttnBF16<128>>(p, st);
  return a->d == 64 ? launch_fwd<AttnF32<64>>(p, st) : launch_fwd<AttnF32<128>>(p, st);
}
