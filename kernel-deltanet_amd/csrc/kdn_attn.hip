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

constexpr int FWD_ROWS = 128, FWD_KEYS = 64, FWD_BLOCKS = FWD_KEYS / 32;

template <class P>
__global__ void __launch_bounds__(256, sizeof(typename P::elem) == 2 ? 2 : 1) attn_fwd_kernel(AttnParams p, int64_t slots) {
  typedef typename P::elem E;
  constexpr int D = P::D, KS = D / 16, CT = D / 32, TILE = FWD_KEYS * P::ROW;
  __shared__ __attribute__((aligned(256))) unsigned char lds[4 * TILE];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the last tiles (the longest rows) first, and an XCD's heads next to one another so that its L2 holds their keys
  int64_t id = blockIdx.x;
  int h;
  if (p.H % 8 == 0) {
    const int per = p.H / 8;
    h = (int)(id % 8) * per + (int)(id / 8 % per);
  } else {
    h = (int)(id % p.H);
  }
  const int64_t slot = slots - 1 - id / p.H;
  const SeqTile t = find_tile<FWD_ROWS>(p.cu_q, p.nseq, p.total_q, slot, lane);
  if (t.row0 < 0) return;
  const int64_t lenq = t.len;
  int64_t klo, lenk;
  other_rows(p.cu_k, p.nseq, p.total_k, t.seq, klo, lenk);
  const int64_t off = lenk - lenq;  // query i sees keys 0 .. i + off
  const int row = t.row0 + 32 * w + (lane & 31);
  const bool live = row < lenq;
  const E* kb = reinterpret_cast<const E*>(p.k) + klo * p.ks[0] + (int64_t)(h / p.G) * p.ks[1];
  const E* vb = reinterpret_cast<const E*>(p.v) + klo * p.vs[0] + (int64_t)(h / p.G) * p.vs[1];

  typename P::frag q[KS];
  {
    const E* src = reinterpret_cast<const E*>(p.q) + (t.lo + min((int64_t)row, lenq - 1)) * p.qs[0] + (int64_t)h * p.qs[1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = P::load(src + 16 * ks + 8 * half);
  }
  f32x16 o[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) o[ct] = zero16();
  float m = -INFINITY, l = 0.f;
  const float c = p.scale * LOG2E;

  const int64_t sees = min(lenk, t.row0 + FWD_ROWS + off);  // keys that any row of the workgroup sees
  const int ntiles = sees > 0 ? (int)((sees + FWD_KEYS - 1) / FWD_KEYS) : 0;
  const int64_t wfirst = t.row0 + 32 * w + off, wlast = wfirst + 31;  // last key the wave's first / last row sees
  auto stage = [&](int j, unsigned char* to) {
    const int64_t k0 = (int64_t)j * FWD_KEYS;
    const int last = (int)min(lenk - 1 - k0, (int64_t)FWD_KEYS - 1);
    stage_rows<P, FWD_KEYS, 4>(kb + k0 * p.ks[0], p.ks[0], last, to, w, lane);
    stage_rows<P, FWD_KEYS, 4>(vb + k0 * p.vs[0], p.vs[0], last, to + TILE, w, lane);
  };
  // One tile, read from `kt`, while the next one's copies go to `next`.  That the two do not overlap is said to the compiler
  // (__restrict): it would wait for the copies before it reads V otherwise.
  auto step = [&](int j, const unsigned char* __restrict kt, unsigned char* __restrict next) {
    if (j + 1 < ntiles) stage(j + 1, next);
    const int64_t k0 = (int64_t)j * FWD_KEYS;
    if (k0 > wlast) return;  // nothing of this tile is visible to the wave
    const unsigned char* vt = kt + TILE;
    f32x16 s[FWD_BLOCKS];
#pragma unroll
    for (int b = 0; b < FWD_BLOCKS; ++b) {
      s[b] = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[b] = P::mma(s[b], P::row_frag(kt, 32 * b + (lane & 31), ks, half), q[ks]);
    }
    if (k0 + FWD_KEYS - 1 > wfirst) {
      const int limit = (int)min(max((int64_t)row + off - k0, (int64_t)-1), (int64_t)FWD_KEYS);
#pragma unroll
      for (int b = 0; b < FWD_BLOCKS; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = 32 * b + rho(half, i) <= limit ? s[b][i] : -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < FWD_BLOCKS; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    top = half_max(top);
    // the maximum moves only where it grows by more than 2^6 (the sums stay far inside fp32): most tiles rescale nothing
    if (__any((top - m) * c > 6.f || (m == -INFINITY && top > m))) {
      const float next = fmaxf(m, top);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - next) * c);
      m = next;
      l *= f;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[ct][i] *= f;
    }
    const float mc = m == -INFINITY ? 0.f : m * c;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < FWD_BLOCKS; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], c, -mc));
        sum += s[b][i];
      }
    l += sum;
#pragma unroll
    for (int kk = 0; kk < 2 * FWD_BLOCKS; ++kk) {
      const typename P::frag pf = P::from_acc(s[kk >> 1], kk & 1);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[ct] = P::mma(o[ct], P::col_frag(vt, 16 * kk, ct, lane), pf);
    }
  };
  if (ntiles > 0) stage(0, lds);
  for (int j = 0; j < ntiles; ++j) {
    staged_barrier();
    step(j, lds + (j & 1) * 2 * TILE, lds + (~j & 1) * 2 * TILE);
  }
  l = half_sum(l);
  const float f = l == 0.f ? 0.f : 1.f / l;
  E* dst = reinterpret_cast<E*>(p.out) + (t.lo + row) * p.ys[0] + (int64_t)h * p.ys[1];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) store_row32(dst + 32 * ct, o[ct], f, half, live);
  if (p.lse && live && half == 0) p.lse[(int64_t)h * p.total_q + t.lo + row] = l == 0.f ? -INFINITY : m * p.scale + logf(l);
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
  if (a->total_q > INT32_MAX || a->total_k > INT32_MAX || a->num_seqs > INT32_MAX) return KDN_ERR_UNSUPPORTED;
  if (!a->cu_k && a->total_k != a->total_q) return KDN_ERR_INVALID_ARGUMENT;
  return KDN_OK;
}

int attn_check_tensors(const kdn_attn_args* a) {
  if (!a->cu_q || !a->q || !a->y) return KDN_ERR_INVALID_ARGUMENT;
  if (a->total_k > 0 && (!a->k || !a->v)) return KDN_ERR_INVALID_ARGUMENT;
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->y, 16) || !aligned(a->lse, 4) ||
      !attn_strides_ok(a->q_stride, a->dtype) || !attn_strides_ok(a->k_stride, a->dtype) ||
      !attn_strides_ok(a->v_stride, a->dtype) || !attn_strides_ok(a->y_stride, a->dtype))
    return KDN_ERR_MISALIGNED;
  return KDN_OK;
}

AttnParams attn_params(const kdn_attn_args* a) {
  AttnParams p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.y = a->y; p.out = a->y;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; p.ys[i] = a->y_stride[i];
  }
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

extern "C" int kdn_attn_fwd(const kdn_attn_args* a, void* stream) {
  int rc = attn_check(a);
  if (rc != KDN_OK) return rc;
  if (a->total_q == 0) return KDN_OK;
  if ((rc = attn_check_tensors(a)) != KDN_OK) return rc;
  const AttnParams p = attn_params(a);
  const int64_t slots = a->total_q / FWD_ROWS + a->num_seqs + 1, grid = slots * a->H;
  if (grid > INT32_MAX) return KDN_ERR_UNSUPPORTED;
  const dim3 g((unsigned)grid), b(256);
  hipStream_t st = as_stream(stream);
  if (a->dtype == KDN_DTYPE_BF16) {
    if (a->d == 64) hipLaunchKernelGGL(attn_fwd_kernel<AttnBF16<64>>, g, b, 0, st, p, slots);
    else hipLaunchKernelGGL(attn_fwd_kernel<AttnBF16<128>>, g, b, 0, st, p, slots);
  } else {
    if (a->d == 64) hipLaunchKernelGGL(attn_fwd_kernel<AttnF32<64>>, g, b, 0, st, p, slots);
    else hipLaunchKernelGGL(attn_fwd_kernel<AttnF32<128>>, g, b, 0, st, p, slots);
  }
  return launch_status();
}
