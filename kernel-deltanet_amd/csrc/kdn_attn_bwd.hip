// Causal attention over packed sequences: the backward.
//
//   p_ij = exp(scale q_i.k_j - lse_i),  delta_i = dy_i . y_i,  ds_ij = p_ij (dy_i.v_j - delta_i),
//   dv_j = sum_i p_ij dy_i,  dk_j = scale sum_i ds_ij q_i,  dq_i = scale sum_j ds_ij k_j,
// with the sums over i of a key head running over all query heads that share it.
//
// Three kernels: delta; dk and dv, a workgroup per 128 keys of a key head walking the query rows that see them; dq, a
// workgroup per 128 query rows of a head walking its keys.  The scores are formed twice (seven products for the five that
// one pass with atomic sums of dq would take): every sum then has one owner and one order, so that the gradients are the
// same bits every time.  As in the forward a product's accumulator is the next one's B operand in registers.
#include "kdn_attn_tile.hpp"

namespace kdn {

constexpr int BWD_ROWS = 128, BWD_TILE = 64;

// delta: sixteen lanes a row, eight values each at a time.
template <class P>
__global__ void __launch_bounds__(256) attn_delta_kernel(AttnParams p, float* delta) {
  typedef typename P::elem E;
  const int64_t at = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);  // (row, head), heads fastest
  const int j = threadIdx.x & 15;
  if (at >= p.total_q * p.H) return;
  const int64_t row = at / p.H, h = at % p.H;
  const E* y = reinterpret_cast<const E*>(p.y) + row * p.ys[0] + h * p.ys[1];
  const E* dy = reinterpret_cast<const E*>(p.dy) + row * p.dys[0] + h * p.dys[1];
  float sum = 0.f;
  if (8 * j < P::D) {
    const typename P::frag a = P::load(y + 8 * j), b = P::load(dy + 8 * j);
#pragma unroll
    for (int s = 0; s < 8; ++s) sum = __builtin_fmaf((float)a[s], (float)b[s], sum);
  }
  sum += xor_shuffle<1>(sum);
  sum += xor_shuffle<2>(sum);
  sum += xor_shuffle<4>(sum);
  sum += xor_shuffle<8>(sum);
  if (j == 0) delta[h * p.total_q + row] = sum;
}

// dk, dv of 128 keys: a wave owns 32 keys (a lane one), their K and V fragments and the transposed sums in registers.
// The query rows pass in tiles of 64 with their lse and delta; S = Q K^T and dP = dY V^T have the queries in registers,
// so that P and dS are the B operands of dV^T += dY^T P and dK^T += Q^T dS.
template <class P>
__global__ void __launch_bounds__(256, sizeof(typename P::elem) == 2 && P::D == 64 ? 2 : 1)
    attn_dkdv_kernel(AttnParams p, int64_t slots) {
  typedef typename P::elem E;
  constexpr int D = P::D, KS = D / 16, CT = D / 32, TILE = BWD_TILE * P::ROW;
  constexpr int SLOT = 2 * TILE + 2 * BWD_TILE * 4;  // Q and dY rows, their lse and delta
  constexpr int NBUF = 2 * SLOT <= 160 * 1024 ? 2 : 1;
  __shared__ __attribute__((aligned(256))) unsigned char lds[NBUF * SLOT];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = blockIdx.x;
  const int e = (int)(id % p.KV);
  const SeqTile t = find_tile<BWD_ROWS>(p.cu_k, p.nseq, p.total_k, id / p.KV, lane);
  if (t.row0 < 0) return;
  const int64_t lenk = t.len;
  int64_t qlo, lenq;
  other_rows(p.cu_q, p.nseq, p.total_q, t.seq, qlo, lenq);
  const int64_t off = lenk - lenq;
  const int key = t.row0 + 32 * w + (lane & 31);
  const bool live = key < lenk;
  typename P::frag k[KS], v[KS];
  {
    const int64_t at = t.lo + min((int64_t)key, lenk - 1);
    const E* ksrc = reinterpret_cast<const E*>(p.k) + at * p.ks[0] + (int64_t)e * p.ks[1];
    const E* vsrc = reinterpret_cast<const E*>(p.v) + at * p.vs[0] + (int64_t)e * p.vs[1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      k[ks] = P::load(ksrc + 16 * ks + 8 * half);
      v[ks] = P::load(vsrc + 16 * ks + 8 * half);
    }
  }
  f32x16 dk[CT], dv[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) dk[ct] = dv[ct] = zero16();
  const float c = p.scale * LOG2E;

  // the query tiles that see key row0: rows from row0 - off on, of each head of the group
  const int64_t q0 = max(t.row0 - off, (int64_t)0) / BWD_TILE * BWD_TILE;
  const int per = q0 < lenq ? (int)((lenq - q0 + BWD_TILE - 1) / BWD_TILE) : 0;
  const int ntiles = per * p.G;
  auto stage = [&](int j, unsigned char* to) {
    const int h = e * p.G + j / per;
    const int64_t r0 = q0 + (int64_t)(j % per) * BWD_TILE;
    const int last = (int)min(lenq - 1 - r0, (int64_t)BWD_TILE - 1);
    const E* qb = reinterpret_cast<const E*>(p.q) + (qlo + r0) * p.qs[0] + (int64_t)h * p.qs[1];
    const E* yb = reinterpret_cast<const E*>(p.dy) + (qlo + r0) * p.dys[0] + (int64_t)h * p.dys[1];
    stage_rows<P, BWD_TILE, 4>(qb, p.qs[0], last, to, w, lane);
    stage_rows<P, BWD_TILE, 4>(yb, p.dys[0], last, to + TILE, w, lane);
    if (w < 2) {
      const float* src = (w == 0 ? p.lse : p.delta) + (int64_t)h * p.total_q + qlo + r0 + min(lane, last);
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const void*>(src),
                                       (__attribute__((address_space(3))) void*)(to + 2 * TILE + w * BWD_TILE * 4), 4, 0, 0);
    }
  };
  // as in the forward: the next tile's copies and this one's reads do not overlap
  auto step = [&](int j, const unsigned char* __restrict qt, unsigned char* __restrict next) {
    if (NBUF == 2 && j + 1 < ntiles) stage(j + 1, next);
    const int64_t r0 = q0 + (int64_t)(j % per) * BWD_TILE;
    const unsigned char *yt = qt + TILE, *stat = qt + 2 * TILE;
#pragma unroll(sizeof(E) == 2 ? 2 : 1)
    for (int u = 0; u < BWD_TILE / 32; ++u) {
      const int64_t i0 = r0 + 32 * u;  // rows i0 .. i0 + 31
      if (i0 >= lenq || i0 + 31 + off < t.row0 + 32 * w) continue;  // none of them sees a key of this wave
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = P::mma(s, P::row_frag(qt, 32 * u + (lane & 31), ks, half), k[ks]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) dp = P::mma(dp, P::row_frag(yt, 32 * u + (lane & 31), ks, half), v[ks]);
      const bool whole = i0 + off >= t.row0 + 32 * w + 31 && i0 + 32 <= lenq;
      const int64_t first = max((int64_t)key - off, (int64_t)0) - i0;  // rows of the tile from `first` to `end` see the key
      const int lo = (int)min(first, (int64_t)32), hi = (int)min(lenq - i0, (int64_t)32);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const f32x4 ls = *reinterpret_cast<const f32x4*>(stat + 4 * (32 * u + 8 * a + 4 * half));
        const f32x4 de = *reinterpret_cast<const f32x4*>(stat + 4 * (BWD_TILE + 32 * u + 8 * a + 4 * half));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = 4 * a + x, r = rho(half, i);
          float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -ls[x] * LOG2E));
          float d = pr * (dp[i] - de[x]);
          if (!whole) {
            const bool sees = r >= lo && r < hi;
            pr = sees ? pr : 0.f;
            d = sees ? d : 0.f;
          }
          s[i] = pr;
          dp[i] = d;
        }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const typename P::frag pf = P::from_acc(s, m), df = P::from_acc(dp, m);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          dv[ct] = P::mma(dv[ct], P::col_frag(yt, 32 * u + 16 * m, ct, lane), pf);
          dk[ct] = P::mma(dk[ct], P::col_frag(qt, 32 * u + 16 * m, ct, lane), df);
        }
      }
    }
  };
  if (NBUF == 2 && ntiles > 0) stage(0, lds);
  for (int j = 0; j < ntiles; ++j) {
    if (NBUF == 1) {
      staged_barrier();
      stage(j, lds);
    }
    staged_barrier();
    if constexpr (NBUF == 2) step(j, lds + (j & 1) * SLOT, lds + (~j & 1) * SLOT);
    else step(j, lds, lds);
  }
  E* dkr = reinterpret_cast<E*>(p.dk) + (t.lo + key) * p.dks[0] + (int64_t)e * p.dks[1];
  E* dvr = reinterpret_cast<E*>(p.dv) + (t.lo + key) * p.dvs[0] + (int64_t)e * p.dvs[1];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    store_row32(dkr + 32 * ct, dk[ct], p.scale, half, live);
    store_row32(dvr + 32 * ct, dv[ct], 1.f, half, live);
  }
}

// dq of 128 query rows of a head: the forward's walk over the keys with S^T = K Q^T and dP^T = V dY^T, and
// dQ^T += K^T dS^T.
template <class P>
__global__ void __launch_bounds__(256, sizeof(typename P::elem) == 2 ? 2 : 1) attn_dq_kernel(AttnParams p, int64_t slots) {
  typedef typename P::elem E;
  constexpr int D = P::D, KS = D / 16, CT = D / 32, TILE = BWD_TILE * P::ROW;
  __shared__ __attribute__((aligned(256))) unsigned char lds[4 * TILE];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t id = blockIdx.x;
  int h;
  if (p.H % 8 == 0) {
    const int per = p.H / 8;
    h = (int)(id % 8) * per + (int)(id / 8 % per);
  } else {
    h = (int)(id % p.H);
  }
  const SeqTile t = find_tile<BWD_ROWS>(p.cu_q, p.nseq, p.total_q, slots - 1 - id / p.H, lane);
  if (t.row0 < 0) return;
  const int64_t lenq = t.len;
  int64_t klo, lenk;
  other_rows(p.cu_k, p.nseq, p.total_k, t.seq, klo, lenk);
  const int64_t off = lenk - lenq;
  const int row = t.row0 + 32 * w + (lane & 31);
  const bool live = row < lenq;
  const int64_t at = t.lo + min((int64_t)row, lenq - 1);
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
  const float ls = p.lse[(int64_t)h * p.total_q + at] * LOG2E, de = p.delta[(int64_t)h * p.total_q + at];
  f32x16 dq[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) dq[ct] = zero16();

  const int64_t sees = min(lenk, t.row0 + BWD_ROWS + off);
  const int ntiles = sees > 0 ? (int)((sees + BWD_TILE - 1) / BWD_TILE) : 0;
  const int64_t wfirst = t.row0 + 32 * w + off, wlast = wfirst + 31;
  auto stage = [&](int j, unsigned char* to) {
    const int64_t k0 = (int64_t)j * BWD_TILE;
    const int last = (int)min(lenk - 1 - k0, (int64_t)BWD_TILE - 1);
    stage_rows<P, BWD_TILE, 4>(kb + k0 * p.ks[0], p.ks[0], last, to, w, lane);
    stage_rows<P, BWD_TILE, 4>(vb + k0 * p.vs[0], p.vs[0], last, to + TILE, w, lane);
  };
  auto step = [&](int j, const unsigned char* __restrict kt, unsigned char* __restrict next) {
    if (j + 1 < ntiles) stage(j + 1, next);
    const int64_t k0 = (int64_t)j * BWD_TILE;
    const unsigned char* vt = kt + TILE;
#pragma unroll
    for (int u = 0; u < BWD_TILE / 32; ++u) {
      const int64_t j0 = k0 + 32 * u;
      if (j0 > wlast || j0 >= lenk) continue;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = P::mma(s, P::row_frag(kt, 32 * u + (lane & 31), ks, half), q[ks]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) dp = P::mma(dp, P::row_frag(vt, 32 * u + (lane & 31), ks, half), dy[ks]);
      const bool whole = j0 + 31 <= wfirst;
      const int limit = (int)min(max((int64_t)row + off - j0, (int64_t)-1), (int64_t)32);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float d = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -ls)) * (dp[i] - de);
        if (!whole) d = rho(half, i) <= limit ? d : 0.f;
        dp[i] = d;
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const typename P::frag df = P::from_acc(dp, m);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) dq[ct] = P::mma(dq[ct], P::col_frag(kt, 32 * u + 16 * m, ct, lane), df);
      }
    }
  };
  if (ntiles > 0) stage(0, lds);
  for (int j = 0; j < ntiles; ++j) {
    staged_barrier();
    step(j, lds + (j & 1) * 2 * TILE, lds + (~j & 1) * 2 * TILE);
  }
  E* dst = reinterpret_cast<E*>(p.dq) + (t.lo + row) * p.dqs[0] + (int64_t)h * p.dqs[1];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) store_row32(dst + 32 * ct, dq[ct], p.scale, half, live);
}

template <class P>
static int launch_bwd(const AttnParams& p, float* delta, hipStream_t st) {
  const int64_t rows = p.total_q * p.H;
  const int64_t kslots = p.total_k / BWD_ROWS + p.nseq + 1, qslots = p.total_q / BWD_ROWS + p.nseq + 1;
  if ((rows + 15) / 16 > INT32_MAX || kslots * p.KV > INT32_MAX || qslots * p.H > INT32_MAX) return KDN_ERR_UNSUPPORTED;
  if (p.total_q > 0)
    hipLaunchKernelGGL(attn_delta_kernel<P>, dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, p, delta);
  if (p.total_k > 0)
    hipLaunchKernelGGL(attn_dkdv_kernel<P>, dim3((unsigned)(kslots * p.KV)), dim3(256), 0, st, p, kslots);
  if (p.total_q > 0)
    hipLaunchKernelGGL(attn_dq_kernel<P>, dim3((unsigned)(qslots * p.H)), dim3(256), 0, st, p, qslots);
  return launch_status();
}

}  // namespace kdn

using namespace kdn;

extern "C" size_t kdn_attn_bwd_workspace_bytes(const kdn_attn_bwd_args* a) {
  if (!a || attn_check(a->fwd) != KDN_OK) return 0;
  const size_t bytes = (size_t)a->fwd->H * (size_t)a->fwd->total_q * 4;
  return bytes < 16 ? 16 : bytes;
}

extern "C" int kdn_attn_bwd(const kdn_attn_bwd_args* a, void* stream) {
  if (!a) return KDN_ERR_INVALID_ARGUMENT;
  const kdn_attn_args* f = a->fwd;
  int rc = attn_check(f);
  if (rc != KDN_OK) return rc;
  if (f->total_q == 0 && f->total_k == 0) return KDN_OK;
  if (f->total_q > 0) {
    if ((rc = attn_check_tensors(f)) != KDN_OK) return rc;
    if (!f->lse || !a->dy || !a->dq || !a->workspace) return KDN_ERR_INVALID_ARGUMENT;
  }
  if (!f->cu_q || (f->total_k > 0 && (!f->k || !f->v || !a->dk || !a->dv))) return KDN_ERR_INVALID_ARGUMENT;
  if (!aligned(a->dy, 16) || !aligned(a->dq, 16) || !aligned(a->dk, 16) || !aligned(a->dv, 16) || !aligned(a->workspace, 16) ||
      !attn_strides_ok(a->dy_stride, f->dtype) || !attn_strides_ok(a->dq_stride, f->dtype) ||
      !attn_strides_ok(a->dk_stride, f->dtype) || !attn_strides_ok(a->dv_stride, f->dtype) ||
      !attn_strides_ok(f->k_stride, f->dtype) || !attn_strides_ok(f->v_stride, f->dtype) || !aligned(f->k, 16) || !aligned(f->v, 16))
    return KDN_ERR_MISALIGNED;
  if (f->total_q > 0 && a->workspace_bytes < kdn_attn_bwd_workspace_bytes(a)) return KDN_ERR_WORKSPACE_TOO_SMALL;
  AttnParams p = attn_params(f);
  p.dy = a->dy; p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
  p.delta = reinterpret_cast<const float*>(a->workspace);
  for (int i = 0; i < 2; ++i) {
    p.dys[i] = a->dy_stride[i]; p.dqs[i] = a->dq_stride[i]; p.dks[i] = a->dk_stride[i]; p.dvs[i] = a->dv_stride[i];
  }
  float* delta = reinterpret_cast<float*>(a->workspace);
  hipStream_t st = as_stream(stream);
  if (f->dtype == KDN_DTYPE_BF16)
    return f->d == 64 ? launch_bwd<AttnBF16<64>>(p, delta, st) : launch_bwd<AttnBF16<128>>(p, delta, st);
  return f->d == 64 ? launch_bwd<AttnF32<64>>(p, delta, st) : launch_bwd<AttnF32<128>>(p, delta, st);
}
