// Rotary positions: pair j of a head's first rotary_dim values turns by positions[token] * inv_freq[j].
//
// Memory-bound: every value is read and written once.  The angle of a token's pair is the same in all heads: a workgroup
// forms the sines and cosines of its tokens once, in LDS.  A position times a frequency needs more bits than fp32 has (at
// position 131072 an fp32 product is off by up to 0.004 radians): it is formed in 64 bits, reduced to a turn, and only the
// sine and cosine of the rest, within half a turn, are fp32.
//   65536 tokens of 32 + 8 heads of 128, bf16 (1.34 GB): 253 us, 5.3 TB/s, where a large copy reaches 4.9.  Nine tokens of
// 16 + 4 heads: 3.1 us, a launch's latency.
#include <cmath>
#include "kdn_io.hpp"
#include "kdn_internal.hpp"
#include "../../include/kdn_anchor.h"

namespace kdn {

struct RotaryParams {
  const int64_t* pos;
  const double* freq;
  const void *q, *k;
  void *qo, *ko;
  int64_t qs[2], ks[2], qos[2], kos[2], tokens;
  int H, heads, rot, pairs, units, inverse, per;  // pairs: rotated units of a head; units: all; per: tokens a workgroup
  float mag;
};

// One unit of V values (or two of V, one of either half): 16 bytes where the rotated part divides into them, else one.
template <class E, int V>
__device__ __forceinline__ void load_unit(const E* p, float* x) {
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    if constexpr (V == 1) x[0] = (float)p[0];
    else if constexpr (sizeof(E) == 4) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p + i);
      x[i] = a[0]; x[i + 1] = a[1]; x[i + 2] = a[2]; x[i + 3] = a[3];
    } else if (i == 0) {
      load8(p, x);
    }
  }
}
template <class E, int V>
__device__ __forceinline__ void store_unit(E* p, const float* x) {
  if constexpr (V == 1) p[0] = (E)x[0];
  else if constexpr (V == 4) store4(p, x);
  else store_row8(p, x);
}

template <class E, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryParams p) {
  extern __shared__ float turn[];  // [token][pair] cosine and sine
  const int64_t t0 = (int64_t)blockIdx.x * p.per;
  const int nt = (int)min((int64_t)p.per, p.tokens - t0), half = p.rot / 2;
  for (int i = threadIdx.x; i < nt * half; i += 256) {
    const int t = i / half, j = i % half;
    const double turns = (double)p.pos[t0 + t] * p.freq[j] * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    turn[2 * i] = c * p.mag;
    turn[2 * i + 1] = p.inverse ? -s * p.mag : s * p.mag;
  }
  __syncthreads();
  const int each = p.heads * p.units;
  for (int i = threadIdx.x; i < nt * each; i += 256) {
    const int t = i / each, r = i - t * each, h = r / p.units, u = r - h * p.units;
    const bool is_q = h < p.H;
    const int hh = is_q ? h : h - p.H;
    const E* src = is_q ? reinterpret_cast<const E*>(p.q) + (t0 + t) * p.qs[0] + hh * p.qs[1]
                        : reinterpret_cast<const E*>(p.k) + (t0 + t) * p.ks[0] + hh * p.ks[1];
    E* dst = is_q ? reinterpret_cast<E*>(p.qo) + (t0 + t) * p.qos[0] + hh * p.qos[1]
                  : reinterpret_cast<E*>(p.ko) + (t0 + t) * p.kos[0] + hh * p.kos[1];
    const float* cs = turn + 2 * t * half;
    if (u >= p.pairs) {
      const int at = p.rot + (u - p.pairs) * V;
      float x[V];
      load_unit<E, V>(src + at, x);
      store_unit<E, V>(dst + at, x);
    } else if constexpr (INTERLEAVED) {
      if constexpr (V == 1) {
        const float a = (float)src[2 * u], b = (float)src[2 * u + 1], c = cs[2 * u], s = cs[2 * u + 1];
        dst[2 * u] = (E)(a * c - b * s);
        dst[2 * u + 1] = (E)(b * c + a * s);
      } else {
        float x[V], y[V];
        load_unit<E, V>(src + V * u, x);
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float c = cs[V * u + e], s = cs[V * u + e + 1];
          y[e] = x[e] * c - x[e + 1] * s;
          y[e + 1] = x[e + 1] * c + x[e] * s;
        }
        store_unit<E, V>(dst + V * u, y);
      }
    } else {
      float a[V], b[V], x[V], y[V];
      load_unit<E, V>(src + V * u, a);
      load_unit<E, V>(src + half + V * u, b);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float c = cs[2 * (V * u + e)], s = cs[2 * (V * u + e) + 1];
        x[e] = a[e] * c - b[e] * s;
        y[e] = b[e] * c + a[e] * s;
      }
      store_unit<E, V>(dst + V * u, x);
      store_unit<E, V>(dst + half + V * u, y);
    }
  }
}

template <class E, int V>
static void launch_rotary(RotaryParams& p, int d, bool interleaved, hipStream_t st) {
  p.pairs = interleaved ? (V == 1 ? p.rot / 2 : p.rot / V) : p.rot / 2 / V;
  p.units = p.pairs + (d - p.rot) / V;
  const dim3 grid((unsigned)((p.tokens + p.per - 1) / p.per));
  const size_t lds = (size_t)p.per * p.rot * 4;
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<E, V, true>), grid, dim3(256), lds, st, p);
  else hipLaunchKernelGGL((rotary_kernel<E, V, false>), grid, dim3(256), lds, st, p);
}

}  // namespace kdn

using namespace kdn;

extern "C" int kdn_rotary(const kdn_rotary_args* a, void* stream) {
  if (!a || a->tokens < 0 || a->H <= 0 || a->H_kv < 0 || a->H > (1 << 20) || a->H_kv > (1 << 20) || !valid_dtype(a->dtype) ||
      a->rotary_dim <= 0 || a->rotary_dim % 2 != 0 || a->rotary_dim > a->d || !std::isfinite(a->magnitude))
    return KDN_ERR_INVALID_ARGUMENT;
  if ((a->d != 64 && a->d != 128) || a->tokens > INT32_MAX) return KDN_ERR_UNSUPPORTED;
  if (a->tokens == 0) return KDN_OK;
  const bool has_k = a->H_kv > 0;
  if (!a->positions || !a->inv_freq || !a->q || !a->q_out || (has_k && (!a->k || !a->k_out))) return KDN_ERR_INVALID_ARGUMENT;
  const int64_t per = 16 / (int64_t)dtype_size(a->dtype);
  bool fits = aligned(a->q, 16) && aligned(a->q_out, 16) && (!has_k || (aligned(a->k, 16) && aligned(a->k_out, 16)));
  for (int i = 0; i < 2; ++i)
    fits = fits && a->q_stride[i] % per == 0 && a->q_out_stride[i] % per == 0 &&
           (!has_k || (a->k_stride[i] % per == 0 && a->k_out_stride[i] % per == 0));
  if (!fits) return KDN_ERR_MISALIGNED;
  RotaryParams p = {};
  p.pos = a->positions; p.freq = a->inv_freq;
  p.q = a->q; p.k = a->k; p.qo = a->q_out; p.ko = a->k_out;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.qos[i] = a->q_out_stride[i]; p.kos[i] = a->k_out_stride[i];
  }
  p.tokens = a->tokens;
  p.H = (int)a->H; p.heads = (int)(a->H + a->H_kv); p.rot = a->rotary_dim; p.inverse = a->inverse != 0;
  p.mag = a->magnitude;
  p.per = a->tokens >= 8192 ? 4 : 1;
  const bool il = a->interleaved != 0;
  const bool wide = il ? a->rotary_dim % per == 0 : a->rotary_dim % (2 * per) == 0;
  hipStream_t st = as_stream(stream);
  if (a->dtype == KDN_DTYPE_BF16) {
    if (wide) launch_rotary<__bf16, 8>(p, a->d, il, st);
    else launch_rotary<__bf16, 1>(p, a->d, il, st);
  } else {
    if (wide) launch_rotary<float, 4>(p, a->d, il, st);
    else launch_rotary<float, 1>(p, a->d, il, st);
  }
  return launch_status();
}
