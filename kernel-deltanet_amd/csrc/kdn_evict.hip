// Eviction from the pages by accumulated attention weight: of each stream, layer and key head the places of largest weight stay,
// and the kept ones behind the new length fill the given-up places before it.
//
//   select: a workgroup per (stream, layer, head).  A place's rank is 32 bits: its weight's (the order of floats that are not
//     negative is that of their bits), and above all weights the sinks and the latest tokens.  The rank of the last place that stays is
//     found by its digits from the top, 11, 11 and 10 bits: a histogram in LDS of the places that agree with the digits so
//     far, and the bin that the wanted count falls into.  Then every wave goes over its stretch of the places three times: equals
//     of that rank (the lowest of them stay), holes and fillers counted, holes and fillers listed.  32 streams, two layers, eight heads,
//     4096 to 16384 places, half kept: 48 us for 22 MB of weights read and as much of lists written: a chain of passes over LDS, with a
//     barrier after each.  144 heads of 1025 places, of which one goes: 12.6.  (The weights one load at a time: 82 for 48.)
//   move: the i-th filler's key, value go to the i-th hole.  The two lists are disjoint (fillers lie behind the new length), so that
//     the moves need no order, and no row moves that has not to.
#include <algorithm>
#include "kdn_io.hpp"
#include "kdn_internal.hpp"
#include "../../include/kdn_bounded.h"

namespace kdn {

struct EvictParams {
  unsigned char *kp, *vp;
  int64_t kps[4], vps[4];  // bytes, [page][layer][head][token]
  const int32_t *table, *lens, *keep, *settled, *evicted, *slots;
  float* weights;
  int32_t* positions;
  int64_t ws[3], ps[3];    // elements, [slot][layer][head]
  int32_t *count, *holes, *fillers;  // [unit]; [unit][room] each
  int64_t table_stride, num_pages, num_slots, max_len, room, sinks, recent;
  int layers, heads, nseq, shift, pieces;  // 16-byte pieces of a row: 1 << pieces
};

constexpr int EVICT_THREADS = 1024, EVICT_WAVES = EVICT_THREADS / 64;
constexpr int EVICT_BINS = 2048;
// Ranks kept in LDS: with the histogram 72 KB, two workgroups a CU.  Those of places behind are formed anew each time.
constexpr int EVICT_CACHED = 16384;
constexpr uint32_t RANK_SINK = 0xffffffffu, RANK_RECENT = 0xfffffffeu;

// A stream's numbers, within what the tensors hold.
struct EvictStream {
  int len, kept, settled;
  int64_t evicted, slot;
};
__device__ __forceinline__ EvictStream evict_stream(const EvictParams& p, int b) {
  EvictStream s;
  s.len = (int)min((int64_t)max(p.lens[b], 0), p.max_len);
  s.kept = min(s.len, max(p.keep[b], 0));
  s.settled = p.settled ? min(max(p.settled[b], 0), s.len) : 0;
  s.evicted = p.evicted ? max(p.evicted[b], 0) : 0;
  s.slot = p.slots ? p.slots[b] : b;
  return s;
}

__global__ void __launch_bounds__(EVICT_THREADS) evict_select_kernel(EvictParams p) {
  __shared__ uint32_t ranks[EVICT_CACHED];
  __shared__ int bins[EVICT_BINS];
  __shared__ int wave_sum[EVICT_WAVES], found[2];
  const int unit = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int e = unit % p.heads, layer = unit / p.heads % p.layers, b = unit / p.heads / p.layers;
  const EvictStream s = evict_stream(p, b);
  if (s.slot < 0 || s.slot >= p.num_slots) {
    if (tid == 0) p.count[unit] = 0;
    return;
  }
  float* weights = p.weights + s.slot * p.ws[0] + layer * p.ws[1] + e * p.ws[2];
  int32_t* positions = p.positions + s.slot * p.ps[0] + layer * p.ps[1] + e * p.ps[2];
  const int len = s.len, kept = s.kept;
  auto position = [&](int j) -> int64_t { return j < s.settled ? positions[j] : j + s.evicted; };
  if (kept == len) {
    for (int j = s.settled + tid; j < len; j += EVICT_THREADS) positions[j] = (int32_t)(j + s.evicted);
    if (tid == 0) p.count[unit] = 0;
    return;
  }
  const int64_t latest = len + s.evicted - p.recent;  // positions from here on stay if they can
  auto rank_of = [&](int64_t at, float x) -> uint32_t {
    return at < p.sinks ? RANK_SINK : at >= latest ? RANK_RECENT : x > 0.f ? __builtin_bit_cast(uint32_t, x) : 0u;
  };
  const int cached = min(len, EVICT_CACHED);
  constexpr int AHEAD = 8;  // loads on their way at a time: one by one a head's 16384 places take 25 us
  for (int j0 = tid; j0 < cached; j0 += AHEAD * EVICT_THREADS) {
    float x[AHEAD];
    int32_t at[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int j = min(j0 + i * EVICT_THREADS, cached - 1);
      x[i] = weights[j];
      at[i] = j < s.settled ? positions[j] : 0;
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int j = j0 + i * EVICT_THREADS;
      if (j < cached) ranks[j] = rank_of(j < s.settled ? at[i] : j + s.evicted, x[i]);
    }
  }
  __syncthreads();
  auto rank = [&](int j) -> uint32_t { return j < EVICT_CACHED ? ranks[j] : rank_of(position(j), weights[j]); };

  // the rank of the kept-th place, and how many of its equals stay
  uint32_t last = 0;
  int want = kept;
  if (kept > 0) {
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, size = digit == 2 ? 1024 : 2048;
      const uint32_t above = digit == 0 ? 0u : digit == 1 ? 0xffffffffu << 21 : 0xffffffffu << 10;  // the digits that are known
      for (int i = tid; i < EVICT_BINS; i += EVICT_THREADS) bins[i] = 0;
      __syncthreads();
      for (int j = tid; j < len; j += EVICT_THREADS) {
        const uint32_t r = rank(j);
        if (((r ^ last) & above) == 0) atomicAdd(&bins[(r >> shift) & (size - 1)], 1);
      }
      __syncthreads();
      // from the highest bin down: thread t has bins size - 1 - 2 t and the one below it
      const int hi = size - 1 - 2 * tid, first = hi >= 0 ? bins[hi] : 0, second = hi >= 1 ? bins[hi - 1] : 0;
      int upto = first + second;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int x = __shfl_up(upto, d);
        if (lane >= d) upto += x;
      }
      if (lane == 63) wave_sum[w] = upto;
      __syncthreads();
      int before = upto - first - second;
      for (int x = 0; x < w; ++x) before += wave_sum[x];
      if (before < want && want <= before + first + second) {  // one thread
        const bool low = want > before + first;
        found[0] = low ? hi - 1 : hi;
        found[1] = want - before - (low ? first : 0);
      }
      __syncthreads();
      last |= (uint32_t)found[0] << shift;
      want = found[1];
      __syncthreads();
    }
  } else {
    last = 0xffffffffu;  // nothing stays
  }

  // a wave's stretch of the places, 64 at a time
  const int each = (len + EVICT_THREADS - 1) / EVICT_THREADS * 64, begin = min(w * each, len), end = min(begin + each, len);
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  auto sums_before = [&](int mine) {  // of the waves before this one
    __syncthreads();
    if (lane == 0) wave_sum[w] = mine;
    __syncthreads();
    int sum = 0;
    for (int x = 0; x < w; ++x) sum += wave_sum[x];
    return sum;
  };
  int equals = 0;
  for (int j = begin; j < end; j += 64) equals += __popcll(__ballot(j + lane < end && rank(min(j + lane, len - 1)) == last));
  const int first_equal = sums_before(equals);
  auto walk = [&](auto visit) {
    int seen = first_equal;
    for (int j = begin; j < end; j += 64) {
      const int at = j + lane;
      const uint32_t r = rank(min(at, len - 1));
      const uint64_t same = __ballot(at < end && r == last);
      const bool stays = at < end && (r > last || (r == last && seen + __popcll(same & below) < want));
      seen += __popcll(same);
      visit(at, stays, __ballot(at < end && at < kept && !stays), __ballot(stays && at >= kept));
    }
  };
  int nholes = 0, nfillers = 0;
  walk([&](int, bool, uint64_t hole, uint64_t filler) {
    nholes += __popcll(hole);
    nfillers += __popcll(filler);
  });
  int hole_at = sums_before(nholes), filler_at = sums_before(nfillers);
  int32_t *holes = p.holes + unit * p.room, *fillers = p.fillers + unit * p.room;
  walk([&](int at, bool stays, uint64_t hole, uint64_t filler) {
    const int to = hole_at + __popcll(hole & below), from = filler_at + __popcll(filler & below);
    if ((hole >> lane & 1) && to < p.room) holes[to] = at;
    if ((filler >> lane & 1) && from < p.room) fillers[from] = at;
    if (stays && at < kept && at >= s.settled) positions[at] = (int32_t)(at + s.evicted);
    hole_at += __popcll(hole);
    filler_at += __popcll(filler);
  });
  __syncthreads();
  if (w == EVICT_WAVES - 1 && lane == 0) {
    // as many fillers as holes; should another writer change weights meanwhile, still as many as both lists hold
    found[0] = (int)min((int64_t)min(hole_at, filler_at), p.room);
    p.count[unit] = found[0];
  }
  __syncthreads();
  const int moves = found[0];
  for (int i0 = tid; i0 < moves; i0 += 4 * EVICT_THREADS) {
    int from[4], to[4];
    float x[4];
    int32_t at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = min(i0 + i * EVICT_THREADS, moves - 1);
      from[i] = fillers[m], to[i] = holes[m];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = weights[from[i]];
      at[i] = (int32_t)position(from[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i0 + i * EVICT_THREADS < moves) weights[to[i]] = x[i], positions[to[i]] = at[i];
  }
}

// Sixteen bytes of a row a lane, rows of keys and of values in turn, two on their way at a time; none of them soon read again:
// nontemporal.  Of 32 streams' 16 heads of 4096 to 16384 places half kept, 256-byte rows, 1.29 GB read and written: 315 us, 4.1 TB/s
// (a large copy 4.9); with four rows at a time 354, eight 793, with plain loads and stores two 331.
constexpr int MOVE_ROWS = 2;
__global__ void __launch_bounds__(256) evict_move_kernel(EvictParams p, int blocks, int first_unit) {
  const int unit = first_unit + blockIdx.x / blocks, block = blockIdx.x % blocks;
  const int lanes = 1 << p.pieces, piece = threadIdx.x & (lanes - 1), row = threadIdx.x >> p.pieces, rows = 256 >> p.pieces;
  const int n = 2 * p.count[unit], first = block * rows * MOVE_ROWS + row;
  if (block * rows * MOVE_ROWS >= n) return;
  const int e = unit % p.heads, layer = unit / p.heads % p.layers, b = unit / p.heads / p.layers;
  const int32_t *holes = p.holes + unit * p.room, *fillers = p.fillers + unit * p.room, *table = p.table + b * p.table_stride;
  auto at = [&](int place, bool v) {
    const int64_t* s = v ? p.vps : p.kps;
    const int64_t page = min(max((int64_t)table[place >> p.shift], (int64_t)0), p.num_pages - 1);  // a number outside the pool is its nearest page's
    return reinterpret_cast<u32x4*>((v ? p.vp : p.kp) + page * s[0] + layer * s[1] + e * s[2] + (int64_t)(place & ((1 << p.shift) - 1)) * s[3]) + piece;
  };
  u32x4 x[MOVE_ROWS];
#pragma unroll
  for (int i = 0; i < MOVE_ROWS; ++i) {
    const int r = first + i * rows;
    if (r < n) x[i] = __builtin_nontemporal_load(at(fillers[r >> 1], r & 1));
  }
#pragma unroll
  for (int i = 0; i < MOVE_ROWS; ++i) {
    const int r = first + i * rows;
    if (r < n) __builtin_nontemporal_store(x[i], at(holes[r >> 1], r & 1));
  }
}

static int evict_check(const kdn_evict_args* a) {
  if (!a || a->num_seqs < 0 || a->layers <= 0 || a->H_kv <= 0 || !valid_dtype(a->dtype) || a->page_tokens <= 0 || a->num_pages < 0 ||
      a->table_width < 0 || a->max_len < 0 || a->places < 0 || a->num_slots < 0 || a->sinks < 0 || a->recent < 0)
    return KDN_ERR_INVALID_ARGUMENT;
  if ((a->d != 64 && a->d != 128) || a->page_tokens < 16 || (a->page_tokens & (a->page_tokens - 1)) != 0 || a->page_tokens > (1 << 30) ||
      a->num_seqs > INT32_MAX || a->layers > (1 << 20) || a->H_kv > (1 << 20) || a->num_pages > INT32_MAX || a->num_slots > INT32_MAX ||
      a->max_len > (1 << 30))
    return KDN_ERR_UNSUPPORTED;
  if (a->max_len > 0 && (a->num_pages == 0 || (a->max_len + a->page_tokens - 1) / a->page_tokens > a->table_width || a->max_len > a->places))
    return KDN_ERR_INVALID_ARGUMENT;
  if (!a->slots && a->num_slots < a->num_seqs) return KDN_ERR_INVALID_ARGUMENT;
  int64_t units;
  if (__builtin_mul_overflow(a->layers * a->H_kv, a->num_seqs, &units) || units > max_groups(EVICT_THREADS)) return KDN_ERR_UNSUPPORTED;
  return KDN_OK;
}

// No more moves than half the places: fillers are kept and holes are not, and both are as many.
static int64_t evict_room(const kdn_evict_args* a) { return (a->max_len / 2 + 3) / 4 * 4; }
static int64_t evict_units(const kdn_evict_args* a) { return a->num_seqs * a->layers * a->H_kv; }

}  // namespace kdn

using namespace kdn;

extern "C" size_t kdn_evict_workspace_bytes(const kdn_evict_args* a) {
  if (evict_check(a) != KDN_OK) return 0;
  return (size_t)evict_units(a) * 4 * (1 + 2 * (size_t)evict_room(a)) + 16;
}

extern "C" int kdn_evict(const kdn_evict_args* a, void* stream) {
  int rc = evict_check(a);
  if (rc != KDN_OK) return rc;
  if (a->num_seqs == 0 || a->max_len == 0 || a->num_slots == 0) return KDN_OK;
  if (!a->lens || !a->keep || !a->page_table || !a->k_pages || !a->v_pages || !a->weights || !a->positions) return KDN_ERR_INVALID_ARGUMENT;
  if (!a->workspace || a->workspace_bytes < kdn_evict_workspace_bytes(a)) return KDN_ERR_WORKSPACE_TOO_SMALL;
  const int64_t size = (int64_t)dtype_size(a->dtype);
  EvictParams p = {};
  bool fits = aligned(a->k_pages, 16) && aligned(a->v_pages, 16) && aligned(a->workspace, 16) && aligned(a->weights, 4) && aligned(a->positions, 4);
  for (int i = 0; i < 4; ++i) {
    p.kps[i] = a->k_pages_stride[i] * size; p.vps[i] = a->v_pages_stride[i] * size;
    fits = fits && p.kps[i] % 16 == 0 && p.vps[i] % 16 == 0;
  }
  if (!fits) return KDN_ERR_MISALIGNED;
  // rows, weights and positions that lie on one another would be written more than once, in no order
  const int64_t sizes[4] = {a->num_pages, a->layers, a->H_kv, a->page_tokens}, slots[3] = {a->num_slots, a->layers, a->H_kv};
  for (int i = 0; i < 4; ++i)
    if (sizes[i] > 1 && (a->k_pages_stride[i] == 0 || a->v_pages_stride[i] == 0)) return KDN_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 3; ++i)
    if (slots[i] > 1 && (a->weights_stride[i] == 0 || a->positions_stride[i] == 0)) return KDN_ERR_INVALID_ARGUMENT;
  p.kp = (unsigned char*)a->k_pages; p.vp = (unsigned char*)a->v_pages;
  p.table = a->page_table; p.lens = a->lens; p.keep = a->keep; p.settled = a->settled; p.evicted = a->evicted; p.slots = a->slots;
  p.weights = a->weights; p.positions = a->positions;
  for (int i = 0; i < 3; ++i) {
    p.ws[i] = a->weights_stride[i]; p.ps[i] = a->positions_stride[i];
  }
  const int64_t units = evict_units(a);
  p.room = evict_room(a);
  p.holes = reinterpret_cast<int32_t*>(a->workspace);
  p.fillers = p.holes + units * p.room;
  p.count = p.fillers + units * p.room;
  p.table_stride = a->table_stride; p.num_pages = a->num_pages; p.num_slots = a->num_slots; p.max_len = a->max_len;
  p.sinks = a->sinks; p.recent = a->recent;
  p.layers = (int)a->layers; p.heads = (int)a->H_kv; p.nseq = (int)a->num_seqs;
  p.shift = __builtin_ctz((unsigned)a->page_tokens);
  p.pieces = __builtin_ctz((unsigned)(a->d * size / 16));
  const int rows = (256 >> p.pieces) * MOVE_ROWS;
  const int64_t blocks = (2 * (a->max_len / 2) + rows - 1) / rows;
  const int64_t most = max_groups(256);
  if (blocks > most) return KDN_ERR_UNSUPPORTED;
  hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)units), dim3(EVICT_THREADS), 0, st, p);
  if ((rc = launch_status()) != KDN_OK || blocks == 0) return rc;
  for (int64_t first = 0, n; first < units && rc == KDN_OK; first += n) {  // 64 streams of 32 layers, eight heads and 32768 places are more than one grid
    n = std::min(most / blocks, units - first);
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)(blocks * n)), dim3(256), 0, st, p, (int)blocks, (int)first);
    rc = launch_status();
  }
  return rc;
}
