// Attention of each sequence's new tokens over its pages and over themselves: one token of a decode step, a run of them, or
// a tree of drafts.  Token t of a sequence sees the whole context, itself, its parent and what that sees.
//
// The keys and values are what has to be read, each once: a sequence's context is cut into chunks, a workgroup per chunk
// and key head, and the rows of all query heads that share the key head (G heads of every new token) go through the matrix
// cores together, 32 to a tile.  A chunk leaves its rows' maximum, sum and unnormalised sum of values; a second launch joins
// them in the chunks' order.  Sequences of one chunk are written at once.
//   - up to 32 rows: the waves of a workgroup share the rows and take every fourth tile of 32 keys each, through two LDS
//     slots of their own with no barrier; they meet once at the end;
//   - more: each wave has 32 rows of its own, and all read the same tiles of 64 or 32 keys, as in the prompt's kernel.
// What bounds them: few rows, HBM (one token of 224 streams, contexts of 512 to 16384, 16 heads of 128 over 4: 2.07 GB in 373 us,
// 5.5 TB/s; a large copy 4.9, a read 4.0); many, a wave's own chain of copies, products and softmax for each tile, two to a SIMD where
// 160 rows are five waves on two workgroups, and the unequal chunks' tail (16 trees of 40 drafts, contexts of 1500 to 16384, 32 heads
// over 8: 0.53 GB in 158 us, of which the join 14; matrix cores busy 16 %, CUs 75 %).
// One token of three streams, contexts of 700 to 2500, fp32: 14 us, and 5 for the join.  Of these the products take 3.4 (a wave has
// two tiles in turn, 64 products of 64 cycles each, 4 of their 32 columns in use), the rest is the chain from the chunk's number
// over its page's to the copies.  fp32 of larger sizes is bound by its products: one token of 64 streams, contexts of 512 to 16384,
// 16 heads of 128 over 4: 655 us for 1.3 GB (one wave a workgroup, two of four SIMDs idle; with heads of 64 199 us for 0.65 GB); the
// 16 trees 1315 us, matrix cores busy 30 %, one workgroup a CU.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "kdn_attn_tile.hpp"

namespace kdn {

struct TreeParams {
  const void *q, *k, *v, *kp, *vp;
  void* y;
  int64_t qs[2], ks[2], vs[2], ys[2], kps[3], vps[3];  // [token][head]; pages [page][head][token]
  const int64_t* cu;
  const int32_t *lens, *table, *parents;
  float *po, *pml;  // partial sums [sequence][key head][chunk][row][D] and maxima / sums [..][2]
  int64_t table_stride, num_pages, total, max_context;
  int H, KV, G, max_new, max_chunks, chunk, shift, nseq;
  int zero_from;  // the workgroups from this number on have tree_zero's rows
  float scale;
};

// What a workgroup works on: chunk `ch` of sequence b.
struct TreeWork {
  int64_t lo;          // first new token
  int n, c0, c1;       // new tokens; the chunk's keys
  int chunks, ctx;     // chunks of the sequence; its context
  int b, ch;           // b negative: nothing
};

__device__ __forceinline__ TreeWork tree_seq(const TreeParams& p, int b) {
  TreeWork t;
  t.lo = min(max(p.cu[b], (int64_t)0), p.total);
  t.n = (int)min(min(max(p.cu[b + 1], t.lo), p.total) - t.lo, (int64_t)p.max_new);
  t.ctx = (int)min((int64_t)max(p.lens[b], 0), p.max_context);
  t.chunks = t.n > 0 ? max(1, (t.ctx + p.chunk - 1) / p.chunk) : 0;
  return t;
}

// Lane `at`'s value (`at` the same in all lanes), as a scalar.
__device__ __forceinline__ int lane_value(int v, int at) { return __builtin_amdgcn_readlane(v, __builtin_amdgcn_readfirstlane(at)); }

// The u-th chunk of all the sequences' chunks, one sequence's after another's.  The grid is sized from the longest context
// that the host allows for; the chunks that are there come first in it and the rest of the grid ends at once.  (Numbered by
// sequence and place, the workgroups without a chunk came between the others, each holding a CU for its start: 16 trees
// over 6000 tokens took 244 us, the CUs two thirds busy.)  Every lane counts the chunks of its share of the sequences, 64
// shares make a prefix sum, and the share that has chunk u is looked through in the same way.
__device__ __forceinline__ TreeWork tree_work(const TreeParams& p, int u, int lane) {
  TreeWork mine = {};
  int first = 0, n = p.nseq;  // the sequences still in question
  for (;;) {
    const int share = (n + 63) / 64, begin = first + min(lane * share, n), end = first + min(lane * share + share, n);
    int count = 0;
    for (int b = begin; b < end; ++b) {
      mine = tree_seq(p, b);
      count += mine.chunks;
    }
    int upto = count;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const int x = __shfl_up(upto, s);
      if (lane >= s) upto += x;
    }
    const int at = __popcll(__ballot(upto <= u));  // shares that lie wholly before chunk u
    if (at == 64) {
      mine.b = -1;
      return mine;
    }
    u -= lane_value(upto - count, at);
    first = lane_value(begin, at);
    n = lane_value(end, at) - first;
    if (share > 1) continue;
    TreeWork t;
    t.b = first;
    t.ch = u;
    t.lo = (int64_t)lane_value((int)(mine.lo >> 32), at) << 32 | (uint32_t)lane_value((int)mine.lo, at);
    t.n = lane_value(mine.n, at);
    t.ctx = lane_value(mine.ctx, at);
    t.chunks = lane_value(mine.chunks, at);
    t.c0 = t.ch * p.chunk;
    t.c1 = min(t.c0 + p.chunk, t.ctx);
    return t;
  }
}

// Rows of y that no token within the bounds has, as zeros: those before the first sequence and behind the last (a step padded to
// a fixed size), and those past max_new of a sequence.  The last ZERO_GROUPS workgroups of the grid: the first two kinds all of
// them share, of the third, which no step should have, a wave writes what it finds.
constexpr int ZERO_GROUPS = 16;
template <class E, int D>
__device__ __forceinline__ void tree_zero(const TreeParams& p, int group) {
  constexpr int PIECES = D * (int)sizeof(E) / 16;
  const int lane = threadIdx.x & 63, waves = ZERO_GROUPS * (blockDim.x / 64), wave = group * (blockDim.x / 64) + threadIdx.x / 64;
  auto start = [&](int64_t b) { return min(max(p.cu[b], (int64_t)0), p.total); };
  auto rows = [&](int64_t from, int64_t to, int64_t first, int64_t step) {
    for (int64_t i = first; i < (to - from) * p.H * PIECES; i += step) {
      const int64_t row = i / PIECES, t = from + row / p.H, h = row % p.H;
      *reinterpret_cast<u32x4*>(reinterpret_cast<E*>(p.y) + t * p.ys[0] + h * p.ys[1] + i % PIECES * (16 / (int)sizeof(E))) = u32x4{0, 0, 0, 0};
    }
  };
  rows(0, p.nseq > 0 ? start(0) : p.total, 64 * wave + lane, 64 * waves);
  if (p.nseq > 0) rows(start(p.nseq), p.total, 64 * wave + lane, 64 * waves);
  for (int64_t b0 = 64 * wave; b0 < p.nseq; b0 += 64 * waves) {
    const int64_t b = min(b0 + lane, (int64_t)p.nseq - 1), lo = start(b) + p.max_new, hi = start(b + 1);
    for (uint64_t over = __ballot(b0 + lane < p.nseq && hi > lo); over; over &= over - 1) {
      const int64_t at = b0 + __builtin_ctzll(over);
      rows(start(at) + p.max_new, start(at + 1), lane, 64);
    }
  }
}

// Bit u of a token's mask: it sees new token u.  Lane t of a wave has token t's; doubling along the parents, six steps for
// up to 64 tokens.  A parent that is not an earlier token of the sequence hangs the token on the context alone.
__device__ __forceinline__ uint64_t ancestors(const TreeParams& p, const TreeWork& t, int lane) {
  if (!p.parents) return lane >= 63 ? ~0ull : (2ull << lane) - 1;
  int up = lane < t.n ? p.parents[t.lo + lane] : -1;
  if (up < 0 || up >= lane) up = -1;
  uint64_t sees = 1ull << lane;
#pragma unroll
  for (int step = 0; step < 6; ++step) {
    const int from = up < 0 ? lane : up;
    const uint32_t lo = __shfl((uint32_t)sees, from), hi = __shfl((uint32_t)(sees >> 32), from);
    const int next = __shfl(up, from);
    sees |= (uint64_t)hi << 32 | lo;
    up = up < 0 ? -1 : next;
  }
  return sees;
}

// Sixteen keys (or values) into rows 16 g .. of an LDS tile: row r from base + min(r, last) * row_bytes, the base the same
// in all lanes, so that a copy takes one 32-bit offset a lane.
template <class P>
__device__ __forceinline__ void stage_group(const unsigned char* base, uint32_t row_bytes, int last, unsigned char* tile, int g, int lane) {
  constexpr int N = 16 * P::PIECES / 64, RPI = 64 / P::PIECES;
  const __amdgpu_buffer_rsrc_t from = buffer_at(base);
  // the offsets are formed here: kept from one tile to the next they take registers that the products need
  asm volatile("" : "+s"(row_bytes), "+v"(lane));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int row = i * RPI + lane / P::PIECES, piece = (lane % P::PIECES) ^ piece_swizzle<P::PIECES>(row);
    copy16_to_lds(from, (uint32_t)min(row, last) * row_bytes + 16 * piece, 0, tile + (g * N + i) * 1024);
  }
}

// Which sixteen keys a group has: its own, or where none of them is there, the last ones that are; `last` the last of them.
struct Group {
  int key, last;
};
__device__ __forceinline__ Group key_group(int key, int last_key) {
  Group g;
  g.key = key <= last_key ? key : last_key & ~15;
  g.last = min(last_key - g.key, 15);
  return g;
}
// The page number of a key, as the table has it: it is used (stage_paged) a tile later, and anything done to it here would
// wait for it here.
__device__ __forceinline__ int page_of(const TreeParams& p, int b, int key) {
  typedef const __attribute__((address_space(4))) int32_t* Table;  // nothing writes it meanwhile: scalar loads
  return ((Table)(p.table + (int64_t)b * p.table_stride))[__builtin_amdgcn_readfirstlane(key >> p.shift)];
}
// A group's keys (or with `v` its values) from the pages, or from the new tokens' own tensor, into group `at` of a tile.
template <class P>
__device__ __forceinline__ void stage_paged(const TreeParams& p, int page, int e, Group g, bool v, unsigned char* tile, int at, int lane) {
  constexpr int64_t S = sizeof(typename P::elem);
  const int off = g.key & ((1 << p.shift) - 1);
  page = min(max(page, 0), (int)p.num_pages - 1);  // a number outside the pool is its nearest page's
  const int64_t* s = v ? p.vps : p.kps;
  stage_group<P>(reinterpret_cast<const unsigned char*>(v ? p.vp : p.kp) + S * (page * s[0] + e * s[1] + off * s[2]), (uint32_t)(S * s[2]), g.last,
                 tile, at, lane);
}
template <class P>
__device__ __forceinline__ void stage_new(const TreeParams& p, int64_t lo, int e, Group g, bool v, unsigned char* tile, int at, int lane) {
  constexpr int64_t S = sizeof(typename P::elem);
  const int64_t* s = v ? p.vs : p.ks;
  stage_group<P>(reinterpret_cast<const unsigned char*>(v ? p.v : p.k) + S * ((lo + g.key) * s[0] + e * s[1]), (uint32_t)(S * s[0]), g.last, tile,
                 at, lane);
}

// The same of sixteen keys that are all there: where a lane's copies come from behind the first key, formed once.  (Formed for each
// tile they were half of the vector instructions: 16 trees of drafts 170 us, 157 with these.)
template <class P>
struct WholeGroup {
  static constexpr int N = 16 * P::PIECES / 64, RPI = 64 / P::PIECES;
  uint32_t from[N];
  __device__ __forceinline__ WholeGroup(int64_t stride, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = i * RPI + lane / P::PIECES, piece = (lane % P::PIECES) ^ piece_swizzle<P::PIECES>(r);
      from[i] = (uint32_t)(r * sizeof(typename P::elem)) * (uint32_t)stride + 16 * piece;
    }
  }
  __device__ __forceinline__ void operator()(const TreeParams& p, int page, int e, int key, bool v, unsigned char* tile, int g) const {
    const int off = key & ((1 << p.shift) - 1), pg = min(max(page, 0), (int)p.num_pages - 1);
    const int64_t* s = v ? p.vps : p.kps;
    const __amdgpu_buffer_rsrc_t rows = buffer_at(reinterpret_cast<const unsigned char*>(v ? p.vp : p.kp) +
                                                  (int64_t)sizeof(typename P::elem) * (pg * s[0] + e * s[1] + off * s[2]));
#pragma unroll
    for (int i = 0; i < N; ++i) copy16_to_lds(rows, from[i], 0, tile + (g * N + i) * 1024);
  }
};

// The running softmax of one 32-row tile over 32 N more keys: scores -> weights in `s`, the sums rescaled where the maximum
// moved (by more than 2^6, as in the prompt's kernel).
template <int N, int CT>
__device__ __forceinline__ void softmax_step(f32x16 (&s)[N], float& m, float& l, f32x16 (&o)[CT], float c) {
  float top = s[0][0];
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
  top = half_max(top);
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
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], c, -mc));
      l += s[u][i];
    }
}

template <class P>
struct TreeFew {
  static constexpr int STAGE = 2 * 32 * P::ROW;          // 32 keys and their values
  static constexpr int WAVES = 65536 / (2 * STAGE);      // two workgroups a CU: one starts or ends while the other reads
  static constexpr int LDS = WAVES * 2 * STAGE;
  static constexpr int PITCH = P::D + 4;
  static_assert(STAGE == 8192 || STAGE == 16384 || STAGE == 32768, "the waits below count the copies of one stage");
  static_assert(WAVES * 32 * PITCH * 4 <= LDS, "the waves' sums meet in the stages' place");
};

template <class P>
__global__ void __launch_bounds__(64 * TreeFew<P>::WAVES) tree_few_kernel(TreeParams p) {
  typedef typename P::elem E;
  constexpr int D = P::D, KS = D / 16, CT = D / 32, W = TreeFew<P>::WAVES, STAGE = TreeFew<P>::STAGE;
  __shared__ __attribute__((aligned(256))) unsigned char lds[TreeFew<P>::LDS + 2 * W * 32 * 4];
  float(*wm)[32] = reinterpret_cast<float(*)[32]>(lds + TreeFew<P>::LDS), (*wl)[32] = wm + W;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= p.zero_from) return tree_zero<E, D>(p, blockIdx.x - p.zero_from);
  const int e = blockIdx.x % p.KV;  // the key heads of a chunk next to one another: they go round the XCDs
  const TreeWork t = tree_work(p, blockIdx.x / p.KV, lane);
  if (t.b < 0) return;
  const int b = t.b, ch = t.ch, be = b * p.KV + e;
  const int rows = t.n * p.G, row = min(lane & 31, rows - 1), tok = row / p.G, h = e * p.G + row % p.G;
  const bool drafts = ch == t.chunks - 1;  // the last chunk has the new tokens too
  const int nt = t.c1 > t.c0 ? (t.c1 - t.c0 + 31) / 32 : 0, total = nt + (drafts ? 1 : 0);
  unsigned char* mine = lds + w * 2 * STAGE;
  // the pages of a tile's two groups, known a tile ahead of its copies
  int page0 = 0, page1 = 0;
  auto pages = [&](int at) {
    if (at >= nt) return;
    page0 = page_of(p, b, key_group(t.c0 + 32 * at, t.c1 - 1).key);
    page1 = page_of(p, b, key_group(t.c0 + 32 * at + 16, t.c1 - 1).key);
  };
  auto stage_drafts = [&](unsigned char* to) {
#pragma unroll
    for (int x = 0; x < 4; ++x)
      stage_new<P>(p, t.lo, e, key_group(16 * (x & 1), t.n - 1), x >> 1, to + (x >> 1) * STAGE / 2, x & 1, lane);
  };
  const WholeGroup<P> whole_k(p.kps[2], lane), whole_v(p.vps[2], lane);
  const int full = (t.c1 - t.c0) / 32;
  auto stage = [&](int at, unsigned char* to) {
    if (at < full) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
        (x >> 1 ? whole_v : whole_k)(p, x & 1 ? page1 : page0, e, t.c0 + 32 * at + 16 * (x & 1), x >> 1, to + (x >> 1) * STAGE / 2, x & 1);
      return;
    }
    if (at >= nt) return stage_drafts(to);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      stage_paged<P>(p, x & 1 ? page1 : page0, e, key_group(t.c0 + 32 * at + 16 * (x & 1), t.c1 - 1), x >> 1, to + (x >> 1) * STAGE / 2, x & 1, lane);
  };
  pages(w);
  if (w < total) stage(w, mine);
  pages(w + W);
  uint64_t sees = 0;
  if (drafts) {
    const uint64_t all = ancestors(p, t, lane);
    sees = (uint64_t)__shfl((uint32_t)(all >> 32), tok) << 32 | __shfl((uint32_t)all, tok);
  }
  typename P::frag q[KS];
  {
    const E* src = reinterpret_cast<const E*>(p.q) + (t.lo + tok) * p.qs[0] + (int64_t)h * p.qs[1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = P::load(src + 16 * ks + 8 * half);
  }
  f32x16 o[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) o[ct] = zero16();
  float m = -INFINITY, l = 0.f;
  const float c = p.scale * LOG2E;
  // one tile, read from `kt` while the next one's copies go to `next` (as in the prompt's kernel);
  // `whole`: of the context, all 32 keys of it there
  auto step = [&](auto whole, int at, const unsigned char* __restrict kt, unsigned char* __restrict next) {
    if (at + W < total) {
      if constexpr (whole.value) {
        stage(at + W, next);
        pages(at + 2 * W);
      } else {
        stage_drafts(next);
      }
      // everything but the last STAGE / 1024 copies, the next tile's, has arrived
      if constexpr (STAGE == 8192) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      else if constexpr (STAGE == 16384) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(32)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const unsigned char* vt = kt + STAGE / 2;
    f32x16 s[1] = {zero16()};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s[0] = P::mma(s[0], P::row_frag(kt, lane & 31, ks, half), q[ks]);
    sched_products<P, KS, P::ROW_READS>();
    uint32_t bits = ~0u;  // the keys of the tile that the row sees
    if constexpr (!whole.value) {
      bits = at >= nt ? (uint32_t)sees : (uint32_t)((1ull << (t.c1 - t.c0 - 32 * at)) - 1);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[0][i] = bits >> rho(half, i) & 1 ? s[0][i] : -INFINITY;
    }
    softmax_step<1>(s, m, l, o, c);
    if constexpr (whole.value) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const typename P::frag pf = P::from_acc(s[0], kk);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) o[ct] = P::mma(o[ct], P::col_frag(vt, 16 * kk, ct, lane), pf);
      }
      sched_products<P, 2 * CT, P::COL_READS>();
    } else {
      masked_values<P, 2>(o, vt, 0, lane, s, [&](int x) { return bits >> x & 1; });
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile is read: its slot may be written again
  };
  int at = w, buf = 0;
  for (; at < full; at += W, buf ^= 1) step(std::true_type{}, at, mine + buf * STAGE, mine + (buf ^ 1) * STAGE);
#pragma unroll 1
  for (; at < total; at += W, buf ^= 1) step(std::false_type{}, at, mine + buf * STAGE, mine + (buf ^ 1) * STAGE);
  // the waves' sums, each scaled to the common maximum, added in the waves' order
  l = half_sum(l);
  if (half == 0) wm[w][lane] = m, wl[w][lane] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int x = 0; x < W; ++x) top = fmaxf(top, wm[x][lane & 31]);
  const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - top) * c);
  constexpr int PITCH = TreeFew<P>::PITCH;
  float* ob = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 x = {o[ct][4 * a] * f, o[ct][4 * a + 1] * f, o[ct][4 * a + 2] * f, o[ct][4 * a + 3] * f};
      *reinterpret_cast<f32x4*>(ob + (w * 32 + (lane & 31)) * PITCH + 32 * ct + 8 * a + 4 * half) = x;
    }
#pragma unroll
  for (int x = 0; x < W; ++x)
    sum += wm[x][lane & 31] == -INFINITY ? 0.f : wl[x][lane & 31] * __builtin_amdgcn_exp2f((wm[x][lane & 31] - top) * c);
  __syncthreads();
  if (w == 0 && half == 0) wl[0][lane] = sum, wm[0][lane] = top;
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (D / 4); i += 64 * W) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    f32x4 x = *reinterpret_cast<const f32x4*>(ob + r * PITCH + d);
#pragma unroll
    for (int y = 1; y < W; ++y) x += *reinterpret_cast<const f32x4*>(ob + (y * 32 + r) * PITCH + d);
    if (t.chunks == 1) {
      const float g = wl[0][r] == 0.f ? 0.f : 1.f / wl[0][r];
      float out[4] = {x[0] * g, x[1] * g, x[2] * g, x[3] * g};
      E* dst = reinterpret_cast<E*>(p.y) + (t.lo + r / p.G) * p.ys[0] + (int64_t)(e * p.G + r % p.G) * p.ys[1] + d;
      if constexpr (sizeof(E) == 2) {
        const bf16x4 v = {(__bf16)out[0], (__bf16)out[1], (__bf16)out[2], (__bf16)out[3]};
        *reinterpret_cast<bf16x4*>(dst) = v;
      } else {
        *reinterpret_cast<f32x4*>(dst) = f32x4{out[0], out[1], out[2], out[3]};
      }
    } else {
      const int64_t at = ((int64_t)be * p.max_chunks + ch) * p.max_new * p.G + r;
      *reinterpret_cast<f32x4*>(p.po + at * D + d) = x;
      if (d == 0) p.pml[2 * at] = wm[0][r] * c, p.pml[2 * at + 1] = wl[0][r];
    }
  }
}

// More than 32 rows: workgroups of four waves, `per` of them with 32 rows each, as even as they come (160 rows: three and
// two; the others only copy).
template <class P>
struct TreeMany {
  static constexpr int KEYS = P::ROW <= 128 ? 64 : 32, TILE = KEYS * P::ROW;
  // tiles in LDS, all but the one in use on their way; two workgroups a CU, or of fp32, whose registers allow one, one
  static constexpr int BUFS = 4, COPIES = KEYS / 32 * 16 * P::PIECES / 64;  // copies of a wave and tile
  static int blocks(int rows) { return (rows + 127) / 128; }
  static int per(int rows) { return ((rows + 31) / 32 + blocks(rows) - 1) / blocks(rows); }
};

template <class P>
__global__ void __launch_bounds__(256, sizeof(typename P::elem) == 2 ? 2 : 1) tree_many_kernel(TreeParams p, int blocks, int per) {
  typedef typename P::elem E;
  constexpr int D = P::D, KS = D / 16, CT = D / 32, KEYS = TreeMany<P>::KEYS, TILE = TreeMany<P>::TILE;
  constexpr int BUFS = TreeMany<P>::BUFS, COPIES = TreeMany<P>::COPIES;
  __shared__ __attribute__((aligned(256))) unsigned char lds[2 * BUFS * TILE];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= p.zero_from) return tree_zero<E, D>(p, blockIdx.x - p.zero_from);
  // The row blocks of one chunk on one XCD, one after another: its L2 has the keys from the second on.  Which comes first
  // changes every 32 workgroups, an XCD's CUs: a CU gets its turn's larger and smaller blocks (16 trees 198 -> 186 us).
  const int at8 = blockIdx.x / 8, unit = at8 / blocks * 8 + blockIdx.x % 8, rb = (at8 + at8 / blocks * blocks / 32) % blocks;
  const int e = unit % p.KV;
  const TreeWork t = tree_work(p, unit / p.KV, lane);
  if (t.b < 0) return;
  const int b = t.b, ch = t.ch, be = b * p.KV + e;
  const int rows = t.n * p.G, first = 32 * (per * rb + w);
  if (32 * per * rb >= rows) return;
  const bool busy = w < per && first < rows, live = busy && first + (lane & 31) < rows;
  const int row = min(first + (lane & 31), rows - 1), tok = row / p.G, h = e * p.G + row % p.G;
  const bool drafts = ch == t.chunks - 1;
  const int nt = t.c1 > t.c0 ? (t.c1 - t.c0 + KEYS - 1) / KEYS : 0, total = nt + (drafts ? (t.n + KEYS - 1) / KEYS : 0);
  // of 64 keys wave w copies keys 16 w .. of each tile and their values, of 32 either; their page is known a tile ahead
  const int mine = KEYS == 64 ? w : w & 1;
  int page = 0;
  auto pages = [&](int at) {
    if (at < nt) page = page_of(p, b, key_group(t.c0 + KEYS * at + 16 * mine, t.c1 - 1).key);
  };
  const WholeGroup<P> whole_k(KEYS == 64 || w < 2 ? p.kps[2] : p.vps[2], lane), whole_v(p.vps[2], lane);
  auto stage_whole = [&](int at, unsigned char* to) {
    const int key = t.c0 + KEYS * at + 16 * mine;
    if constexpr (KEYS == 64) {
      whole_k(p, page, e, key, false, to, mine);
      whole_v(p, page, e, key, true, to + TILE, mine);
    } else {
      whole_k(p, page, e, key, w >> 1, to + (w >> 1) * TILE, mine);
    }
  };
  const int full = (t.c1 - t.c0) / KEYS;
  auto stage = [&](int at, unsigned char* to) {
    if (at < full) return stage_whole(at, to);
    const Group g = at < nt ? key_group(t.c0 + KEYS * at + 16 * mine, t.c1 - 1) : key_group(KEYS * (at - nt) + 16 * mine, t.n - 1);
    auto part = [&](bool v) {
      if (at < nt) stage_paged<P>(p, page, e, g, v, to + v * TILE, mine, lane);
      else stage_new<P>(p, t.lo, e, g, v, to + v * TILE, mine, lane);
    };
    if constexpr (KEYS == 64) part(false), part(true);
    else part(w >> 1);
  };
#pragma unroll
  for (int x = 0; x < BUFS - 1; ++x) {
    pages(x);
    if (x < total) stage(x, lds + x * 2 * TILE);
  }
  pages(BUFS - 1);
  uint64_t sees = 0;
  if (drafts) {
    const uint64_t all = ancestors(p, t, lane);
    sees = (uint64_t)__shfl((uint32_t)(all >> 32), tok) << 32 | __shfl((uint32_t)all, tok);
  }
  typename P::frag q[KS];
  {
    const E* src = reinterpret_cast<const E*>(p.q) + (t.lo + tok) * p.qs[0] + (int64_t)h * p.qs[1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = P::load(src + 16 * ks + 8 * half);
  }
  f32x16 o[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) o[ct] = zero16();
  float m = -INFINITY, l = 0.f;
  const float c = p.scale * LOG2E;
  auto step = [&](auto whole, int at, const unsigned char* __restrict kt, unsigned char* __restrict next) {
    if (at + BUFS - 1 < total) {
      stage(at + BUFS - 1, next);
      pages(at + BUFS);
    }
    if (!busy) return;
    const unsigned char* vt = kt + TILE;
    f32x16 s[KEYS / 32];
#pragma unroll
    for (int u = 0; u < KEYS / 32; ++u) s[u] = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int u = 0; u < KEYS / 32; ++u) s[u] = P::mma(s[u], P::row_frag(kt, 32 * u + (lane & 31), ks, half), q[ks]);
    sched_products<P, KEYS / 32 * KS, P::ROW_READS>();
    uint64_t bits = ~0ull;  // the keys of the tile that the row sees
    if constexpr (!whole.value) {
      bits = at >= nt ? sees >> (KEYS * (at - nt)) : (1ull << (t.c1 - t.c0 - KEYS * at)) - 1;
#pragma unroll
      for (int u = 0; u < KEYS / 32; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = (uint32_t)(bits >> (32 * u)) >> (4 * half) >> rho(0, i) & 1 ? s[u][i] : -INFINITY;
    }
    softmax_step<KEYS / 32>(s, m, l, o, c);
    if constexpr (whole.value) {
#pragma unroll
      for (int kk = 0; kk < KEYS / 16; ++kk) {
        const typename P::frag pf = P::from_acc(s[kk >> 1], kk & 1);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) o[ct] = P::mma(o[ct], P::col_frag(vt, 16 * kk, ct, lane), pf);
      }
      sched_products<P, KEYS / 16 * CT, P::COL_READS>();
    } else {
      masked_values<P, KEYS / 16>(o, vt, 0, lane, s, [&](int x) { return bits >> x & 1; });
    }
  };
  int at = 0, now = 0;
  auto turn = [&](auto whole) {
    if (at + BUFS - 2 >= total) staged_barrier();
    else staged_barrier<(BUFS - 2) * COPIES>();
    const int then = now == 0 ? BUFS - 1 : now - 1;  // the tile before: read by all
    step(whole, at, lds + now * 2 * TILE, lds + then * 2 * TILE);
    now = now == BUFS - 1 ? 0 : now + 1;
  };
  for (; at < full; ++at) turn(std::true_type{});
#pragma unroll 1
  for (; at < total; ++at) turn(std::false_type{});
  l = half_sum(l);
  if (t.chunks == 1) {
    const float f = l == 0.f ? 0.f : 1.f / l;
    E* dst = reinterpret_cast<E*>(p.y) + (t.lo + tok) * p.ys[0] + (int64_t)h * p.ys[1];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) store_row32(dst + 32 * ct, o[ct], f, half, live);
  } else {
    const int64_t at = ((int64_t)be * p.max_chunks + ch) * p.max_new * p.G + row;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) store_row32(p.po + at * D + 32 * ct, o[ct], 1.f, half, live);
    if (live && half == 0) p.pml[2 * at] = m * c, p.pml[2 * at + 1] = l;
  }
}

// The chunks of one row joined in their order: a wave a row, D / 64 values a lane.
template <class E, int D>
__global__ void __launch_bounds__(256) tree_join_kernel(TreeParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int most = p.max_new * p.G, r = (int)(id % most);
  const int64_t be = id / most;
  if (be >= (int64_t)p.nseq * p.KV) return;
  const int b = (int)(be / p.KV), e = (int)(be % p.KV);
  const TreeWork t = tree_seq(p, b);
  if (r >= t.n * p.G || t.chunks == 1) return;
  const int64_t first = be * p.max_chunks * most + r;
  float top = -INFINITY;
  for (int x = lane; x < t.chunks; x += 64) top = fmaxf(top, p.pml[2 * (first + (int64_t)x * most)]);
#pragma unroll
  for (int s = 1; s < 64; s *= 2) top = fmaxf(top, __shfl_xor(top, s));
  constexpr int V = D / 64;
  float sum = 0.f, o[V] = {};
#pragma unroll 4
  for (int x = 0; x < t.chunks; ++x) {
    const int64_t at = first + (int64_t)x * most;
    const float m = p.pml[2 * at], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    sum += p.pml[2 * at + 1] * f;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = __builtin_fmaf(p.po[at * D + V * lane + i], f, o[i]);
  }
  const float g = sum == 0.f ? 0.f : 1.f / sum;
  E* dst = reinterpret_cast<E*>(p.y) + (t.lo + r / p.G) * p.ys[0] + (int64_t)(e * p.G + r % p.G) * p.ys[1] + V * lane;
#pragma unroll
  for (int i = 0; i < V; ++i) dst[i] = (E)(o[i] * g);
}

// A product of sizes that no caller's numbers take past 64 bits.
static int64_t times(int64_t a, int64_t b) {
  int64_t r;
  return __builtin_mul_overflow(a, b, &r) ? INT64_MAX : r;
}
static int64_t tree_rows(const kdn_tree_attn_args* a) { return a->max_new * (a->H / a->H_kv); }  // to a sequence and key head
static int64_t tree_blocks(const kdn_tree_attn_args* a) { return tree_rows(a) <= 32 ? 1 : (tree_rows(a) + 127) / 128; }

constexpr int MAX_CHUNK = 2048;
// Keys of a chunk: 128 to 2048, the fewest with which the grid stays within 512 workgroups, or from 256 keys on 2048 (a
// chunk's own cost, its queries and its partial sums, is that of a few dozen keys; short chunks even out unequal contexts).
// With chunks of at most 1024 keys 16 trees of 40 drafts, contexts of 1500 to 16384, took 186 us where these took 177, one
// token of 224 streams 396 where these took 378; with up to 4096 the 224 streams took 395.
static int tree_chunk(const kdn_tree_attn_args* a) {
  const int64_t each = times(a->num_seqs * a->H_kv, tree_blocks(a));
  int chunk = 128;
  while (chunk < MAX_CHUNK && times(each, (a->max_context + chunk - 1) / chunk) > (chunk < 256 ? 512 : 2048)) chunk *= 2;
  return chunk;
}
static int64_t tree_chunks(const kdn_tree_attn_args* a) {
  const int chunk = tree_chunk(a);
  return a->max_context > 0 ? (a->max_context + chunk - 1) / chunk : 1;
}

static int tree_check(const kdn_tree_attn_args* a) {
  if (!a || a->num_seqs < 0 || a->total_new < 0 || a->H <= 0 || a->H_kv <= 0 || a->H > (1 << 20) || a->H % a->H_kv != 0 ||
      !valid_dtype(a->dtype) || !(a->scale > 0.f) || !std::isfinite(a->scale) || a->max_context < 0 ||
      a->max_new < 0 || (a->max_new == 0 && a->total_new > 0) ||
      a->page_tokens <= 0 || a->num_pages < 0 || a->table_width < 0)
    return KDN_ERR_INVALID_ARGUMENT;
  if ((a->d != 64 && a->d != 128) || a->max_new > 64 || a->page_tokens < 16 || (a->page_tokens & (a->page_tokens - 1)) != 0 ||
      a->page_tokens > (1 << 30) || a->total_new > INT32_MAX || a->num_seqs > INT32_MAX || a->num_pages > INT32_MAX ||
      a->max_context > (1 << 30))
    return KDN_ERR_UNSUPPORTED;
  if (a->max_context > 0 && (a->num_pages == 0 || (a->max_context + a->page_tokens - 1) / a->page_tokens > a->table_width))
    return KDN_ERR_INVALID_ARGUMENT;
  // a grid's workgroups, and the join's rows
  const int64_t heads = a->num_seqs * a->H_kv, blocks = tree_blocks(a);
  if (times(times(heads, tree_chunks(a)), blocks) > INT32_MAX - 8 * blocks - ZERO_GROUPS || times(heads, tree_rows(a)) > INT32_MAX)
    return KDN_ERR_UNSUPPORTED;
  return KDN_OK;
}

template <class P>
static int launch_tree(TreeParams& p, hipStream_t st) {
  const int rows = p.max_new * p.G;
  const int64_t units = (int64_t)p.nseq * p.KV * p.max_chunks;
  if (rows <= 32) {
    p.zero_from = (int)units;
    hipLaunchKernelGGL(tree_few_kernel<P>, dim3((unsigned)units + ZERO_GROUPS), dim3(64 * TreeFew<P>::WAVES), 0, st, p);
  } else {
    const int blocks = TreeMany<P>::blocks(rows);
    p.zero_from = (int)((units + 7) / 8 * 8 * blocks);
    hipLaunchKernelGGL(tree_many_kernel<P>, dim3((unsigned)p.zero_from + ZERO_GROUPS), dim3(256), 0, st, p, blocks, TreeMany<P>::per(rows));
  }
  if (p.max_chunks > 1 && p.nseq > 0) {
    const int64_t joins = (int64_t)p.nseq * p.KV * rows;
    hipLaunchKernelGGL((tree_join_kernel<typename P::elem, P::D>), dim3((unsigned)((joins + 3) / 4)), dim3(256), 0, st, p);
  }
  return launch_status();
}

}  // namespace kdn

using namespace kdn;

// Bytes of the partial sums of `units` chunks.
static size_t tree_partial_bytes(const kdn_tree_attn_args* a, int64_t units) {
  return (size_t)units * (size_t)tree_rows(a) * (size_t)(a->d + 2) * 4 + 16;
}

// Not the call's own number of chunks but a bound that grows with every size, so that a workspace for the largest call
// holds for the others: the rule for a chunk's length gives a smaller call shorter chunks, and at times more of them.
extern "C" size_t kdn_tree_attn_workspace_bytes(const kdn_tree_attn_args* a) {
  if (tree_check(a) != KDN_OK) return 0;
  const int64_t heads = a->num_seqs * a->H_kv, fine = heads * ((a->max_context + 127) / 128), coarse = heads * ((a->max_context + MAX_CHUNK - 1) / MAX_CHUNK);
  return a->max_context <= 128 ? 16 : tree_partial_bytes(a, std::min(fine, std::max<int64_t>(2048, coarse)));
}

extern "C" int kdn_tree_attn(const kdn_tree_attn_args* a, void* stream) {
  int rc = tree_check(a);
  if (rc != KDN_OK) return rc;
  if (a->total_new == 0 || (a->num_seqs == 0 && !a->y)) return KDN_OK;
  if (!a->y || (a->num_seqs > 0 && (!a->cu_new || !a->context_lens || !a->q || !a->k || !a->v ||
                                    (a->max_context > 0 && (!a->page_table || !a->k_pages || !a->v_pages)))))
    return KDN_ERR_INVALID_ARGUMENT;
  const int64_t per = 16 / (int64_t)dtype_size(a->dtype);
  bool fits = aligned(a->q, 16) && aligned(a->k, 16) && aligned(a->v, 16) && aligned(a->y, 16) && aligned(a->k_pages, 16) &&
              aligned(a->v_pages, 16) && aligned(a->workspace, 16) && attn_strides_ok(a->q_stride, a->dtype) &&
              attn_strides_ok(a->k_stride, a->dtype) && attn_strides_ok(a->v_stride, a->dtype) && attn_strides_ok(a->y_stride, a->dtype);
  for (int i = 0; i < 3; ++i)
    fits = fits && a->k_pages_stride[i] >= 0 && a->v_pages_stride[i] >= 0 && a->k_pages_stride[i] % per == 0 && a->v_pages_stride[i] % per == 0;
  if (!fits) return KDN_ERR_MISALIGNED;
  const int64_t chunks = tree_chunks(a);
  // a copy's lanes have 32-bit offsets from its first row
  const int64_t size = (int64_t)dtype_size(a->dtype), far = INT32_MAX / (16 * size);
  if (a->k_stride[0] > far || a->v_stride[0] > far || a->k_pages_stride[2] > far || a->v_pages_stride[2] > far) return KDN_ERR_UNSUPPORTED;
  if (a->num_seqs > 0 && chunks > 1 && (!a->workspace || a->workspace_bytes < tree_partial_bytes(a, a->num_seqs * a->H_kv * chunks))) return KDN_ERR_WORKSPACE_TOO_SMALL;
  TreeParams p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.kp = a->k_pages; p.vp = a->v_pages; p.y = a->y;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; p.ys[i] = a->y_stride[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.kps[i] = a->k_pages_stride[i]; p.vps[i] = a->v_pages_stride[i];
  }
  p.cu = a->cu_new; p.lens = a->context_lens; p.table = a->page_table; p.parents = a->parents;
  p.table_stride = a->table_stride; p.num_pages = a->num_pages; p.total = a->total_new; p.max_context = a->max_context;
  p.H = (int)a->H; p.KV = (int)a->H_kv; p.G = (int)(a->H / a->H_kv);
  p.max_new = (int)a->max_new; p.max_chunks = (int)chunks; p.chunk = tree_chunk(a); p.nseq = (int)a->num_seqs;
  p.shift = __builtin_ctz((unsigned)a->page_tokens);
  p.scale = a->scale;
  p.po = reinterpret_cast<float*>(a->workspace);
  p.pml = p.po + (size_t)a->num_seqs * a->H * chunks * a->max_new * a->d;
  hipStream_t st = as_stream(stream);
  if (a->dtype == KDN_DTYPE_BF16) return a->d == 64 ? launch_tree<AttnBF16<64>>(p, st) : launch_tree<AttnBF16<128>>(p, st);
  return a->d == 64 ? launch_tree<AttnF32<64>>(p, st) : launch_tree<AttnF32<128>>(p, st);
}
