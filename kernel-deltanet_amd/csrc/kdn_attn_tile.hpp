// Tiles and fragments of the softmax attention kernels (kdn_attn*.hip), all on the 32x32 output-tile MFMAs of CDNA4:
//   v_mfma_f32_32x32x16_bf16 : lane l holds A[l%32][8*(l/32)+s], B[8*(l/32)+s][l%32], s = 0..7
//   v_mfma_f32_32x32x2_f32   : lane l holds A[l%32][l/32],       B[l/32][l%32]
//   D (both)                 : lane l holds D[rho(l, i)][l%32], rho(l, i) = 8*(i/4) + 4*(l/32) + i%4, i = 0..15
// A fragment is eight values a lane, a 16-deep operand: one bf16 MFMA, or eight fp32 ones (slot s of every lane feeds the
// s-th).  A and B take the same (lane, slot) -> depth map, so any order of the depth will do.  The attention kernels use
// that: the accumulator of a product, its rows rho, is the B operand of the next one register for register (slots 8m ..
// 8m + 7 are one fragment), if that product's A operand reads depth 16m + 8*(s/4) + 4*(l/32) + s%4 at slot s (col_frag).
// So the scores never leave their registers.  32x32 tiles take half the LDS bytes per product of 16x16 ones: a wave reads
// 1 KB of A per 32 cycles of its matrix core, the four waves of a CU 128 bytes a cycle, all that LDS gives; two 16x16
// tiles would take twice that.
#pragma once
#include "kdn_frag.hpp"
#include "kdn_internal.hpp"
#include "../../include/kdn_anchor.h"

namespace kdn {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ int rho(int half, int i) { return 8 * (i >> 2) + 4 * half + (i & 3); }

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// Rows of D elements in LDS, in 16-byte pieces: piece c of row r lies at c ^ piece_swizzle(r).  Of the accesses:
//   row_frag: 16 lanes read one piece c of 16 consecutive rows; the swizzle is a permutation of the row's low four bits
//     (128-byte rows: of bits 1-3, bit 0 being the half of the 256 bytes), so that they take all 64 banks once;
//   col_frag (bf16): 32 lanes read 8-byte runs of four rows r0 .. r0+3 (r0 a multiple of 4) and 32 columns; the row's low
//     two bits are on bits 2-3 of the piece, its pieces c .. c+3 on bits 0-1: 64 banks once again.
template <int PIECES>
__device__ __host__ __forceinline__ constexpr int piece_swizzle(int r) {
  return PIECES == 8 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r & 3) << 2 | ((r >> 2) & 3);
}

// 0: a number, 1: infinity, 2: minus infinity, 3: no number.
__device__ __forceinline__ int value_kind(float x) { return x != x ? 3 : x == INFINITY ? 1 : x == -INFINITY ? 2 : 0; }

template <int D_>
struct AttnBF16 {
  typedef __bf16 elem;
  typedef bf16x8 frag;
  static constexpr int D = D_, ROW = 2 * D, PIECES = ROW / 16;
  static constexpr int MFMAS = 1, ROW_READS = 1, COL_READS = 2, AHEAD = 4;  // of a product; operands read ahead
  __device__ __forceinline__ static f32x16 mma(const f32x16& acc, const frag& a, const frag& b) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
  }
  __device__ __forceinline__ static frag load(const elem* p) { return *reinterpret_cast<const frag*>(p); }
  // values 8m .. 8m + 7 of an accumulator as a fragment (rounded to bf16: what the matrix cores take; the sums stay fp32)
  __device__ __forceinline__ static frag from_acc(const f32x16& v, int m) {
    frag r;
#pragma unroll
    for (int s = 0; s < 8; ++s) r[s] = (__bf16)v[8 * m + s];
    return r;
  }
  // the fragment with its infinities and NaNs as zeros; `rest` keeps whether there was one
  __device__ __forceinline__ static frag finite(const frag& f, bool& rest) {
    typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
    const u16x8 x = __builtin_bit_cast(u16x8, f), gap = (x & (unsigned short)0x7f80) ^ (unsigned short)0x7f80;  // 0: no number
    const u16x8 one = __builtin_elementwise_min(gap, (u16x8)(unsigned short)1);
    const u32x4 all = __builtin_bit_cast(u32x4, one);
    rest |= (all[0] & all[1] & all[2] & all[3]) != 0x00010001u;
    return __builtin_bit_cast(frag, (u16x8)(x & (u16x8)((unsigned short)0 - one)));
  }
  __device__ __forceinline__ static bool is_kind(const frag& f, int s, int kind) { return value_kind((float)f[s]) == kind; }
  // lane l slot s = T[row][16 ks + 8 (l/32) + s], row the lane's own
  __device__ __forceinline__ static frag row_frag(const unsigned char* t, int row, int ks, int half) {
    return *reinterpret_cast<const frag*>(t + row * ROW + 16 * ((2 * ks + half) ^ piece_swizzle<PIECES>(row)));
  }
  // lane l slot s = T[r0 + 8 (s/4) + 4 (l/32) + s%4][32 ct + l%32]: two transposing reads of four rows each.  In a
  // 16-lane group lane j addresses the 8-byte run of row j/4 and columns 4 (j%4) ..+3 of the group's 16.
  __device__ __forceinline__ static frag col_frag(const unsigned char* t, int r0, int ct, int lane) {
    const int j = lane & 15, half = lane >> 5, c = 4 * ct + 2 * ((lane >> 4) & 1) + ((j & 3) >> 1);
    bf16x4 part[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int row = r0 + 8 * p + 4 * half + (j >> 2);
      const unsigned char* a = t + row * ROW + 16 * (c ^ piece_swizzle<PIECES>(row)) + 8 * (j & 1);
      part[p] = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a)));
    }
    return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

template <int D_>
struct AttnF32 {
  typedef float elem;
  typedef f32x8 frag;
  static constexpr int D = D_, ROW = 4 * D, PIECES = ROW / 16;
  static constexpr int MFMAS = 8, ROW_READS = 2, COL_READS = 8, AHEAD = 2;
  __device__ __forceinline__ static f32x16 mma(f32x16 acc, const frag& a, const frag& b) {
#pragma unroll
    for (int s = 0; s < 8; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], b[s], acc, 0, 0, 0);
    return acc;
  }
  __device__ __forceinline__ static frag load(const elem* p) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
    return pair_to8(a, b);
  }
  __device__ __forceinline__ static frag from_acc(const f32x16& v, int m) {
    frag r;
#pragma unroll
    for (int s = 0; s < 8; ++s) r[s] = v[8 * m + s];
    return r;
  }
  __device__ __forceinline__ static frag finite(const frag& f, bool& rest) {
    frag r;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const bool number = __builtin_fabsf(f[s]) < INFINITY;
      rest |= !number;
      r[s] = number ? f[s] : 0.f;
    }
    return r;
  }
  __device__ __forceinline__ static bool is_kind(const frag& f, int s, int kind) { return value_kind(f[s]) == kind; }
  __device__ __forceinline__ static frag row_frag(const unsigned char* t, int row, int ks, int half) {
    const int c = 4 * ks + 2 * half, f = piece_swizzle<PIECES>(row);
    return pair_to8(*reinterpret_cast<const f32x4*>(t + row * ROW + 16 * (c ^ f)),
                    *reinterpret_cast<const f32x4*>(t + row * ROW + 16 * ((c + 1) ^ f)));
  }
  __device__ __forceinline__ static frag col_frag(const unsigned char* t, int r0, int ct, int lane) {
    const int half = lane >> 5, col = 32 * ct + (lane & 31);
    frag r;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const int row = r0 + 8 * (s >> 2) + 4 * half + (s & 3);
      r[s] = *reinterpret_cast<const float*>(t + row * ROW + 16 * ((col >> 2) ^ piece_swizzle<PIECES>(row)) + 4 * (col & 3));
    }
    return r;
  }
};

// A copy by the load unit from memory to LDS, 16 or 4 bytes a lane: from the buffer's start + lane_off + off to `to`, the
// lanes one after another.
// The buffer form of it: the compiler takes the global one for an access that may be to either memory, and waits for all
// of a wave's LDS reads wherever it needs one while such a copy is on its way.
// `start` is the same in all lanes: said to the compiler, which goes through the lanes' values one by one otherwise.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* start) {
  const uint64_t at = reinterpret_cast<uint64_t>(start);
  const uint64_t one = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(one), 0, -1, 0x00027000);  // raw bytes, no bound of its own
}
__device__ __forceinline__ void copy16_to_lds(__amdgpu_buffer_rsrc_t from, uint32_t lane_off, uint32_t off, unsigned char* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)(to), 16, (int)lane_off, (int)off, 0, 0);
}
__device__ __forceinline__ void copy4_to_lds(__amdgpu_buffer_rsrc_t from, uint32_t lane_off, unsigned char* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)(to), 4, (int)lane_off, 0, 0, 0);
}

// The copy of ROWS rows of D elements into an LDS tile by the load unit itself (16 bytes a lane, 1 KB an instruction,
// nothing in registers): the WAVES waves of a workgroup share it.  The first row's address is the same in all lanes, a lane's
// offset from it the same for every tile, so that a whole tile's copies take no vector arithmetic.  (With each lane's own
// 64-bit address formed for each copy, the multiplications were a fifth of the forward's vector cycles.)  Rows past `last`
// repeat it, so that every address is inside the tensor and every value one that is there.
template <class P, int ROWS, int WAVES>
struct Stager {
  static constexpr int RPI = 64 / P::PIECES, N = ROWS * P::PIECES / 64 / WAVES, STEP = WAVES * RPI, NV = STEP >= 16 ? 1 : 16 / STEP;
  static_assert(N * WAVES * RPI == ROWS, "the waves share the copies evenly");
  uint32_t row_bytes, off[NV];
  int wave, lane;
  __device__ __forceinline__ Stager(int64_t stride, int wave_, int lane_) : wave(wave_), lane(lane_) {
    row_bytes = (uint32_t)(stride * (int64_t)sizeof(typename P::elem));
#pragma unroll
    for (int v = 0; v < NV; ++v) off[v] = (uint32_t)(wave * RPI + lane / P::PIECES) * row_bytes + 16 * piece(v);
  }
  __device__ __forceinline__ int piece(int i) const {
    return (lane % P::PIECES) ^ piece_swizzle<P::PIECES>(i * STEP + wave * RPI + lane / P::PIECES);
  }
  __device__ __forceinline__ void operator()(const typename P::elem* first, int last, unsigned char* tile) const {
    const __amdgpu_buffer_rsrc_t rows = buffer_at(first);
    if (last >= ROWS - 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) copy16_to_lds(rows, off[i % NV], i * STEP * row_bytes, tile + (i * WAVES + wave) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        copy16_to_lds(rows, (uint32_t)min(i * STEP + wave * RPI + lane / P::PIECES, last) * row_bytes + 16 * piece(i % NV), 0,
                        tile + (i * WAVES + wave) * 1024);
    }
  }
};
// Strides that a copy's 32-bit offsets reach over.
inline bool stage_reach(int64_t stride, int dtype) { return stride <= INT32_MAX / (64 * (int64_t)dtype_size(dtype)); }

// All but this wave's last N copies have arrived; after the barrier, so have every wave's, and every wave has read the tile
// that the next copies overwrite.
template <int N = 0>
__device__ __forceinline__ void staged_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// The order of N products and of the LDS reads of their operands (READS each) in the instructions around this: the first
// AHEAD operands, then a product and the operand of the one AHEAD after it, in turn.  Left to itself the compiler keeps one
// operand's registers and waits for LDS, 100 cycles and more, before each product of 32.
template <class P, int N, int READS>
__device__ __forceinline__ void sched_products() {
  constexpr int AHEAD = N < P::AHEAD ? N : P::AHEAD;
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
  for (int i = 0; i < N - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, P::MFMAS, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * P::MFMAS, 0);
}

// The values of lanes l % 32 and l % 32 + 32, in both.  (The elements are copied out before they are cast: a bit cast of an
// element of the builtin's result takes element 0 whichever it names.)
__device__ __forceinline__ void halves(float v, float& lower, float& upper) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  const unsigned a = r[0], b = r[1];
  lower = __builtin_bit_cast(float, a);
  upper = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float half_max(float v) {
  float a, b;
  halves(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float half_sum(float v) {
  float a, b;
  halves(v, a, b);
  return a + b;
}

// One 32-wide tile of a transposed accumulator (lane: row of the tensor; registers: 32 of its columns) times `f`, as the
// columns 0 .. 31 of a row.  bf16: the halves of the wave exchange their 4-column runs, 16 bytes a store.
__device__ __forceinline__ void store_row32(__bf16* row, const f32x16& v, float f, int half, bool live) {
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    unsigned a[2], b[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
      bf16x2 lo = {(__bf16)(v[8 * m + 2 * e] * f), (__bf16)(v[8 * m + 2 * e + 1] * f)};
      bf16x2 hi = {(__bf16)(v[8 * m + 4 + 2 * e] * f), (__bf16)(v[8 * m + 5 + 2 * e] * f)};
      const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi), false, false);
      a[e] = r[0];
      b[e] = r[1];
    }
    const u32x4 out = {a[0], a[1], b[0], b[1]};
    if (live) *reinterpret_cast<u32x4*>(row + 16 * m + 8 * half) = out;
  }
}
__device__ __forceinline__ void store_row32(float* row, const f32x16& v, float f, int half, bool live) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const f32x4 out = {v[4 * m] * f, v[4 * m + 1] * f, v[4 * m + 2] * f, v[4 * m + 3] * f};
    if (live) *reinterpret_cast<f32x4*>(row + 8 * m + 4 * half) = out;
  }
}

// o += V^T P over 16 KK keys of which rows see only some: `s` the weights (zero where unseen), seen(x) whether the lane's row
// sees key x of them.  A weight of zero times an infinity is no number, and a row would get what a key that it
// does not see holds: V goes into the products with such values as zeros, and where there are any, three more products count,
// for each sum, the infinities, minus infinities and NaNs of seen keys alone.
template <class P, int KK, int CT, class Seen>
__device__ __forceinline__ void masked_values(f32x16 (&o)[CT], const unsigned char* vt, int r0, int lane, const f32x16* s, Seen seen) {
  bool rest = false;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    __builtin_amdgcn_sched_barrier(0);  // one block's operands at a time: registers
    const typename P::frag pf = P::from_acc(s[kk >> 1], kk & 1);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] = P::mma(o[ct], P::finite(P::col_frag(vt, r0 + 16 * kk, ct, lane), rest), pf);
  }
  __builtin_amdgcn_sched_barrier(0);
  if (!__any(rest)) return;
  const int half = lane >> 5;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
#pragma unroll 1
    for (int kind = 1; kind <= 3; ++kind) {
      f32x16 count = zero16();
#pragma unroll 1
      for (int kk = 0; kk < KK; ++kk) {
        const typename P::frag v = P::col_frag(vt, r0 + 16 * kk, ct, lane);
        typename P::frag is, sees;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          is[x] = (typename P::elem)(P::is_kind(v, x, kind) ? 1.f : 0.f);
          sees[x] = (typename P::elem)(seen(16 * kk + rho(half, x)) ? 1.f : 0.f);
        }
        count = P::mma(count, is, sees);
      }
      const float value = kind == 1 ? INFINITY : kind == 2 ? -INFINITY : NAN;
#pragma unroll
      for (int i = 0; i < 16; ++i) o[ct][i] += count[i] > 0.f ? value : 0.f;
    }
  }
}

// The waves of a workgroup that share rows (SPLIT of them; the workgroup's four waves are 4 / SPLIT groups) add their sums
// in the waves' order: each wave puts the column tiles it does not finish into LDS, as they lie in its registers, and adds
// the others' to those it does (column tile ct is finished by wave ct % SPLIT).  `mine` scales a wave's own sums first.
// `ends` runs for the tiles that the wave finishes.  4 KB of LDS a wave and column tile; ends with all waves having read.
template <int SPLIT, int CT, class F>
__device__ __forceinline__ void join_sums(f32x16 (&o)[CT], float mine, unsigned char* lds, int w, int lane, F ends) {
  const int part = w % SPLIT, group = w / SPLIT;
  f32x4* box = reinterpret_cast<f32x4*>(lds) + lane;
  auto at = [&](int ct, int from) { return (((group * CT + ct) * SPLIT + from) * 4) * 64; };
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
    for (int i = 0; i < 16; ++i) o[ct][i] *= mine;
    if (ct % SPLIT != part)
#pragma unroll
      for (int a = 0; a < 4; ++a) box[at(ct, part) + 64 * a] = f32x4{o[ct][4 * a], o[ct][4 * a + 1], o[ct][4 * a + 2], o[ct][4 * a + 3]};
  }
  __syncthreads();
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
    if (ct % SPLIT == part) {
      f32x16 sum = zero16();
#pragma unroll
      for (int from = 0; from < SPLIT; ++from)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const f32x4 x = from == ct % SPLIT ? f32x4{o[ct][4 * a], o[ct][4 * a + 1], o[ct][4 * a + 2], o[ct][4 * a + 3]} : box[at(ct, from) + 64 * a];
#pragma unroll
          for (int y = 0; y < 4; ++y) sum[4 * a + y] += x[y];
        }
      ends(ct, sum);
    }
  __syncthreads();
}

// Tile slots over a packed batch: sequence b has the slots [cu[b] / ROWS + b, cu[b + 1] / ROWS + b + 1), at least as many
// as it has tiles of ROWS rows, so that a grid of total / ROWS + sequences slots covers every batch without its lengths
// being known to the host.  The rows outside the offsets are two sequences more, that see nothing and that nothing sees: those
// before the first one, number -1, and those past the last one's end (a batch padded to a fixed size), number nseq.  They
// count in the slots, `entry` being a sequence's number and one.  The sequence of a slot is found 64 offsets at a time by the
// whole wave.  Offsets are clamped to the tensor: a wrong one gives wrong rows, never an access outside.
struct SeqTile {
  int seq, row0;  // row0: first row of the tile in the sequence; negative: no tile
  int64_t lo;     // the sequence's first row
  int len;        // and length
};
__device__ __forceinline__ int64_t seq_start(const int64_t* cu, int64_t total, int64_t b) {
  return min(max(cu[b], (int64_t)0), total);
}
__device__ __forceinline__ int64_t entry_start(const int64_t* cu, int64_t nseq, int64_t total, int64_t entry) {
  const int64_t first = seq_start(cu, total, min(max(entry - 1, (int64_t)0), nseq));  // in every lane: no branch around a load
  return entry == 0 ? 0 : entry > nseq + 1 ? total : first;
}
inline int64_t tile_slots(int64_t total, int64_t rows, int64_t nseq) { return total / rows + nseq + 2; }
template <int ROWS>
__device__ __forceinline__ SeqTile find_tile(const int64_t* cu, int64_t nseq, int64_t total, int64_t slot, int lane) {
  int64_t lo = 0, n = nseq + 2;
  while (n > 1) {
    const int64_t step = (n + 63) / 64, at = lo + lane * step;
    const bool before = lane * step < n && entry_start(cu, nseq, total, at) / ROWS + at <= slot;
    const int hits = __popcll(__ballot(before));
    const int64_t skip = (hits > 0 ? hits - 1 : 0) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  SeqTile t;
  t.seq = (int)lo - 1;
  t.lo = entry_start(cu, nseq, total, lo);
  t.len = (int)(max(entry_start(cu, nseq, total, lo + 1), t.lo) - t.lo);
  const int64_t tile = slot - (t.lo / ROWS + lo);
  t.row0 = tile < 0 || tile * ROWS >= t.len ? -1 : (int)(tile * ROWS);
  return t;
}
// The tile that is the id-th in the order of most work first, a tile's work being its place in its sequence (its rows see
// that many tiles of keys; counted from the sequence's end for the keys, whose first ones the most rows see): what runs
// longest starts first, whichever sequence it is of.  Up to 62 sequences; with more, slot `slots` - 1 - id of find_tile (each
// sequence's own tiles most work first).  Lane b has entry b's tiles nt; N(t), the tiles at place t or behind it, is
// the sum of max(nt - t, 0), and the tile's place the last t with N(t) > id.
template <int ROWS, bool FROM_END>
__device__ __forceinline__ SeqTile find_heavy(const int64_t* cu, int64_t nseq, int64_t total, int64_t id, int64_t slots, int lane) {
  if (nseq > 62) {
    SeqTile t = find_tile<ROWS>(cu, nseq, total, slots - 1 - id, lane);
    if (FROM_END && t.row0 >= 0) t.row0 = (t.len - 1) / ROWS * ROWS - t.row0;
    return t;
  }
  const int n = (int)nseq + 2;
  const int64_t lo = entry_start(cu, nseq, total, lane), hi = max(entry_start(cu, nseq, total, lane + 1), lo);
  const int len = lane < n ? (int)(hi - lo) : 0, nt = (len + ROWS - 1) / ROWS;
  auto behind = [&](int t) {
    int sum = 0;
    for (int b = 0; b < n; ++b) sum += max(__builtin_amdgcn_readlane(nt, b) - t, 0);
    return sum;
  };
  int most = 0;
  for (int b = 0; b < n; ++b) most = max(most, __builtin_amdgcn_readlane(nt, b));
  SeqTile s;
  s.row0 = -1;
  if (id >= behind(0)) return s;
  int t = 0;
  for (int range = most; range > 1;) {
    const int step = (range + 63) / 64, hits = __popcll(__ballot(lane * step < range && behind(t + lane * step) > id));
    t += (hits - 1) * step;
    range = min(step, range - (hits - 1) * step);
  }
  const int rank = (int)id - behind(t + 1);
  const uint64_t there = __ballot(nt > t);
  const int at = __ffsll((unsigned long long)__ballot((there >> lane & 1) && __popcll(there & ((1ull << lane) - 1)) == rank)) - 1;
  const int entry = __builtin_amdgcn_readfirstlane(at);
  s.seq = entry - 1;
  s.len = __builtin_amdgcn_readlane(len, entry);
  s.lo = (int64_t)__builtin_amdgcn_readlane((int)(lo >> 32), entry) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)lo, entry);
  s.row0 = (FROM_END ? __builtin_amdgcn_readlane(nt, entry) - 1 - t : t) * ROWS;
  return s;
}
// The other tensor's rows of a tile's sequence: none for the rows outside the offsets.
__device__ __forceinline__ void other_rows(const int64_t* cu, int64_t nseq, int64_t total, int seq, int64_t& lo, int& len) {
  const bool there = seq >= 0 && seq < nseq;
  lo = there ? seq_start(cu, total, seq) : 0;
  len = there ? (int)(max(seq_start(cu, total, seq + 1), lo) - lo) : 0;
}

// Device-side arguments of the attention kernels (kdn_attn_args with the defaults filled in).
struct AttnParams {
  const void *q, *k, *v, *y, *dy;
  void *out, *dq, *dk, *dv;
  void* low;           // what rounding took from y, or NULL
  int64_t lows[2];
  int64_t qs[2], ks[2], vs[2], ys[2], dys[2], dqs[2], dks[2], dvs[2];  // element strides [token][head]
  float* lse;          // [H][total_q]
  const float *stat, *delta;  // [H][total_q]: minus lse / scale, and minus dy . y of each row (backward)
  const int64_t *cu_q, *cu_k;
  int64_t nseq, total_q, total_k;
  float *part_dk, *part_dv;  // [subset][total_k][KV][D] sums of dk and dv over a subset of a key head's query heads (subsets > 1)
  int H, KV, G, subsets;
  float scale;
};

int attn_check(const kdn_attn_args* a);          // sizes
int attn_check_tensors(const kdn_attn_args* a);  // pointers, strides, alignment
bool attn_strides_ok(const int64_t s[2], int dtype);
AttnParams attn_params(const kdn_attn_args* a);
int attn_split(int64_t rows, int64_t heads);     // waves that share 32 rows

}  // namespace kdn
