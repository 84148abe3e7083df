// The pages of the anchor layers' keys and values: copies of whole pages, new tokens into their places, and the host's
// bookkeeping of who has which page (the softmax anchor pages of the reference's HybridMemoryPool,
// serving/hybrid_memory_pool.{h,cpp}: reference-counted pages, shared by a fork until one of the two writes).
#include <hip/hip_runtime.h>
#include <algorithm>
#include <new>
#include <vector>
#include "kdn_io.hpp"
#include "kdn_internal.hpp"
#include "../../include/kdn_bounded.h"

namespace kdn {

// Pairs of a launch, in its arguments: no device copy of the host's list, whose life the caller would have to keep.
constexpr int COPY_PAIRS = 448;
struct CopyPairs {
  int32_t at[2 * COPY_PAIRS];
};
constexpr int COPY_UNITS = 4;  // 16-byte units a lane has in flight

// One workgroup copies 16 KB of one page (its last one the rest).  Nothing is read again soon: nontemporal.  537 MB of pages
// in three launches of up to 448 pairs: 211 us, 5.1 TB/s read and written (a large copy 4.9); nine pages of 64 KB 2.9 us.
__global__ void __launch_bounds__(256) page_copy_kernel(unsigned char* slab, int64_t page_bytes, CopyPairs pairs) {
  const u32x4* src = reinterpret_cast<const u32x4*>(slab + pairs.at[2 * blockIdx.y] * page_bytes);
  u32x4* dst = reinterpret_cast<u32x4*>(slab + pairs.at[2 * blockIdx.y + 1] * page_bytes);
  const int64_t n = page_bytes / 16, first = (int64_t)blockIdx.x * (256 * COPY_UNITS) + threadIdx.x;
  u32x4 x[COPY_UNITS];
#pragma unroll
  for (int i = 0; i < COPY_UNITS; ++i)
    if (first + 256 * i < n) x[i] = __builtin_nontemporal_load(src + first + 256 * i);
#pragma unroll
  for (int i = 0; i < COPY_UNITS; ++i)
    if (first + 256 * i < n) __builtin_nontemporal_store(x[i], dst + first + 256 * i);
}

struct AppendParams {
  const unsigned char *k, *v;
  unsigned char *kp, *vp;
  int64_t ks[2], vs[2], kps[3], vps[3];  // bytes
  const int64_t* rows;
  int64_t tokens, slots;
  int heads, pieces, shift;  // 16-byte pieces of a row: 1 << pieces
};

// A lane moves one 16-byte piece of one head of a token's key or value.  131 MB read and written in 20.7 us, out of the
// caches in part.
__global__ void __launch_bounds__(256) page_append_kernel(AppendParams p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int piece = (int)(i & ((1 << p.pieces) - 1));
  const uint32_t row = (uint32_t)(i >> p.pieces), per = 2u * p.heads, t = row / per, h = row - t * per;
  if (t >= p.tokens) return;
  const int64_t at = p.rows[t];
  if (at < 0 || at >= p.slots) return;
  const bool is_v = h >= (uint32_t)p.heads;
  const int64_t hh = is_v ? h - p.heads : h, page = at >> p.shift, off = at & ((1 << p.shift) - 1);
  const unsigned char* src = is_v ? p.v + t * p.vs[0] + hh * p.vs[1] : p.k + t * p.ks[0] + hh * p.ks[1];
  unsigned char* dst = is_v ? p.vp + page * p.vps[0] + hh * p.vps[1] + off * p.vps[2]
                            : p.kp + page * p.kps[0] + hh * p.kps[1] + off * p.kps[2];
  reinterpret_cast<u32x4*>(dst)[piece] = reinterpret_cast<const u32x4*>(src)[piece];
}

}  // namespace kdn

struct kdn_page_pool {
  struct Stream {
    std::vector<int32_t> pages;
    int64_t tokens = 0;
    bool open = false;
  };
  int64_t num_pages = 0, page_tokens = 0;
  std::vector<int32_t> free_pages;  // top = back(); page 0 is handed out first
  std::vector<int32_t> shares;      // streams that have a page
  std::vector<Stream> streams;
  std::vector<int32_t> free_streams;

  Stream* at(int s) { return s >= 0 && s < (int)streams.size() && streams[(size_t)s].open ? &streams[(size_t)s] : nullptr; }
  const Stream* at(int s) const { return const_cast<kdn_page_pool*>(this)->at(s); }
  void drop(int32_t page) {
    if (--shares[(size_t)page] == 0) free_pages.push_back(page);  // never over its reserved size
  }
};

using namespace kdn;

// The standard library's containers may throw where memory runs out: nothing may leave a C entry.
template <class F>
static auto guarded(F f) -> decltype(f()) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return KDN_ERR_CAPACITY;
  } catch (...) {
    return KDN_ERR_INVALID_ARGUMENT;
  }
}

extern "C" int kdn_page_copy(void* slab, int64_t num_pages, int64_t page_bytes, const int32_t* pairs, int64_t n, void* stream) {
  if (n < 0 || num_pages < 0 || page_bytes <= 0 || page_bytes % 16 != 0) return KDN_ERR_INVALID_ARGUMENT;
  if (n == 0) return KDN_OK;
  if (!slab || !pairs) return KDN_ERR_INVALID_ARGUMENT;
  if (!aligned(slab, 16)) return KDN_ERR_MISALIGNED;
  const int64_t blocks = (page_bytes / 16 + 256 * COPY_UNITS - 1) / (256 * COPY_UNITS);
  if (n > num_pages || num_pages > INT32_MAX || blocks > max_groups(256)) return KDN_ERR_INVALID_ARGUMENT;
  const int rc = guarded([&]() -> int {
    std::vector<int32_t> to((size_t)n);
    for (int64_t i = 0; i < n; ++i) {
      if (pairs[2 * i] < 0 || pairs[2 * i] >= num_pages || pairs[2 * i + 1] < 0 || pairs[2 * i + 1] >= num_pages)
        return KDN_ERR_INVALID_ARGUMENT;
      to[(size_t)i] = pairs[2 * i + 1];
    }
    std::sort(to.begin(), to.end());
    for (int64_t i = 0; i < n; ++i)
      if ((i > 0 && to[(size_t)i] == to[(size_t)i - 1]) || std::binary_search(to.begin(), to.end(), pairs[2 * i]))
        return KDN_ERR_INVALID_ARGUMENT;
    return KDN_OK;
  });
  if (rc != KDN_OK) return rc;
  for (int64_t i = 0; i < n; i += COPY_PAIRS) {
    const int64_t m = std::min<int64_t>(COPY_PAIRS, n - i);
    CopyPairs c;
    std::copy(pairs + 2 * i, pairs + 2 * (i + m), c.at);
    std::fill(c.at + 2 * m, c.at + 2 * COPY_PAIRS, 0);
    hipLaunchKernelGGL(page_copy_kernel, dim3((unsigned)blocks, (unsigned)m), dim3(256), 0, as_stream(stream),
                       (unsigned char*)slab, page_bytes, c);
    const int st = launch_status();
    if (st != KDN_OK) return st;
  }
  return KDN_OK;
}

extern "C" int kdn_page_append(const kdn_page_append_args* a, void* stream) {
  if (!a || a->tokens < 0 || a->H_kv <= 0 || a->H_kv > (1 << 20) || !valid_dtype(a->dtype) || a->num_pages < 0 || a->page_tokens <= 0)
    return KDN_ERR_INVALID_ARGUMENT;
  if ((a->d != 64 && a->d != 128) || a->page_tokens < 16 || (a->page_tokens & (a->page_tokens - 1)) != 0 || a->page_tokens > (1 << 20) ||
      a->num_pages > INT32_MAX || a->tokens > INT32_MAX / (2 * a->H_kv))
    return KDN_ERR_UNSUPPORTED;
  if (a->tokens == 0) return KDN_OK;
  if (!a->rows || !a->k || !a->v || (a->num_pages > 0 && (!a->k_pages || !a->v_pages))) return KDN_ERR_INVALID_ARGUMENT;
  const int64_t size = (int64_t)dtype_size(a->dtype);
  AppendParams p = {};
  bool fits = aligned(a->k, 16) && aligned(a->v, 16) && aligned(a->k_pages, 16) && aligned(a->v_pages, 16);
  for (int i = 0; i < 2; ++i) {
    p.ks[i] = a->k_stride[i] * size; p.vs[i] = a->v_stride[i] * size;
    fits = fits && p.ks[i] % 16 == 0 && p.vs[i] % 16 == 0;
  }
  for (int i = 0; i < 3; ++i) {
    p.kps[i] = a->k_pages_stride[i] * size; p.vps[i] = a->v_pages_stride[i] * size;
    fits = fits && p.kps[i] % 16 == 0 && p.vps[i] % 16 == 0;
  }
  if (!fits) return KDN_ERR_MISALIGNED;
  p.k = (const unsigned char*)a->k; p.v = (const unsigned char*)a->v;
  p.kp = (unsigned char*)a->k_pages; p.vp = (unsigned char*)a->v_pages;
  p.rows = a->rows;
  p.tokens = a->tokens; p.slots = a->num_pages * a->page_tokens;
  p.heads = (int)a->H_kv;
  p.pieces = __builtin_ctz((unsigned)(a->d * size / 16));
  p.shift = __builtin_ctz((unsigned)a->page_tokens);
  const int64_t blocks = (((a->tokens * 2 * a->H_kv) << p.pieces) + 255) / 256;
  if (blocks > max_groups(256)) return KDN_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(page_append_kernel, dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), p);
  return launch_status();
}

extern "C" int kdn_page_pool_create(int64_t num_pages, int64_t page_tokens, int64_t max_streams, kdn_page_pool** out) {
  if (!out) return KDN_ERR_INVALID_ARGUMENT;
  *out = nullptr;
  if (num_pages <= 0 || num_pages > INT32_MAX || max_streams <= 0 || max_streams > INT32_MAX || page_tokens < 16 ||
      page_tokens > (1 << 20) || (page_tokens & (page_tokens - 1)) != 0)
    return KDN_ERR_INVALID_ARGUMENT;
  kdn_page_pool* p = new (std::nothrow) kdn_page_pool;
  if (!p) return KDN_ERR_CAPACITY;
  const int rc = guarded([&]() -> int {
    p->num_pages = num_pages;
    p->page_tokens = page_tokens;
    p->free_pages.resize((size_t)num_pages);
    for (int64_t i = 0; i < num_pages; ++i) p->free_pages[(size_t)i] = (int32_t)(num_pages - 1 - i);
    p->shares.assign((size_t)num_pages, 0);
    p->streams.resize((size_t)max_streams);
    p->free_streams.resize((size_t)max_streams);
    for (int64_t i = 0; i < max_streams; ++i) p->free_streams[(size_t)i] = (int32_t)(max_streams - 1 - i);
    return KDN_OK;
  });
  if (rc != KDN_OK) {
    delete p;
    return rc;
  }
  *out = p;
  return KDN_OK;
}

extern "C" void kdn_page_pool_destroy(kdn_page_pool* pool) { delete pool; }

extern "C" int kdn_page_pool_open(kdn_page_pool* pool) {
  if (!pool) return KDN_ERR_INVALID_ARGUMENT;
  if (pool->free_streams.empty()) return KDN_ERR_CAPACITY;
  const int32_t s = pool->free_streams.back();
  pool->free_streams.pop_back();
  pool->streams[(size_t)s].open = true;
  return s;
}

extern "C" int kdn_page_pool_fork(kdn_page_pool* pool, int stream) {
  if (!pool || !pool->at(stream)) return KDN_ERR_INVALID_ARGUMENT;
  if (pool->free_streams.empty()) return KDN_ERR_CAPACITY;
  return guarded([&]() -> int {
    const int32_t s = pool->free_streams.back();
    kdn_page_pool::Stream &child = pool->streams[(size_t)s], &from = *pool->at(stream);
    child.pages = from.pages;  // the one step that can fail
    child.tokens = from.tokens;
    child.open = true;
    pool->free_streams.pop_back();
    for (int32_t page : child.pages) ++pool->shares[(size_t)page];
    return s;
  });
}

extern "C" int kdn_page_pool_close(kdn_page_pool* pool, int stream) {
  kdn_page_pool::Stream* s = pool ? pool->at(stream) : nullptr;
  if (!s) return KDN_ERR_INVALID_ARGUMENT;
  for (size_t i = s->pages.size(); i-- > 0;) pool->drop(s->pages[i]);
  s->pages.clear();
  s->tokens = 0;
  s->open = false;
  pool->free_streams.push_back(stream);
  return KDN_OK;
}

extern "C" int kdn_page_pool_extend(kdn_page_pool* pool, int stream, int64_t tokens, int32_t pair[2]) {
  kdn_page_pool::Stream* s = pool ? pool->at(stream) : nullptr;
  if (!s || tokens < 0 || tokens > INT64_MAX / 2 - s->tokens || !pair) return KDN_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return 0;
  const int64_t P = pool->page_tokens, have = (int64_t)s->pages.size(), need = (s->tokens + tokens + P - 1) / P - have;
  const bool own = s->tokens % P != 0 && pool->shares[(size_t)s->pages.back()] > 1;
  if (need + (own ? 1 : 0) > (int64_t)pool->free_pages.size()) return KDN_ERR_CAPACITY;
  return guarded([&]() -> int {
    s->pages.reserve((size_t)(have + need));
    if (own) {
      const int32_t to = pool->free_pages.back();
      pool->free_pages.pop_back();
      pair[0] = s->pages.back();
      pair[1] = to;
      --pool->shares[(size_t)pair[0]];  // over one before
      pool->shares[(size_t)to] = 1;
      s->pages.back() = to;
    }
    for (int64_t i = 0; i < need; ++i) {
      const int32_t page = pool->free_pages.back();
      pool->free_pages.pop_back();
      pool->shares[(size_t)page] = 1;
      s->pages.push_back(page);
    }
    s->tokens += tokens;
    return own ? 1 : 0;
  });
}

extern "C" int kdn_page_pool_truncate(kdn_page_pool* pool, int stream, int64_t tokens) {
  kdn_page_pool::Stream* s = pool ? pool->at(stream) : nullptr;
  if (!s || tokens < 0 || tokens > s->tokens) return KDN_ERR_INVALID_ARGUMENT;
  const size_t keep = (size_t)((tokens + pool->page_tokens - 1) / pool->page_tokens);
  while (s->pages.size() > keep) {
    pool->drop(s->pages.back());
    s->pages.pop_back();
  }
  s->tokens = tokens;
  return KDN_OK;
}

extern "C" int64_t kdn_page_pool_length(const kdn_page_pool* pool, int stream) {
  const kdn_page_pool::Stream* s = pool ? pool->at(stream) : nullptr;
  return s ? s->tokens : KDN_ERR_INVALID_ARGUMENT;
}

extern "C" int64_t kdn_page_pool_table(const kdn_page_pool* pool, int stream, int32_t* table, int64_t width) {
  const kdn_page_pool::Stream* s = pool ? pool->at(stream) : nullptr;
  if (!s || width < 0 || (width > 0 && !table)) return KDN_ERR_INVALID_ARGUMENT;
  if ((int64_t)s->pages.size() > width) return KDN_ERR_CAPACITY;
  std::copy(s->pages.begin(), s->pages.end(), table);
  return (int64_t)s->pages.size();
}

extern "C" int kdn_page_pool_rows(const kdn_page_pool* pool, int stream, int64_t first, int64_t n, int64_t* rows) {
  const kdn_page_pool::Stream* s = pool ? pool->at(stream) : nullptr;
  if (!s || first < 0 || n < 0 || first > s->tokens - n || (n > 0 && !rows)) return KDN_ERR_INVALID_ARGUMENT;
  const int64_t P = pool->page_tokens;
  for (int64_t i = 0; i < n; ++i) rows[i] = s->pages[(size_t)((first + i) / P)] * P + (first + i) % P;
  return KDN_OK;
}

extern "C" int64_t kdn_page_pool_compact(kdn_page_pool* pool, int32_t* pairs, int64_t room) {
  if (!pool || room < 0 || (room > 0 && !pairs)) return KDN_ERR_INVALID_ARGUMENT;
  return guarded([&]() -> int64_t {
    const int64_t used = pool->num_pages - (int64_t)pool->free_pages.size();
    // pages in use at or above `used` go to the free ones below it, in order
    std::vector<int32_t> to((size_t)pool->num_pages, -1);
    int64_t moves = 0, hole = 0;
    for (int64_t page = used; page < pool->num_pages; ++page) {
      if (pool->shares[(size_t)page] == 0) continue;
      while (pool->shares[(size_t)hole] != 0) ++hole;  // as many holes below `used` as pages above
      if (moves < room) pairs[2 * moves] = (int32_t)page, pairs[2 * moves + 1] = (int32_t)hole;
      to[(size_t)page] = (int32_t)hole++;
      ++moves;
    }
    if (moves > room) return KDN_ERR_CAPACITY;
    if (moves == 0) return 0;
    for (auto& s : pool->streams)
      for (auto& page : s.pages)
        if (to[(size_t)page] >= 0) page = to[(size_t)page];
    for (int64_t page = used; page < pool->num_pages; ++page)
      if (to[(size_t)page] >= 0) {
        pool->shares[(size_t)to[(size_t)page]] = pool->shares[(size_t)page];
        pool->shares[(size_t)page] = 0;
      }
    pool->free_pages.clear();
    for (int64_t page = pool->num_pages; page-- > used;) pool->free_pages.push_back((int32_t)page);
    return moves;
  });
}

extern "C" int64_t kdn_page_pool_own(kdn_page_pool* pool, int stream, int64_t tokens, int32_t* pairs, int64_t room) {
  kdn_page_pool::Stream* s = pool ? pool->at(stream) : nullptr;
  if (!s || tokens < 0 || tokens > s->tokens || room < 0 || (room > 0 && !pairs)) return KDN_ERR_INVALID_ARGUMENT;
  const size_t n = (size_t)((tokens + pool->page_tokens - 1) / pool->page_tokens);
  int64_t shared = 0;
  for (size_t i = 0; i < n; ++i) shared += pool->shares[(size_t)s->pages[i]] > 1;
  if (shared > room || shared > (int64_t)pool->free_pages.size()) return KDN_ERR_CAPACITY;
  int64_t at = 0;
  for (size_t i = 0; i < n; ++i) {
    const int32_t from = s->pages[i];
    if (pool->shares[(size_t)from] == 1) continue;
    const int32_t to = pool->free_pages.back();
    pool->free_pages.pop_back();
    pairs[2 * at] = from, pairs[2 * at + 1] = to;
    ++at;
    --pool->shares[(size_t)from];  // over one before
    pool->shares[(size_t)to] = 1;
    s->pages[i] = to;
  }
  return at;
}

extern "C" int kdn_page_pool_drop(kdn_page_pool* pool, int stream, int64_t first, int64_t pages) {
  kdn_page_pool::Stream* s = pool ? pool->at(stream) : nullptr;
  if (!s || first < 0 || pages < 0 || first > s->tokens / pool->page_tokens - pages) return KDN_ERR_INVALID_ARGUMENT;
  for (int64_t i = first + pages; i-- > first;) pool->drop(s->pages[(size_t)i]);
  s->pages.erase(s->pages.begin() + first, s->pages.begin() + first + pages);
  s->tokens -= pages * pool->page_tokens;
  return KDN_OK;
}

extern "C" int64_t kdn_page_pool_free(const kdn_page_pool* pool) { return pool ? (int64_t)pool->free_pages.size() : 0; }
extern "C" int64_t kdn_page_pool_used(const kdn_page_pool* pool) {
  return pool ? pool->num_pages - (int64_t)pool->free_pages.size() : 0;
}
