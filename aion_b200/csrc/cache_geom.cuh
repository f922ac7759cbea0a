// Where the rows of a KV cache live. Plain index arithmetic for host and device (no CUDA header is needed), so
// that every row a kernel may touch can be checked on the CPU.
#pragma once

#include <stdint.h>

#if defined(__CUDACC__)
#define CACHE_FN __host__ __device__ __forceinline__
#else
#define CACHE_FN inline
#endif

namespace aion {

// Where the rows of a cache live: contiguous [B][t_cap], a ring of t_cap rows per request, or pages.
struct CacheGeom {
  const int32_t* table;   // [B][pages_per_request], null: not paged
  uint32_t t_cap;
  uint32_t page_tokens, pages_per_request, pool_pages;
  uint32_t rolling;
};

// The row (of all requests, or of the pool) of a logical step; negative: its page is outside the pool.
CACHE_FN int64_t cache_row(const CacheGeom& g, uint32_t b, uint32_t step) {
  if (g.table) {
    const uint32_t pi = step / g.page_tokens;
    const int32_t page = g.table[(uint64_t)b * g.pages_per_request + pi];
    if (page < 0 || (uint32_t)page >= g.pool_pages) return -1;
    return (int64_t)page * g.page_tokens + (step - pi * g.page_tokens);
  }
  return (int64_t)b * g.t_cap + (g.rolling ? step % g.t_cap : step);
}

// The row that receives new row t of n of request b, which begins at logical step e; negative: none (an earlier
// row of a ring that the same append comes round to again). *bad: the request's range or page is not acceptable;
// a request whose rows do not fit is rejected as a whole.
CACHE_FN int64_t append_row(const CacheGeom& g, uint32_t b, int32_t e, uint32_t t, uint32_t n, bool* bad) {
  *bad = e < 0 || (!g.rolling && (uint64_t)e + n > g.t_cap);
  if (*bad || (g.rolling && (uint64_t)t + g.t_cap < n)) return -1;
  const int64_t row = cache_row(g, b, (uint32_t)e + t);
  *bad = row < 0;
  return row;
}

// The logical steps that a request holds; bad: its length or start is not acceptable, and none is read.
struct ReadSpan {
  uint32_t lo, hi;   // steps [lo, hi) are held
  bool bad;
};
CACHE_FN ReadSpan read_span(const CacheGeom& g, const int32_t* start, const int32_t* lengths, uint32_t b) {
  ReadSpan s{0, g.t_cap, false};
  if (start && start[b] < 0) s.bad = true;
  if (lengths) {
    const int32_t n = lengths[b];
    if (n < 0 || (!g.rolling && (uint32_t)n > g.t_cap)) s.bad = true;
    else s.hi = (uint32_t)n;
    if (g.rolling && s.hi > g.t_cap) s.lo = s.hi - g.t_cap;
  }
  if (s.bad) s.lo = s.hi = 0;
  return s;
}

// The attention kernels copy a context in tiles of TILE_KEYS rows, cut so that none straddles a page or the end of a request's
// rows: a segment (a page, a lap of the ring, or the whole contiguous cache) is cut into tiles of TILE_KEYS keys, the last of
// which may be shorter.
constexpr uint32_t TILE_KEYS = 16;
struct TileSpace {
  uint32_t seg_len, per_seg;
};
CACHE_FN TileSpace tile_space(const CacheGeom& g) {
  const uint32_t len = g.table ? g.page_tokens : g.t_cap;
  return TileSpace{len, len / TILE_KEYS + (len % TILE_KEYS != 0)};
}
CACHE_FN uint32_t tile_at(const TileSpace& ts, uint32_t key) {
  const uint32_t seg = key / ts.seg_len;
  return seg * ts.per_seg + (key - seg * ts.seg_len) / TILE_KEYS;
}
// Rows of a segment's tile: no copy may take more.
CACHE_FN uint32_t tile_rows(const TileSpace& ts, uint32_t in_seg) {
  const uint32_t left = ts.seg_len - in_seg * TILE_KEYS;
  return left < TILE_KEYS ? left : TILE_KEYS;
}
// Tiles [first, end) hold the keys [lo, hi).
struct TileRange {
  uint32_t first, end;
};
CACHE_FN TileRange tiles_of_keys(const TileSpace& ts, uint32_t lo, uint32_t hi) {
  if (hi <= lo) return TileRange{0, 0};
  return TileRange{tile_at(ts, lo), tile_at(ts, hi - 1) + 1};
}

}  // namespace aion
