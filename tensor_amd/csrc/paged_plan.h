// How a paged attention call is shared out: plain code without HIP, so that a CPU test can compile it
// by itself; the kernels run the same functions.
//
// The work is two lists of key tiles.  Item = the rows of one request (or of all tokens, against the shared
// prefix) and one key head, in row tiles: wide ones of up to 128 rows against tiles of 64 keys, and
// narrow ones of up to 16 rows (decode) against tiles of 32.  The wide list is cut into equal ranges, one for
// each workgroup, the narrow list into equal ranges, one for each wave; a range crosses items, so the
// work is even whatever the lengths.  The part of an item in one range is a segment; it leaves its
// rows' maxima, sums and outputs in a slot of the workspace, and a second kernel joins the slots of a row.
// Slot = item + range: both only grow along the list, one of them with every segment.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __HIP__
#define PAGED_CODE __host__ __device__ inline
#else
#define PAGED_CODE inline
#endif

namespace tensor_paged {

constexpr int kWaves = 4;                   // of a workgroup
constexpr int kGroups = 512;                // workgroups: two per CU
constexpr int kStreams = kGroups * kWaves;  // waves of the launch
constexpr int kWideRows = 128, kWideKeys = 64, kNarrowRows = 16, kNarrowKeys = 32;

PAGED_CODE int least(int a, int b) { return a < b ? a : b; }
PAGED_CODE int most(int a, int b) { return a > b ? a : b; }

// Extents of a call; rows of wide tiles are whole tokens.
struct Extents {
  int tokens, requests, kv, share, page_shift, columns, prefix_columns;  // share: query heads of a key head
  int per;                                                               // tokens of a wide row tile
};
PAGED_CODE Extents extents(int tokens, int requests, int heads, int kv, int page_shift, int columns, int prefix_columns) {
  const int share = heads / kv;
  return Extents{tokens, requests, kv, share, page_shift, columns, prefix_columns, kWideRows / share};
}

PAGED_CODE size_t plan_bytes(int requests) { return ((size_t)(2 + 2 * (requests + 2)) * 4 + 255) / 256 * 256; }
PAGED_CODE size_t slot_floats(int rows, int dim) { return (size_t)rows * (dim + 2); }
PAGED_CODE int64_t wide_slots(const Extents& e) {
  return (int64_t)e.kv * (e.tokens / e.per + e.requests + (e.tokens + e.per - 1) / e.per) + kGroups;
}
PAGED_CODE int64_t narrow_slots(const Extents& e) { return (int64_t)e.kv * (e.requests + 1) + kStreams; }

// sum over i < n of floor((a i + b) / m), by the Euclidean algorithm
PAGED_CODE unsigned floor_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
  unsigned sum = 0;
  while (n) {
    if (a >= m) {
      sum += (unsigned)((uint64_t)(n - 1) * n / 2) * (a / m);
      a %= m;
    }
    if (b >= m) {
      sum += n * (b / m);
      b %= m;
    }
    const unsigned y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y % m;
    const unsigned t = m;
    m = a;
    a = t;
  }
  return sum;
}

// One request's tokens and keys, or (prefix) all tokens and the shared keys.
struct Request {
  int first, count;  // tokens
  int keys;
  int behind;        // own keys before the first token (negative in a malformed call: some tokens see none)
  bool prefix, narrow;
};
PAGED_CODE int held(int length, int columns, int page_shift) {
  const int64_t room = (int64_t)columns << page_shift;
  return length < 0 ? 0 : length < room ? length : (int)room;
}
// from its offsets and length, whatever they are: rows and keys stay within the extents
PAGED_CODE Request own_request(const Extents& e, int first, int end, int length) {
  Request r;
  r.prefix = false;
  r.first = least(most(first, 0), e.tokens);
  r.count = least(most(end, r.first), e.tokens) - r.first;
  r.keys = held(length, e.columns, e.page_shift);
  r.behind = r.keys - r.count;
  r.narrow = (int64_t)r.count * e.share <= kNarrowRows;
  return r;
}
PAGED_CODE Request prefix_request(const Extents& e, int end, int length) {
  Request r;
  r.prefix = true;
  r.first = 0;
  r.count = least(most(end, 0), e.tokens);
  r.keys = held(length, e.prefix_columns, e.page_shift);
  r.behind = 0;
  r.narrow = (int64_t)r.count * e.share <= kNarrowRows;
  return r;
}

PAGED_CODE int row_tiles(const Extents& e, const Request& r) { return (r.count + e.per - 1) / e.per; }
// key tiles of the first `tiles` row tiles of a wide request, one key head: a row tile goes up to the keys
// its last token sees
PAGED_CODE unsigned wide_tiles(const Extents& e, const Request& r, int tiles) {
  if (r.prefix) return (unsigned)tiles * ((r.keys + kWideKeys - 1) / kWideKeys);
  const int base = most(r.behind, 0), all = row_tiles(e, r);
  const unsigned sum = floor_sum(least(tiles, all - 1), kWideKeys, e.per, base + e.per + kWideKeys - 1);
  return tiles < all ? sum : sum + (base + r.count + kWideKeys - 1) / kWideKeys;
}
// Tiles of both lists in one call, at most (whatever the lengths within the extents): row tiles, and the
// narrow requests' one each, by the key tiles of the longest list.  The call is refused from 2^31 on.
PAGED_CODE int64_t most_tiles(const Extents& e) {
  const int64_t keys = (int64_t)most(e.columns, e.prefix_columns) << e.page_shift;
  return e.kv * (e.tokens / e.per * 2 + e.requests + 3ll) * ((keys + e.tokens) / kNarrowKeys + 2) + 2 * kStreams;
}

// key tiles of one key head
PAGED_CODE unsigned head_tiles(const Extents& e, const Request& r) {
  if (!r.count || !r.keys) return 0;
  if (r.narrow) return (r.keys + kNarrowKeys - 1) / kNarrowKeys;
  return wide_tiles(e, r, row_tiles(e, r));
}

// Items of request b (b = requests: the prefix) grow along the list and stay within the slots.
PAGED_CODE int wide_item(const Extents& e, const Request& r, int b, int head, int tile) {
  return e.kv * ((r.prefix ? r.count : r.first) / e.per + b) + head * row_tiles(e, r) + tile;
}
PAGED_CODE int narrow_item(const Extents& e, int b, int head) { return e.kv * b + head; }

// largest i < count with start[i] <= t; start[0] <= t < start[count]
PAGED_CODE int find(const int32_t* start, int count, int t) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// The segment at tile `at` of a request's list, in a range that takes `left` more tiles.
struct Segment {
  int head, tile, t0, t1;  // key head, row tile, key tiles
  int item;
  bool all;                // the item's only segment
};
PAGED_CODE Segment segment_at(const Extents& e, const Request& r, int b, int per_head, int at, int left) {
  Segment s;
  s.head = at / per_head;
  const int rest = at - s.head * per_head;
  int tiles = per_head, begin = 0;
  s.tile = 0;
  if (!r.narrow) {
    int lo = 0, hi = row_tiles(e, r);  // the last row tile that begins at or before rest
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((int)wide_tiles(e, r, mid) <= rest) lo = mid; else hi = mid;
    }
    s.tile = lo;
    begin = (int)wide_tiles(e, r, lo);
    tiles = (int)wide_tiles(e, r, lo + 1) - begin;
  }
  s.t0 = rest - begin;
  s.t1 = least(tiles, s.t0 + left);
  s.item = r.narrow ? narrow_item(e, b, s.head) : wide_item(e, r, b, s.head, s.tile);
  s.all = s.t0 == 0 && s.t1 == tiles;
  return s;
}

// The slots of a token's rows in request b's list, whose first tile is `start`: `in` gives those of one key
// head, in ranges of `quota` tiles.
struct Slots {
  int first, count;
};
struct TokenSlots {
  int t0, tiles, per_head;  // first key tile of the rows' item of key head 0, its tiles, tiles of a head
  int item, items;          // that item, items of a head
  int row;                  // the token's first row within a slot
  PAGED_CODE Slots in(int head, int quota) const {
    if (!tiles || !quota) return Slots{0, 0};
    const int from = t0 + head * per_head, range = from / quota;
    return Slots{item + head * items + range, (from + tiles - 1) / quota - range + 1};
  }
};
PAGED_CODE TokenSlots token_slots(const Extents& e, const Request& r, int b, int start, int token) {
  TokenSlots s{start, (int)head_tiles(e, r), 0, narrow_item(e, b, 0), 1, (token - r.first) * e.share};
  s.per_head = s.tiles;
  if (s.tiles && !r.narrow) {
    const int i = token - r.first, tile = i / e.per, begin = (int)wide_tiles(e, r, tile);
    s.tiles = (int)wide_tiles(e, r, tile + 1) - begin;
    s.t0 += begin;
    s.item = wide_item(e, r, b, 0, tile);
    s.items = row_tiles(e, r);
    s.row = (i - tile * e.per) * e.share;
  }
  return s;
}

}  // namespace tensor_paged
