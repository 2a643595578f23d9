// How a paged attention call is shared out: plain code without HIP, so that a CPU test can compile it
// by itself; the kernels run the same functions.
//
// The work is two lists of key tiles.  Item = the rows of one request (or of all tokens, against the shared
// prefix) and one key head, in row tiles: wide ones of up to 128 rows against tiles of 64 keys, and
// narrow ones of up to 16 rows (decode) against tiles of 32.  The wide list is cut into equal ranges, one for
// each workgroup, or, if it is short, for each of the first half; the narrow list is cut into ranges for waves, of
// which those of the second half of the workgroups take more where the first has wide work.  A range crosses
// items, so the work is even whatever the lengths.  A list goes through all requests for one key head before the
// next: workgroups of one XCD, which have neighbouring ranges, then read the same prefix (3 requests of 1024 tokens
// behind 8192 keys: 383 us, 395 with a request's key heads one after another; 12 of 5 tokens: 26.2 and 28.8).  The
// part of an item in one range is a segment; it leaves its rows' maxima, sums and outputs in a slot of the workspace,
// and a second kernel joins the slots of a row.
// Slot = item + range: both only grow along the list, one of them with every segment.
//
// Narrow tiles waste the matrix cores, wide ones the loads of rows that are not there: 16 rows are level (16 requests of 4
// tokens and 4 heads a key head, 16000 keys: 203 us narrow, 196 wide; 1000 keys: 25.2 and 26.3), and fewer stay narrow.
//
// To begin a wide item costs a workgroup as much as kItemCost tiles, so where there is an item for every fourth
// workgroup each has that many empty positions before its first tile (a prompt of 1024 tokens: 43 us, 54 without; of 512,
// where a range is shorter than that and some hold no tile: 28.3 and 30.2; 16 requests of 33 tokens behind 8192 keys: 108
// and 232; but 64 requests behind 16384 keys, 16 items: 59 and 56).
//
// The prefix is a list entry of its own where tokens of several requests fill its row tiles; where each request
// fills tiles of its own (prompts, one request), its wide items begin with the prefix's tiles instead (`lead`),
// which leaves one slot less to write and join (3 requests of 1024 tokens behind 8192 keys: 386 us, 417 apart; 8 of 128
// behind 4096: 104 and 116; but 16 of 33 behind 8192, whose tiles would be half empty: 130, and 108 apart).
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __HIP__
#define PAGED_CODE __host__ __device__ __forceinline__
#else
#define PAGED_CODE inline
#endif

namespace tensor_paged {

constexpr int kWaves = 4;                   // of a workgroup
constexpr int kGroups = 512;                // workgroups: two per CU
constexpr int kStreams = kGroups * kWaves;  // waves of the launch
constexpr int kWideRows = 128, kWideKeys = 64, kNarrowRows = 16, kNarrowKeys = 32;
constexpr int kItemCost = 3;                // to begin an item, in tiles
constexpr int kSlotCost = 8;                // that, and to leave its rows in a slot and join them
constexpr int kLongRange = 24;              // tiles of a range from which a wide list is long
constexpr int kBeside = 300;                // narrow tiles of half the workgroups beside each wide tile of a range

PAGED_CODE int least(int a, int b) { return a < b ? a : b; }
PAGED_CODE int most(int a, int b) { return a > b ? a : b; }
PAGED_CODE int64_t most64(int64_t a, int64_t b) { return a > b ? a : b; }

// Extents of a call; rows of wide tiles are whole tokens.
struct Extents {
  int tokens, requests, kv, share, page_shift, columns, prefix_columns;  // share: query heads of a key head
  int per;                                                               // tokens of a wide row tile
  int cost;                                                              // positions before a wide item's first tile
  int lead;                                                              // tiles of the prefix that begin each of them
};
PAGED_CODE Extents extents(int tokens, int requests, int heads, int kv, int page_shift, int columns, int prefix_columns) {
  const int share = heads / kv;
  return Extents{tokens, requests, kv, share, page_shift, columns, prefix_columns, kWideRows / share, 0, 0};
}

// Workspace: a record of each token for the joining kernel, then wide and narrow slots.
constexpr int kRecord = 16;  // 32-bit words
PAGED_CODE size_t record_bytes(int tokens) { return ((size_t)tokens * 4 * kRecord + 255) / 256 * 256; }
PAGED_CODE size_t slot_floats(int rows, int dim) { return (size_t)rows * (dim + 2); }
// numbers of one key head's items
PAGED_CODE int narrow_items(const Extents& e) { return e.requests + 1; }
PAGED_CODE int wide_items(const Extents& e) {
  return e.tokens / e.per + e.requests + (e.tokens + e.per - 1) / e.per;
}
PAGED_CODE int64_t wide_slots(const Extents& e) { return (int64_t)e.kv * wide_items(e) + kGroups; }
PAGED_CODE int64_t narrow_slots(const Extents& e) { return (int64_t)e.kv * narrow_items(e) + kStreams; }

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
  return e.kv * (e.tokens / e.per * 2 + e.requests + 3ll) * ((keys + e.tokens) / kNarrowKeys + 2 + kItemCost) + 2 * kStreams;
}

PAGED_CODE int lead_of(const Extents& e, const Request& r) { return r.prefix ? 0 : e.lead; }
// Where row tile `tile` of a wide request begins within its key head's positions: key tiles, and items' costs.
PAGED_CODE int wide_begin(const Extents& e, const Request& r, int tile) {
  return (int)wide_tiles(e, r, tile) + (e.cost + lead_of(e, r)) * tile;
}
// Positions of one key head in its list.
PAGED_CODE int head_span(const Extents& e, const Request& r) {
  if (!r.count || !r.keys) return 0;
  if (r.narrow) return (r.keys + kNarrowKeys - 1) / kNarrowKeys;
  return wide_begin(e, r, row_tiles(e, r));
}
// Items of one key head in the wide list.
PAGED_CODE int head_items(const Extents& e, const Request& r) { return r.count && r.keys && !r.narrow ? row_tiles(e, r) : 0; }
PAGED_CODE int item_cost(int items) { return items >= kGroups / 4 ? kItemCost : 0; }  // by the wide list's items
// Key tiles of a row tile.
PAGED_CODE int item_tiles(const Extents& e, const Request& r, int tile) {
  if (r.narrow) return (r.keys + kNarrowKeys - 1) / kNarrowKeys;
  const int keys = r.prefix ? r.keys : most(r.behind, 0) + least(r.count, (tile + 1) * e.per);
  return lead_of(e, r) + (keys + kWideKeys - 1) / kWideKeys;
}
// The prefix's tiles if they are to lead `items` wide items (of one key head), all that the requests have; else 0.
// That costs the tiles that more items than the prefix's own have, and saves the latter.
PAGED_CODE int lead_tiles(const Extents& e, const Request& prefix, int items) {
  const int tiles = prefix.count ? (prefix.keys + kWideKeys - 1) / kWideKeys : 0, own = row_tiles(e, prefix);
  return !prefix.narrow && (int64_t)(items - own) * tiles <= (int64_t)own * kSlotCost ? tiles : 0;
}

// Number of an item among its key head's (b = requests: the prefix's): grows along the list.
PAGED_CODE int item_number(const Extents& e, const Request& r, int b, int tile) {
  return r.narrow ? b : (r.first + (r.prefix ? r.count : 0)) / e.per + b + tile;  // (the prefix's first is 0)
}

// largest i < count with start[i] <= t; start[0] <= t < start[count]
PAGED_CODE int find(const int32_t* start, int count, int t) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// A range's way through its list: `requests(b)` gives request b, `start` the first position of each within a key
// head and (the last) the head's positions, `items` the numbers of a head's items.
struct Segment {
  int head, tile, t0, t1;  // key head, row tile, key tiles
  int item;
  bool all;                // the item's only segment
};
template <typename Requests>
struct Walk {
  const Extents& e;
  const int32_t* start;
  const Requests& requests;
  const int items;
  int left;             // positions of the range that are left
  int head, at, b;      // the item, and the position within it
  int tile;
  Request r;

  // the range [from, to) of the list, from < to
  PAGED_CODE Walk(const Extents& e, const int32_t* start, const Requests& requests, int items, int from, int to)
      : e(e), start(start), requests(requests), items(items), left(to - from), head(from / start[e.requests + 1]),
        at(from - head * start[e.requests + 1]), b(find(start, e.requests + 1, at)), r(requests(b)) {
    at -= start[b];
    tile = 0;
    if (!r.narrow) {
      int hi = row_tiles(e, r);  // the last row tile that begins at or before the position
      while (hi - tile > 1) {
        const int mid = (tile + hi) >> 1;
        if (wide_begin(e, r, mid) <= at) tile = mid; else hi = mid;
      }
      at -= wide_begin(e, r, tile);
    }
  }
  // the next segment; false at the end of the range
  PAGED_CODE bool next(Segment& s) {
    const int cost = r.narrow ? 0 : e.cost, skip = most(cost - at, 0);
    if (left <= skip) return false;
    const int tiles = item_tiles(e, r, tile);
    s.head = head;
    s.tile = tile;
    s.t0 = at + skip - cost;
    s.t1 = least(tiles, s.t0 + left - skip);
    s.item = head * items + item_number(e, r, b, tile);
    s.all = s.t0 == 0 && s.t1 == tiles;
    left -= skip + s.t1 - s.t0;
    return true;
  }
  // past the item of the last segment, if the range goes on
  PAGED_CODE void advance() {
    if (left <= 0) return;
    at = 0;
    if (++tile < (r.narrow ? 1 : row_tiles(e, r))) return;
    tile = 0;
    const bool last = start[b + 1] == start[e.requests + 1];
    head += last;
    b = find(start, e.requests + 1, last ? 0 : start[b + 1]);
    r = requests(b);
  }
};

// Positions of a list's ranges: `many` for each (few < 0), or for the first kStreams / 2 and `few` for the others.
struct Quota {
  int many, few;
  PAGED_CODE int range(int at) const {
    constexpr int half = kStreams / 2;
    const int others = at - half * many;
    const bool late = few >= 0 && others >= 0;
    return (late ? others : at) / (late ? few : many) + (late ? half : 0);
  }
  PAGED_CODE int begin(int range) const {
    constexpr int half = kStreams / 2;
    return few < 0 || range <= half ? range * many : half * many + (range - half) * few;
  }
};
// A short list beside a narrow one goes to half the workgroups, one on a CU, whose other one reads the narrow list's
// keys meanwhile, and leaves half the slots (64 requests behind 16384 keys: 56 us, 69 with all; 12 requests of 5 tokens:
// 26.2 and 30.3).  A long one needs all (3 x 1024 tokens: 386 us, 458 with half), and so does one alone (a prompt of
// 4096 tokens: 206 us, 244 with half; of 1024: 43 and 45; of 512: 28.3 and 26.9).
PAGED_CODE Quota wide_quota(int positions, int narrow) {
  const int ranges = narrow && positions < kLongRange * kGroups ? kGroups / 2 : kGroups;
  return Quota{(positions + ranges - 1) / ranges, -1};
}
// `wide`: positions of a wide range.  While the first half of the workgroups have those, the others take kBeside
// narrow tiles for each; the rest is for all (64 requests behind 16384 keys: 56 us, 63 in equal shares; with
// heads of 64, whose narrow tiles are half the bytes: 35 and 41).
PAGED_CODE Quota narrow_quota(int positions, int wide) {
  const int few = (int)(most64(positions - (int64_t)kBeside * wide, 0) / kStreams);
  return Quota{(positions - few * (kStreams / 2) + kStreams / 2 - 1) / (kStreams / 2), few};
}

// The slots of a token's rows in request b's list (`start` and `items` as above): `in` gives those of one key head.
struct Slots {
  int first, count;
};
struct TokenSlots {
  int t0, tiles, span;  // position of the first key tile of the rows' item of key head 0, its tiles, positions of a head
  int item, items;      // that item, items of a head
  int row;              // the token's first row within a slot
  PAGED_CODE Slots in(int head, const Quota& quota) const {
    if (!tiles || !quota.many) return Slots{0, 0};
    const int from = t0 + head * span, range = quota.range(from);
    return Slots{item + head * items + range, quota.range(from + tiles - 1) - range + 1};
  }
};
PAGED_CODE TokenSlots token_slots(const Extents& e, const Request& r, int b, const int32_t* start, int items,
                                  int token) {
  TokenSlots s{start[b], 0, start[e.requests + 1], 0, 0, 0};
  if (!r.count || !r.keys) return s;
  const int i = token - r.first, tile = r.narrow ? 0 : i / e.per;
  s.tiles = item_tiles(e, r, tile);
  s.item = item_number(e, r, b, tile);
  s.items = items;
  if (!r.narrow) s.t0 += wide_begin(e, r, tile) + e.cost;
  s.row = (i - (r.narrow ? 0 : tile * e.per)) * e.share;
  return s;
}

}  // namespace tensor_paged
