"""How a paged attention call is shared out (csrc/paged_plan.h), compiled as plain host code (CPU only).

Every segment of every workgroup and wave is walked as the kernels walk them: each key tile of each
item is taken once, slots are within the workspace and used once, and the slots that the joining kernel
reads for a row are those that its segments wrote.
"""

from __future__ import annotations

import ctypes as c
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "tensor_amd" / "csrc"
SOURCE = r"""
#include <map>
#include <set>
#include <vector>
#include "paged_plan.h"
using namespace tensor_paged;

extern "C" unsigned sum_floor(unsigned n, unsigned m, unsigned a, unsigned b) { return floor_sum(n, m, a, b); }

struct Item { int list, b, head, tile; bool operator<(const Item& o) const {
  return list != o.list ? list < o.list : b != o.b ? b < o.b : head != o.head ? head < o.head : tile < o.tile; } };

// 0, or the line that found a fault
#define NEED(...) if (!(__VA_ARGS__)) return __LINE__
int leads = 0;
extern "C" int led() { return leads; }
extern "C" int walk(int tokens, int requests, int heads, int kv, int shift, int columns, int prefix_columns, const int* offsets,
                    const int* lengths, int prefix_length, int monotone) {
  Extents e = extents(tokens, requests, heads, kv, shift, columns, prefix_columns);
  Request prefix = prefix_request(e, offsets[requests], prefix_length);
  auto request = [&](int b) { return b == requests ? prefix : own_request(e, offsets[b], offsets[b + 1], lengths[b]); };
  int64_t items = 0;
  bool apart = false;
  for (int b = 0; b < requests; ++b) {
    const Request r = request(b);
    apart |= r.count && (r.narrow || !r.keys);
    items += head_items(e, r);
  }
  e.lead = apart || !monotone ? 0 : lead_tiles(e, prefix, (int)items);
  if (e.lead) {
    NEED(e.lead == (prefix.keys + kWideKeys - 1) / kWideKeys);
    NEED((items - row_tiles(e, prefix)) * e.lead <= (int64_t)row_tiles(e, prefix) * kSlotCost);
    prefix.count = prefix.keys = 0;
    ++leads;
  }
  int64_t all = 0;
  for (int b = 0; b <= requests; ++b) all += (int64_t)kv * head_items(e, request(b));
  e.cost = item_cost((int)all);
  std::vector<int32_t> starts[2];
  int64_t done[2] = {0, 0};
  for (int b = 0; b <= requests; ++b) {
    const Request r = request(b);
    NEED(r.first >= 0 && r.count >= 0 && r.first + r.count <= tokens);
    NEED(r.keys >= 0 && r.keys <= (int64_t)(r.prefix ? prefix_columns : columns) << shift);
    for (int k = 0; k < 2; ++k) starts[k].push_back(done[k]);
    done[r.narrow] += head_span(e, r);
  }
  NEED(kv * (done[0] + done[1]) + 2 * kStreams <= most_tiles(e) && most_tiles(e) < (int64_t)1 << 31);
  std::map<Item, std::vector<int64_t>> slots;  // slots of an item's segments, in order
  std::map<Item, int> reached;
  std::set<int64_t> used[2];
  Quota quota[2];
  for (int k = 0; k < 2; ++k) {
    starts[k].push_back(done[k]);
    done[k] *= kv;
    const int ranges = k ? kStreams : kGroups;
    quota[k] = k ? narrow_quota((int)done[1], quota[0].many) : wide_quota((int)done[0], (int)done[1] * kv);
    NEED(quota[k].begin(ranges) >= done[k] && (quota[k].few >= 0) == (k == 1));
    for (int range = 0; range < ranges; ++range) {
      const int64_t from = quota[k].begin(range), to = least(quota[k].begin(range + 1), (int)done[k]);
      if (from >= to) continue;
      NEED(quota[k].range((int)from) == range && quota[k].range((int)to - 1) == range);
      Walk<decltype(request)> walk(e, starts[k].data(), request, k ? narrow_items(e) : wide_items(e), (int)from, (int)to);
      Segment s;
      int taken = 0;
      for (; walk.next(s); walk.advance()) {
        const Request r = walk.r;
        NEED(r.narrow == (k == 1) && s.head >= 0 && s.head < kv && s.tile >= 0 && s.t0 >= 0 && s.t1 > s.t0);
        NEED(r.narrow ? s.tile == 0 : s.tile < row_tiles(e, r));
        NEED(s.t1 <= item_tiles(e, r, s.tile));
        const int64_t slot = s.item + range;
        NEED(slot >= 0 && slot < (k ? narrow_slots(e) : wide_slots(e)));
        if (monotone) NEED(used[k].insert(slot).second);
        const Item item{k, walk.b, s.head, s.tile};
        NEED(reached[item] == s.t0);
        reached[item] = s.t1;
        slots[item].push_back(slot);
        NEED(s.all == (slots[item].size() == 1 && s.t1 == item_tiles(e, r, s.tile)));
        taken += s.t1 - s.t0;
      }
      NEED(taken <= to - from);
    }
  }
  for (int b = 0; b <= requests; ++b) {
    const Request r = request(b);
    for (int i = 0; i < r.count; i += (r.count > 300 ? 7 : 1))
      for (int head = 0; head < kv; ++head) {
        const int tile = r.narrow ? 0 : i / e.per, k = r.narrow, share = heads / kv;
        // the tiles of the item reach all keys that the token sees
        const int sees = r.prefix ? r.keys : least(r.keys, most(0, r.behind + i + 1));
        const auto at = reached.find(Item{k, b, head, tile});
        if (r.keys == 0) { NEED(at == reached.end()); }
        else NEED(at != reached.end() && (int64_t)(at->second - (r.prefix ? 0 : e.lead)) * (k ? kNarrowKeys : kWideKeys) >= sees);
        const TokenSlots rows = token_slots(e, r, b, starts[k].data(), k ? narrow_items(e) : wide_items(e), r.first + i);
        const Slots s = rows.in(head, quota[k]);
        NEED(!rows.tiles || rows.row + share <= (k ? kNarrowRows : kWideRows));
        const auto& wrote = slots[Item{k, b, head, tile}];
        NEED(s.count == (int)wrote.size());
        if (s.count) {
          NEED(reached[Item{k, b, head, tile}] == rows.tiles);
        }
        for (int n = 0; n < s.count; ++n) NEED(wrote[n] == s.first + n);
      }
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    folder = tmp_path_factory.mktemp("paged_plan")
    (folder / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-shared", "-fPIC", "-I", str(CSRC), str(folder / "plan.cpp"), "-o", str(folder / "plan.so")],
                   check=True, capture_output=True)
    return c.CDLL(str(folder / "plan.so"))


def test_floor_sum(library):
    rng = random.Random(1)
    for _ in range(300):
        n, m, a, b = rng.randint(0, 200), rng.choice((32, 64)), rng.randint(1, 200), rng.randint(0, 100000)
        assert library.sum_floor(n, m, a, b) == sum((a * i + b) // m for i in range(n)), (n, m, a, b)


def walk(library, tokens, heads, kv, shift, columns, prefix_columns, offsets, lengths, prefix, monotone=1):
    return library.walk(tokens, len(lengths), heads, kv, shift, columns, prefix_columns, (c.c_int * len(offsets))(*offsets),
                        (c.c_int * len(lengths))(*lengths), prefix, monotone)


def call(rng):
    heads, kv = rng.choice(((32, 8), (16, 16), (28, 4), (16, 1), (24, 8), (128, 1), (5, 5), (17, 1)))
    requests = rng.choice((1, 2, 3, 17, 64, 300))
    counts = [rng.choice((0, 1, 1, 1, rng.randint(0, 9), rng.randint(0, 400) if rng.random() < 8 / requests else 1))
              for _ in range(requests)]
    if not any(counts):
        counts[0] = 1
    shift = rng.choice((0, 3, 4, 6))
    lengths = [n + rng.choice((0, 0, rng.randint(0, 3000))) for n in counts]
    prefix = rng.choice((0, 0, rng.randint(1, 5000)))
    offsets = [0]
    for n in counts:
        offsets.append(offsets[-1] + n)
    columns = -(-max(1, *lengths, 1) // (1 << shift)) + rng.randint(0, 3)
    return heads, kv, shift, columns, max(1, -(-prefix // (1 << shift))), offsets, lengths, prefix


@pytest.mark.parametrize("seed", range(60))
def test_segments_cover_every_item_once(library, seed):
    rng = random.Random(seed)
    heads, kv, shift, columns, prefix_columns, offsets, lengths, prefix = call(rng)
    tokens = offsets[-1] + rng.choice((0, 0, 5))
    assert walk(library, tokens, heads, kv, shift, columns, prefix_columns, offsets, lengths, prefix) == 0


@pytest.mark.parametrize("seed", range(30))
def test_prefix_leads_the_items_of_prompts(library, seed):
    rng = random.Random(500 + seed)
    heads, kv = rng.choice(((32, 8), (16, 16), (28, 4), (16, 1), (5, 5)))
    requests = rng.choice((1, 2, 3, 17))
    counts = [rng.choice((rng.randint(20, 90), 128, rng.randint(200, 600))) for _ in range(requests)]
    if rng.random() < 0.3:
        counts[rng.randrange(requests)] = 0
        counts.append(40)
    shift = rng.choice((0, 4, 6))
    lengths = [n + rng.choice((0, 0, rng.randint(0, 3000))) for n in counts]
    prefix = rng.choice((1, 63, 64, 65, rng.randint(100, 5000)))
    offsets = [sum(counts[:b]) for b in range(len(counts) + 1)]
    columns = -(-max(lengths) // (1 << shift))
    before = library.led()
    assert walk(library, offsets[-1], heads, kv, shift, columns, -(-prefix // (1 << shift)), offsets, lengths, prefix) == 0
    if len(counts) == 1 and counts[0] * (heads // kv) > 16:
        assert library.led() == before + 1


@pytest.mark.parametrize("seed", range(40))
def test_malformed_offsets_and_lengths_stay_in_bounds(library, seed):
    """Offsets out of order or range, lengths below the new tokens or past the table: the extents still hold."""
    rng = random.Random(1000 + seed)
    heads, kv, shift, columns, prefix_columns, offsets, lengths, prefix = call(rng)
    tokens = max(1, offsets[-1] - rng.randint(0, 3))
    for _ in range(4):
        offsets[rng.randrange(len(offsets))] = rng.choice((-1, 0, tokens, tokens + 9, 2 ** 31 - 1, -2 ** 31, rng.randint(0, tokens)))
        lengths[rng.randrange(len(lengths))] = rng.choice((-1, 0, 1, -2 ** 31, 2 ** 31 - 1 if shift == 0 or columns < 4000 else 5))
    prefix = rng.choice((prefix, -1, 2 ** 31 - 1))
    assert walk(library, tokens, heads, kv, shift, columns, prefix_columns, offsets, lengths, prefix, 0) == 0
