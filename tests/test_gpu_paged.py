"""The paged-cache operators on a GPU against their plain forms in 64 bits (tests/paged_cases.py)."""

from __future__ import annotations

import numpy as np
import pytest

from tensor_amd.kernels.paged import rotary_angles
from tests import paged_cases as plain

pytestmark = pytest.mark.gpu


class Buffers:
    """Device buffers of a test, released at its end; outputs start as NaN (all bits set)."""

    def __init__(self, device):
        self.device, self.all = device, []

    def __call__(self, array):
        self.all.append(self.device.from_numpy(array))
        return self.all[-1]

    def empty(self, shape, dtype):
        self.all.append(self.device.empty(shape, dtype))
        self.device.fill_bytes(self.all[-1], 0xFF)
        return self.all[-1]

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for buffer in self.all:
            buffer.release()


# ------------------------------------------------------------------- slots

def run_slots(device, lengths, counts, start, free, free_count, table, tokens, page):
    with Buffers(device) as put:
        kernel = device.load("paged_slots", page_size=page)
        out = kernel(*(put(np.asarray(v, np.int32)) for v in (lengths, counts, [start], free, [free_count], table)), tokens)
        result = tuple(o.to_numpy() for o in out)
        for o in out:
            o.release()
        return result


def check_slots(device, *args):
    for name, got, want in zip(("offsets", "lengths", "positions", "slots", "table", "left"), run_slots(device, *args),
                               plain.slots(*args)):
        assert np.array_equal(got, want), (name, got, want)


@pytest.mark.parametrize("seed", range(12))
def test_slots(hip_device, seed):
    rng = np.random.default_rng(seed)
    page = int(rng.choice([1, 2, 8, 16, 64, 1024]))
    requests, columns = int(rng.choice([1, 2, 7, 63, 300])), int(rng.integers(1, 90))
    lengths = rng.integers(0, page * columns, requests)
    lengths[rng.random(requests) < 0.3] = 0
    lengths[rng.random(requests) < 0.3] //= page
    counts = np.where(rng.random(requests) < 0.5, 1, rng.integers(0, 40, requests))
    pages = 4 * requests * columns + 7
    free = rng.permutation(pages)[:requests * 45 + 3]
    table = rng.integers(0, pages, (requests, columns))
    total = int(counts.sum())
    for tokens in {max(1, total), max(1, total + 5), max(1, total - 2)}:  # whole, padded, cut off
        for free_count in (len(free), int(rng.integers(0, 5)), 0):  # enough pages, few, none
            check_slots(hip_device, lengths, counts, int(rng.integers(0, 1000)), free, free_count, table, tokens, page)


def test_slots_edges(hip_device):
    table = np.arange(8).reshape(2, 4)
    # nothing new but padding; negative lengths and counts; a count of free pages past the list's end
    check_slots(hip_device, [5, 0], [0, 0], 3, [90, 91], 2, table, 1, 4)
    check_slots(hip_device, [-5, -1], [3, -7], 0, [90, 91], 2, table, 4, 4)
    check_slots(hip_device, [4, 8], [1, 1], 0, [90, 91], 50, table, 2, 4)
    check_slots(hip_device, [4, 8], [1, 1], 0, [90, 91], -3, table, 2, 4)
    # tokens past the table's last column, and a held page that is missing
    check_slots(hip_device, [14, 16], [5, 2], 9, [90, 91, 92], 3, table, 7, 4)
    check_slots(hip_device, [6, 1], [1, 1], 0, [90], 1, np.array([[3, -1, -1, -1], [-1, -1, -1, -1]]), 2, 4)


def test_slots_of_pages_past_int32(hip_device):
    """A page whose slots int32 does not hold gives none, not those of another page; the last that fits has its own."""
    page = 1024
    fits, wraps = (1 << 21) - 1, (1 << 22) + 1  # the latter's slots would wrap to page 1's
    table = np.array([[fits, -1], [wraps, -1], [1 << 21, -1]])
    _, _, positions, slots, out, left = run_slots(hip_device, [1023, 5, 0], [2, 1, 1], 0, [wraps, 1 << 21], 2, table, 4, page)
    assert slots.tolist() == [2 ** 31 - 1, -1, -1, -1]
    assert positions.tolist() == [1023, 1024, 5, 0]
    assert out.tolist() == [[fits, 1 << 21], [wraps, -1], [wraps, -1]] and left.tolist() == [0]


def test_slots_share_a_long_prompt_and_a_wide_table(hip_device):
    rng = np.random.default_rng(5)
    table = rng.integers(0, 1 << 20, (3, 9001))
    check_slots(hip_device, [17, 100000, 0], [30011, 1, 4097], 11, rng.permutation(4000), 4000, table, 34109 + 3, 16)


def test_slots_step_by_step_fill_pages(hip_device):
    """Thirty steps fed with their own outputs: every token has a slot of its own."""
    page, requests = 4, 5
    lengths, table = np.zeros(requests, np.int32), np.full((requests, 16), -1, np.int32)
    free, left = np.random.default_rng(1).permutation(64).astype(np.int32), 64
    used = set()
    for step in range(30):
        counts = np.array([(step + b) % 3 for b in range(requests)], np.int32)
        total = int(counts.sum())
        offsets, lengths, positions, slots, table, remaining = run_slots(
            hip_device, lengths, counts, 7, free, left, table, total, page)
        left = int(remaining[0])
        assert left >= 0 and (slots >= 0).all() and not used & set(slots.tolist()) and len(set(slots.tolist())) == total
        used |= set(slots.tolist())
        assert offsets[-1] == total
    assert (lengths == 30).all() and left == 64 - requests * 8


# ------------------------------------------------------------------ rotary

SHAPES = [  # tokens, heads, key heads, dim, rotated
    (1, 1, 1, 2, 2), (3, 5, 5, 6, 4), (7, 32, 8, 128, 128), (2, 4, 2, 128, 64), (5, 3, 1, 80, 32), (4, 8, 1, 96, 46),
    (3, 2, 2, 33, 30), (6, 28, 4, 64, 16), (2, 300, 7, 64, 64), (130, 4, 4, 256, 256),
]


def bound_rotary(x, angles, dtype):
    """One rounding of the output (2^-11 in fp16, 2^-24 in fp32, of values up to |a| + |b|) and two fp32
    roundings of the products and their sum, of at most (|a| + |b|) times the largest cosine."""
    size = 2.0 * np.abs(x.astype(np.float64)).max(axis=-1, keepdims=True) * max(1.0, np.abs(angles).max())
    return size * ((2.0 ** -11 if dtype == "float16" else 2.0 ** -24) + 2.0 ** -23) + 2.0 ** -25


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotary(hip_device, shape, dtype, layout):
    tokens, heads, kv, dim, rotated = shape
    rng = np.random.default_rng(tokens)
    angles = rotary_angles(50, rotated)
    q, k = (rng.standard_normal((tokens, n, dim)).astype(dtype) for n in (heads, kv))
    positions = rng.integers(0, 50, tokens).astype(np.int32)
    if tokens > 2:
        positions[:3] = (-1, 49, 50)  # padding, the last row, past the table
    for inverse in (False, True):
        with Buffers(hip_device) as put:
            kernel = hip_device.load("rotary", layout=layout, dtype=dtype, inverse=inverse)
            outs = [put.empty(x.shape, dtype) for x in (q, k)]
            kernel.launch(put(q), put(k), put(positions), put(angles), *outs)
            for x, out in zip((q, k), outs):
                got, want = out.to_numpy().astype(np.float64), plain.rotary(x, positions, angles, layout, inverse)
                assert np.array_equal(np.isnan(got), np.isnan(want))
                assert (np.abs(got - want) <= bound_rotary(x, angles, dtype))[~np.isnan(want)].all()
                assert np.array_equal(got[..., rotated:][want[..., rotated:] == 0], want[..., rotated:][want[..., rotated:] == 0])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_inverse_is_the_gradient(hip_device, layout):
    """The gradient of sum(g * rotary(x)) is the inverse rotation of g: against differences of the 64-bit
    form (the map is linear: central differences are exact but for rounding) along every dimension."""
    rng = np.random.default_rng(3)
    tokens, heads, dim, rotated = 4, 2, 32, 24
    angles = rotary_angles(9000, rotated, base=500.0)
    positions = np.array([0, 1, 77, 8999], np.int32)
    x, g = (rng.standard_normal((tokens, heads, dim)).astype(np.float32) for _ in range(2))
    with Buffers(hip_device) as put:
        kernel = hip_device.load("rotary", layout=layout, dtype="float32", inverse=True)
        out = [put.empty(g.shape, "float32") for _ in range(2)]
        kernel.launch(put(g), put(g), put(positions), put(angles), *out)
        gradient = out[0].to_numpy()
    for d in range(dim):
        step = np.zeros_like(x, np.float64)
        step[..., d] = 0.5
        change = (g * (plain.rotary(x + step, positions, angles, layout) - plain.rotary(x - step, positions, angles, layout))).sum(-1)
        assert np.abs(gradient[..., d] - change).max() <= 1e-5


def test_rotary_in_place(hip_device):
    """Every value is read before its pair is written: outputs may be the inputs."""
    rng = np.random.default_rng(4)
    angles, positions = rotary_angles(64, 128), rng.integers(0, 64, 9).astype(np.int32)
    q, k = (rng.standard_normal((9, n, 128)).astype(np.float16) for n in (6, 2))
    with Buffers(hip_device) as put:
        kernel = hip_device.load("rotary")
        bq, bk = put(q), put(k)
        kernel.launch(bq, bk, put(positions), put(angles), bq, bk)
        for x, out in ((q, bq), (k, bk)):
            assert (np.abs(out.to_numpy() - plain.rotary(x, positions, angles, "half")) <= bound_rotary(x, angles, "float16")).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("shape,page", [((7, 32, 8, 128, 128), 16), ((5, 3, 1, 80, 32), 1), ((6, 28, 4, 64, 16), 8),
                                        ((4, 8, 1, 96, 46), 1024), ((130, 4, 4, 64, 64), 32)], ids=str)
def test_rotary_store(hip_device, shape, page, dtype, layout):
    tokens, heads, kv, dim, rotated = shape
    rng = np.random.default_rng(page)
    angles = rotary_angles(500, rotated, base=1e5, scaling="linear", factor=3.0)
    q, k, v = (rng.standard_normal((tokens, n, dim)).astype(dtype) for n in (heads, kv, kv))
    pages = -(-tokens // page) + 2
    positions = rng.integers(0, 500, tokens).astype(np.int32)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    positions[0] = -1
    slots[1], slots[2], slots[3] = -1, pages * page, 2 ** 31 - 1  # nowhere: nothing may be stored
    caches = [rng.standard_normal((pages, kv, page, dim)).astype(np.float16) for _ in range(2)]
    with Buffers(hip_device) as put:
        kernel = hip_device.load("rotary_store", layout=layout, dtype=dtype)
        q_out, stored = put.empty(q.shape, "float16"), [put(cache) for cache in caches]
        kernel.launch(put(q), put(k), put(v), put(positions), put(slots), put(angles), q_out, *stored)
        got_q, got_k, got_v = (b.to_numpy() for b in (q_out, *stored))
    bound = bound_rotary(q, angles, "float16")
    assert (np.abs(got_q - plain.rotary(q, positions, angles, layout)) <= bound).all()
    turned, touched = plain.rotary(k, positions, angles, layout), np.zeros((pages, page), bool)
    for t, slot in enumerate(slots):
        if 0 <= slot < pages * page:
            touched[slot // page, slot % page] = True
            where = (slot // page, slice(None), slot % page)
            assert (np.abs(got_k[where] - turned[t]) <= bound_rotary(k, angles, "float16")[t]).all()
            assert np.array_equal(got_v[where], v[t].astype(np.float16))
    for got, was in ((got_k, caches[0]), (got_v, caches[1])):  # every other place is as it was
        assert np.array_equal(got.transpose(0, 2, 1, 3)[~touched], was.transpose(0, 2, 1, 3)[~touched])


# --------------------------------------------------------------- attention

def run_attention(device, q, k_cache, v_cache, offsets, lengths, table, prefix_pages, prefix_length, scale=None):
    tokens, heads, dim = q.shape
    need = device.attention_workspace(tokens, len(lengths), heads, k_cache.shape[1], dim)
    with Buffers(device) as put:
        kernel = device.load("paged_attention") if scale is None else device.load("paged_attention", scale=scale)
        out, workspace = put.empty(q.shape, "float16"), put.empty((need,), "uint8")
        kernel.launch(put(q), put(k_cache), put(v_cache), put(np.asarray(offsets, np.int32)),
                      put(np.asarray(lengths, np.int32)), put(np.asarray(table, np.int32)),
                      put(np.asarray(prefix_pages, np.int32)), put(np.asarray([prefix_length], np.int32)), workspace, out)
        return out.to_numpy().astype(np.float64)


def make(rng, counts, lengths, prefix, heads, kv, dim, page, sharp=1.0, padding=0):
    """Inputs of a call; every place of the cache that no request reads holds NaN."""
    table, prefix_pages, pages = plain.paging(rng, lengths, page, prefix)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = (sharp * rng.standard_normal((offsets[-1] + padding, heads, dim))).astype(np.float16)
    caches = np.full((2, pages, kv, page, dim), np.nan, np.float16)
    for pages_of, count in [(row, n) for row, n in zip(table, lengths)] + [(prefix_pages, prefix)]:
        for at in range(count):
            caches[:, pages_of[at // page], :, at % page] = rng.standard_normal((2, kv, dim))
    return [q, caches[0], caches[1], offsets, np.asarray(lengths, np.int32), table, prefix_pages, prefix]


def check_attention(device, call, scale=None):
    want, bound = plain.attention(*call, scale=scale)
    got = run_attention(device, *call, scale=scale)
    assert np.isfinite(want).all()
    over = np.abs(got - want) - bound
    assert (over <= 0).all(), (np.unravel_index(np.nanargmax(over), over.shape), np.nanmax(over), np.isnan(got).sum())


HEADS = [(4, 1), (2, 2), (8, 2), (7, 1), (6, 2), (16, 1), (24, 1)]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_attention_of_single_tokens(hip_device, heads, dim):
    """Decode: lengths around the key tiles (32, 64), with and without a prefix around them."""
    rng = np.random.default_rng(dim + heads[0])
    lengths = [1, 2, 31, 32, 33, 63, 64, 65, 127, 200]
    for prefix in (0, 1, 64, 131):
        check_attention(hip_device, make(rng, [1] * len(lengths), lengths, prefix, *heads, dim, 16, sharp=2.0))


@pytest.mark.parametrize("page", [1, 2, 8, 32, 64, 128, 1024])
def test_attention_page_sizes(hip_device, page):
    rng = np.random.default_rng(page)
    check_attention(hip_device, make(rng, [1, 3, 40], [70, 131, 90], 97, 4, 2, 64, page))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [(4, 1), (2, 2), (7, 1), (6, 2)], ids=str)
def test_attention_of_many_tokens(hip_device, heads, dim):
    """Prompts and drafted tokens mixed with decode: row tiles of whole tokens end inside requests, the causal
    edge runs through key tiles, requests without new tokens and rows past the last request."""
    rng = np.random.default_rng(dim * heads[0])
    counts = [1, 0, 5, 17, 64, 1, 33, 2, 0]
    lengths = [9, 12, 5, 17, 100, 130, 70, 2, 0]
    for prefix in (0, 40):
        call = make(rng, counts, lengths, prefix, *heads, dim, 16, padding=3)
        check_attention(hip_device, call)
        assert (run_attention(hip_device, *call)[-3:] == 0).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("counts,lengths", [([40], [40]), ([33, 0, 64, 130], [50, 7, 64, 300]), ([90, 5, 64], [90, 0, 9])], ids=str)
def test_attention_of_prompts_behind_a_prefix(hip_device, counts, lengths, dim):
    """Requests that fill row tiles of their own: prefixes that end at a key tile and beside one; tokens without own keys."""
    rng = np.random.default_rng(dim + sum(counts))
    for prefix in (1, 63, 64, 65, 300):
        call = make(rng, counts, lengths, prefix, 8, 1, dim, 16, padding=2)
        check_attention(hip_device, call)
        call[6][prefix // 32] = -1  # a page of the prefix that is not there
        check_attention(hip_device, call)


def test_attention_offsets_that_do_not_ascend_leave_zeros(hip_device):
    rng = np.random.default_rng(21)
    call = make(rng, [3, 40, 1], [9, 50, 70], 30, 4, 1, 64, 16)
    for offsets in ([0, 43, 3, 44], [0, 3, 43, 42], [0, 2 ** 31 - 1, -1, 44]):
        call[3] = np.array(offsets, np.int32)
        assert (run_attention(hip_device, *call) == 0).all()


def test_attention_long_and_short_requests_share_a_call(hip_device):
    rng = np.random.default_rng(2)
    lengths = [4000, 1, 90, 700, 3, 1500]
    check_attention(hip_device, make(rng, [1, 1, 90, 130, 3, 2], lengths, 1000, 4, 1, 64, 16))


def test_attention_of_128_query_heads_on_one_key_head(hip_device):
    check_attention(hip_device, make(np.random.default_rng(8), [1, 3], [77, 40], 66, 128, 1, 64, 16))


def test_attention_many_requests(hip_device):
    """More requests than threads of a workgroup, most of a key or two."""
    rng = np.random.default_rng(9)
    lengths = [int(n) for n in rng.integers(1, 6, 600)]
    check_attention(hip_device, make(rng, [1] * 600, lengths, 5, 2, 1, 64, 8))


def test_attention_sharp_scores_and_scales(hip_device):
    """Scores of hundreds: the running maximum moves from tile to tile, most weights vanish."""
    rng = np.random.default_rng(10)
    call = make(rng, [1, 40], [300, 200], 150, 4, 2, 64, 16, sharp=40.0)
    check_attention(hip_device, call)
    check_attention(hip_device, call, scale=0.02)
    call[1][...] = np.where(np.isnan(call[1]), call[1], 1.0)  # equal keys: the mean of the values
    check_attention(hip_device, call, scale=3.0)


def test_attention_rising_and_falling_maxima(hip_device):
    """Keys whose scores rise (or fall) all along: the maximum passes the step at which sums are rescaled
    between any two tiles, or never."""
    rng = np.random.default_rng(11)
    for sign in (1.0, -1.0):
        call = make(rng, [1, 30], [500, 333], 70, 2, 1, 64, 16)
        call[0][...] = 0.5
        for row, n in ((call[5][0], 500), (call[5][1], 333)):
            for at in range(n):
                call[1][row[at // 16], :, at % 16] = sign * at / 200.0
        check_attention(hip_device, call)


def test_attention_rows_without_keys(hip_device):
    """No prefix and no own keys: zeros.  A length below the new tokens leaves the first of them without keys."""
    rng = np.random.default_rng(12)
    call = make(rng, [1, 4, 1], [3, 4, 5], 0, 4, 1, 64, 8)
    call[4][0] = 0
    check_attention(hip_device, call)
    assert (run_attention(hip_device, *call)[0] == 0).all()
    call[4][1] = 2  # four tokens, two keys
    check_attention(hip_device, call)
    assert (run_attention(hip_device, *call)[1:3] == 0).all()
    for count in (30, 70):
        call = make(rng, [count, 1], [count, 5], 0, 4, 1, 64, 8)
        call[4][0] = 9
        check_attention(hip_device, call)


@pytest.mark.parametrize("bad", [-1, -7, 2 ** 31 - 1, 10 ** 6])
def test_attention_entries_that_are_no_pages_hide_their_keys(hip_device, bad):
    rng = np.random.default_rng(13)
    call = make(rng, [1, 40, 1], [100, 90, 20], 50, 4, 1, 64, 16)
    call[5][0, 2] = call[5][1, 1] = call[6][1] = bad
    check_attention(hip_device, call)
    call[5][2, :] = bad  # a request whose every page is missing: the prefix alone
    check_attention(hip_device, call)


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("counts,lengths", [([4], [70]), ([40], [100]), ([3, 70], [3, 70])], ids=str)
def test_attention_keeps_hidden_values_out(hip_device, counts, lengths, value):
    """Keys or values that are not finite at a late token reach the tokens that see it and no others."""
    rng = np.random.default_rng(14)
    clean = make(rng, counts, lengths, 20, 4, 1, 64, 16)
    want, bound = plain.attention(*clean)
    b, place, d = len(counts) - 1, lengths[-1] - 2, 5  # the last token but one of the last request
    page = clean[5][b, place // 16]
    before = int(clean[3][-1]) - 2  # rows before it see nothing of it
    for which in (1, 2):
        call = [x.copy() if isinstance(x, np.ndarray) else x for x in clean]
        call[which][page, 0, place % 16, d] = value
        got = run_attention(hip_device, *call)
        assert (np.abs(got - want)[:before] <= bound[:before]).all()
        if which == 2:  # the dimension of the value, in the rows that see it
            expected = np.full((2, 4), value)
            assert np.array_equal(got[before:, :, d], expected, equal_nan=True)
            rest = np.delete(got[before:], d, axis=2)
            assert (np.abs(rest - np.delete(want[before:], d, axis=2)) <= np.delete(bound[before:], d, axis=2)).all()


def test_attention_results_repeat(hip_device):
    """No order of arrival enters a result."""
    rng = np.random.default_rng(15)
    call = make(rng, [1] * 20 + [50], [int(n) for n in rng.integers(1, 900, 20)] + [60], 700, 8, 2, 128, 16)
    first = run_attention(hip_device, *call)
    for _ in range(3):
        assert np.array_equal(run_attention(hip_device, *call), first)


def test_attention_past_32_bits(hip_device):
    """A cache of more than 2^32 values: slots at its end are written by rotary_store and read back."""
    kv, page, dim, heads = 8, 1024, 128, 8
    pages = (1 << 32) // (kv * page * dim) + 40
    rng = np.random.default_rng(16)
    tokens, columns = 70, 1
    q, k, v = (rng.standard_normal((tokens, n, dim)).astype(np.float16) for n in (heads, kv, kv))
    angles = np.concatenate([np.ones((1, 8)), np.zeros((1, 8))], 1).astype(np.float32)  # no rotation
    with Buffers(hip_device) as put:
        caches = [hip_device.empty((pages, kv, page, dim), "float16") for _ in range(2)]
        put.all += caches
        slots = ((pages - 1) * page + np.arange(tokens)).astype(np.int32)
        store = hip_device.load("rotary_store")
        store.launch(put(q), put(k), put(v), put(np.zeros(tokens, np.int32)), put(slots), put(angles),
                     put.empty(q.shape, "float16"), *caches)
        attend = hip_device.load("paged_attention")
        for counts, lengths in (([1], [tokens]), ([tokens], [tokens])):
            offsets = np.array([0, counts[0]], np.int32)
            workspace = put.empty((hip_device.attention_workspace(counts[0], 1, heads, kv, dim),), "uint8")
            out = put.empty((counts[0], heads, dim), "float16")
            attend.launch(put(q[-counts[0]:]), *caches, put(offsets), put(np.array(lengths, np.int32)),
                          put(np.full((1, columns), pages - 1, np.int32)), put(np.zeros(1, np.int32)),
                          put(np.zeros(1, np.int32)), workspace, out)
            small = [x.transpose(1, 0, 2)[None] for x in (k, v)]
            small = [np.concatenate([s, np.zeros((1, kv, page - tokens, dim), np.float16)], 2) for s in small]
            want, bound = plain.attention(q[-counts[0]:], *small, offsets, lengths, np.zeros((1, 1), np.int32),
                                          np.zeros(1, np.int32), 0)
            assert (np.abs(out.to_numpy() - want) <= bound).all()


def test_decode_steps_in_a_graph_follow_the_lengths(hip_device):
    """One captured graph of slots, store and attention, replayed while lengths grow on the device; the
    program's own work and synchronizations stand between replays."""
    page, kv, heads, dim, requests, prefix = 8, 2, 8, 64, 3, 21
    rng = np.random.default_rng(17)
    angles = rotary_angles(100, dim)
    pages, columns = 60, 8
    cache = np.full((2, pages, kv, page, dim), np.nan, np.float16)
    prefix_pages = np.array([50, 9, 33], np.int32)
    for at in range(prefix):
        cache[:, prefix_pages[at // page], :, at % page] = rng.standard_normal((2, kv, dim))
    free = np.array([p for p in rng.permutation(pages) if p not in prefix_pages], np.int32)
    counts = np.ones(requests, np.int32)
    with Buffers(hip_device) as put:
        lengths, table, left = put(np.zeros(requests, np.int32)), put(np.full((requests, columns), -1, np.int32)), put(np.array([len(free)], np.int32))
        after, table_after, left_after = put(np.zeros(requests, np.int32)), put.empty((requests, columns), "int32"), put.empty((1,), "int32")
        offsets, positions, slots = put.empty((requests + 1,), "int32"), put.empty((requests,), "int32"), put.empty((requests,), "int32")
        q, k, v = (put(np.zeros((requests, n, dim), np.float16)) for n in (heads, kv, kv))
        turned, out = put.empty((requests, heads, dim), "float16"), put.empty((requests, heads, dim), "float16")
        caches = [put(c) for c in cache]
        start, table_angles, stack, count = put(np.array([prefix], np.int32)), put(angles), put(free), put(counts)
        shared = put(prefix_pages)
        workspace = put.empty((hip_device.attention_workspace(requests, requests, heads, kv, dim),), "uint8")
        plan = hip_device.load("paged_slots", page_size=page).bind(
            lengths, count, start, stack, left, table, requests, offsets, after, positions, slots, table_after, left_after)
        store = hip_device.load("rotary_store").bind(q, k, v, positions, slots, table_angles, turned, *caches)
        attend = hip_device.load("paged_attention").bind(turned, *caches, offsets, after, table_after, shared, start, workspace, out)

        def step():
            plan.launch()
            store.launch()
            attend.launch()

        step()  # eager once; the state is put back
        hip_device.synchronize()
        for buffer, array in zip(caches, cache):
            hip_device.upload(buffer, array)
        graph = hip_device.graph(step)
        for _ in range(19):
            for buffer, n in ((q, heads), (k, kv), (v, kv)):
                hip_device.upload(buffer, rng.standard_normal((requests, n, dim)).astype(np.float16))
            graph.replay()
            hip_device.synchronize()
            now = [b.to_numpy() for b in (turned, *caches, offsets, after, table_after)]
            want, bound = plain.attention(*now, prefix_pages, prefix)
            assert (np.abs(out.to_numpy() - want) <= bound).all()
            hip_device.upload(lengths, now[4])
            hip_device.upload(table, now[5])
            hip_device.upload(left, left_after.to_numpy())
        assert (after.to_numpy() == 19).all() and int(left_after.to_numpy()[0]) == len(free) - requests * 3
        if hasattr(graph, "release"):
            graph.release()
