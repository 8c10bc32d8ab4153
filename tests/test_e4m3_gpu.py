"""A cache in 8 bits against its definition in 64 bits (``plain_e4m3``): the store with the rotation on the way, and the attention
that reads it, for single tokens and portions of prompts.

Tolerances.  A code is half a step off at most: 2^-4 of its value, 2^-10 below the normal range.  Scales, and codes of rows that do
not turn (16-bit rows over a power of two are exact in 32 bits), are equal.  A turned entry comes from two products of 32-bit numbers and an
angle that is exact to 2^-24 turns: some 2^-21 of its pair, which is 448 scales at most.

Attention in bfloat16: 2^-8 of the result for its own rounding, and of the sum of the weights times |v| 2^-11 for the
weights, which are 16-bit floats, and 2^-20 (1 + size) for the scores: a score of products of sum `size` is some 8 sums cut off
at 2^-23, its 32-bit arithmetic and the exponential a few units of 2^-24 of it, and an error of a score is as
large a relative one of its weight.  A weight (times its value's scale) below 2^-14 of a 16-bit float's scale is off by half of 2^-24 whatever
its size; the largest lies at 2^7 or above: 2^-32 of the largest for each key, times a code of 448 at most.  With 32-bit queries sums of
N terms, each rounded to 2^-24, and weights down to 2^-126."""

import numpy as np
import pytest
import torch

import plain_e4m3 as plain

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def scattered_table(reaches, page, rng, spare=2):
    """Block tables whose pages lie anywhere in a pool with ``spare`` pages that nobody has, -1 behind a request's last."""
    blocks = [-(-n // page) for n in reaches]
    total = sum(blocks) + spare
    order, at = rng.permutation(total), 0
    table = np.full((len(reaches), max(blocks)), -1, np.int32)
    for i, count in enumerate(blocks):
        table[i, :count] = order[at:at + count]
        at += count
    return table, total


class Pool:
    """Pages on the device and their twins on the host; every slot that nobody stored holds no number."""

    def __init__(self, pages, kv_heads, page, dim, vdim):
        self.codes, self.scales, self.device_codes, self.device_scales = {}, {}, {}, {}
        for name, size in (("k", dim), ("v", vdim)):
            self.codes[name] = np.full((pages, kv_heads, page, size), 127, np.uint8)
            self.scales[name] = np.full((pages, kv_heads, page // 16), np.nan, np.float32)
        self.up()

    def up(self):
        for name in ("k", "v"):
            self.device_codes[name] = torch.tensor(self.codes[name], device="cuda").view(torch.float8_e4m3fn)
            self.device_scales[name] = torch.tensor(self.scales[name], device="cuda")

    def down(self):
        for name in ("k", "v"):
            self.codes[name] = plain.codes_of(self.device_codes[name])
            self.scales[name] = self.device_scales[name].cpu().numpy()

    @property
    def operands(self):
        return self.device_codes["k"], self.device_codes["v"], self.device_scales["k"], self.device_scales["v"]


def rows_of(rng, n, columns, dtype):
    rows = rng.normal(0, 1, (n, columns)) * 2.0 ** rng.normal(0, 2, (1, columns)) * 2.0 ** rng.normal(0, 1, (n, 1))
    return torch.tensor(rows, dtype=torch.float32, device="cuda").to(dtype)


def steps_arrays(entries):
    positions = [start + i for _, count, start in entries for i in range(count)]
    items = [i for i, (_, count, _) in enumerate(entries) for _ in range(count)]
    return positions, items


def laid_out(counts_and_starts):
    """(offset, count, start) of entries whose rows stand behind one another."""
    entries, offset = [], 0
    for count, start in counts_and_starts:
        entries.append((offset, count, start))
        offset += count
    return entries


def compare_append(pool, before, name, rows, rot, positions, items, table, inv_freq, amplitude):
    codes, scales = before.codes[name].copy(), before.scales[name].copy()
    wanted = plain.append(codes, scales, rows, rot, positions, items, table, inv_freq, amplitude)
    np.testing.assert_array_equal(pool.scales[name], scales)
    new = np.zeros(codes.shape[:3], bool)
    page = codes.shape[2]
    for t, want in enumerate(wanted):
        if want is None:
            continue
        where, slot = table[items[t], positions[t] // page], positions[t] % page
        new[where, :, slot] = True
        for head, value in enumerate(want):
            scale = float(scales[where, head, slot // 16])
            got = plain.VALUES[pool.codes[name][where, head, slot]]
            exact = value / scale
            np.testing.assert_array_equal(np.isnan(got), np.isnan(exact))
            off = np.abs(got - np.clip(exact, -448.0, 448.0))
            assert (off[~np.isnan(got)] <= (np.maximum(np.abs(exact) * 2.0 ** -4, 2.0 ** -10) + 448 * 2.0 ** -21 * (rot > 0))[~np.isnan(got)]).all()
            if rot == 0:
                np.testing.assert_array_equal(pool.codes[name][where, head, slot], codes[where, head, slot])
    # the codes that were there already (raised or not), and all others
    np.testing.assert_array_equal(pool.codes[name][~new], codes[~new])
    return new


STORES = [
    # heads, kv_heads, dim, vdim, rot, page, requests' (tokens a step, step by step)
    (4, 2, 64, 64, 64, 16, [[1], [1], [1]]),
    (3, 3, 64, 64, 0, 64, [[37, 5], [1, 20], [9, 1], [3, 3]]),
    (8, 2, 128, 128, 128, 32, [[100, 1, 16], [1, 1, 1], [33, 15, 2]]),
    (2, 1, 96, 32, 48, 48, [[17, 130], [50, 1], [1, 1]]),
    (6, 2, 16, 256, 10, 16, [[15, 1, 14], [2, 16, 1], [1, 1, 1]]),
    (1, 1, 256, 16, 256, 128, [[300], [21], [1]]),
    (5, 5, 32, 48, 32, 112, [[1] * 20, [1] * 20, [7] * 20]),
    (12, 12, 64, 64, 64, 64, [[700, 1, 350], [300, 60, 1]]),
    (2, 1, 32, 16, 24, 48, [[70 + i for i in range(50)], [1] * 50]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, dim, vdim, rot, page, steps", STORES)
def test_store(heads, kv_heads, dim, vdim, rot, page, steps, dtype):
    from mini_llm_b200.kernels import ops
    rng = np.random.default_rng(heads * 1000 + dim + page)
    starts = [int(rng.integers(0, 40)) for _ in steps[0]]
    table, pages = scattered_table([start + sum(step[i] for step in steps) for i, start in enumerate(starts)], page, rng)
    pool = Pool(pages, kv_heads, page, dim, vdim)
    # what stands before a request's first token here: rows of an earlier step
    steps = [[start or 1 for start in starts]] + steps
    starts = [0] * len(starts)
    inv_freq = 10000.0 ** (-np.arange(max(rot // 2, 1)) / max(rot // 2, 1))
    amplitude = 1.0 if rot == 0 else 1.2079441541679836
    for step in steps:
        step = [min(count, table.shape[1] * page - start) for count, start in zip(step, starts)]
        entries = laid_out(zip(step, starts))
        positions, items = steps_arrays(entries)
        n, columns = len(positions), heads * dim + kv_heads * (dim + vdim)
        # (rows of a wider matrix, from a column of its own on)
        wide = torch.full((n, columns + 24), float("nan"), dtype=dtype, device="cuda")
        qkv = wide[:, 8:8 + columns]
        qkv.copy_(rows_of(rng, n, columns, dtype))
        before = Pool.__new__(Pool)
        before.codes, before.scales = {k: v.copy() for k, v in pool.codes.items()}, {k: v.copy() for k, v in pool.scales.items()}
        q_out = torch.full((n, heads * dim + 8), 7.0, dtype=dtype, device="cuda")
        ops.e4m3_store(q_out[:, :heads * dim], qkv, heads * dim, (heads + kv_heads) * dim, heads, kv_heads, dim, vdim, rot,
                       torch.tensor(inv_freq, dtype=torch.float64, device="cuda"), amplitude, ints(positions), ints(items), ints(table), *pool.operands)
        pool.down()
        host = qkv.float().cpu().numpy()
        k = host[:, heads * dim:(heads + kv_heads) * dim].reshape(n, kv_heads, dim)
        v = host[:, (heads + kv_heads) * dim:].reshape(n, kv_heads, vdim)
        compare_append(pool, before, "k", k, rot, positions, items, table, inv_freq, amplitude)
        compare_append(pool, before, "v", v, 0, positions, items, table, inv_freq, 1.0)
        q = host[:, :heads * dim].reshape(n, heads, dim)
        want = np.stack([[plain.turned(q[t, h], rot, positions[t], inv_freq, amplitude) for h in range(heads)] for t in range(n)]).reshape(n, -1)
        got = q_out.float().cpu().numpy()
        bound = np.abs(want) * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24) + 2.0 ** -21 * np.repeat(
            np.abs(q).max(axis=2), dim, axis=1) * 2 * amplitude
        assert (np.abs(got[:, :heads * dim] - want) <= bound).all()
        assert (got[:, heads * dim:] == 7.0).all()
        # the same step again leaves the same bytes
        ops.e4m3_store(None, qkv, heads * dim, (heads + kv_heads) * dim, heads, kv_heads, dim, vdim, rot,
                       torch.tensor(inv_freq, dtype=torch.float64, device="cuda"), amplitude, ints(positions), ints(items), ints(table), *pool.operands)
        for name in ("k", "v"):
            np.testing.assert_array_equal(plain.codes_of(pool.device_codes[name]), pool.codes[name])
            np.testing.assert_array_equal(pool.device_scales[name].cpu().numpy(), pool.scales[name])
        starts = [start + count for start, count in zip(starts, step)]


def store_one(rows, dtype=torch.bfloat16, position=0, pool=None, table=((0,),), rot=0):
    """Rows [T, size] of one head as keys and as values of one request."""
    from mini_llm_b200.kernels import ops
    rows = torch.as_tensor(rows, dtype=torch.float32, device="cuda").to(dtype)
    n, size = rows.shape
    pool = pool or Pool(2, 1, 32, size, size)
    qkv = torch.cat((rows, rows, rows), dim=1)
    q = torch.empty((n, size), dtype=dtype, device="cuda")
    ops.e4m3_store(q, qkv, size, 2 * size, 1, 1, size, size, rot, torch.full((max(rot // 2, 1),), 0.01, dtype=torch.float64, device="cuda"), 1.0,
                   ints(np.arange(position, position + n)), ints([0] * n), ints(table), *pool.operands)
    pool.down()
    return pool, rows.float().cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store_of_sizes_at_the_borders(dtype):
    size = 16
    for value, scale in ((0.0, 2.0 ** -64), (448.0, 1.0), (450.0, 2.0), (449.0, 2.0 if dtype == torch.float32 else 1.0), (1.75, 2.0 ** -8),
                         (2.0 ** -30, 2.0 ** -38), (1e-30, 2.0 ** -64), (2.0 ** 63, 2.0 ** 55), (2.0 ** 63.9, 2.0 ** 56)):
        row = np.zeros((1, size))
        row[0, 3] = -value
        pool, rows = store_one(row, dtype)
        assert pool.scales["k"][0, 0, 0] == pool.scales["v"][0, 0, 0] == np.float32(scale), value
        np.testing.assert_array_equal(pool.codes["k"][0, 0, 0], plain.nearest_code(rows[0].astype(np.float64) / scale))


@pytest.mark.parametrize("bad", [float("nan"), -float("nan"), float("inf"), -float("inf"), 2.0 ** 64, 1e30])
@pytest.mark.parametrize("rot", [0, 16])
def test_rows_that_are_not_finite_are_no_numbers_and_move_no_scale(bad, rot):
    rows = np.random.default_rng(5).normal(0, 1, (6, 16))
    clean = rows.copy()
    rows[2, 7], rows[5, 0] = bad, bad
    clean[2], clean[5] = 0.0, 0.0
    pool, _ = store_one(rows, rot=rot)
    other, _ = store_one(clean, rot=rot)
    for name in ("k", "v"):
        assert pool.scales[name][0, 0, 0] == other.scales[name][0, 0, 0]
        for slot in range(6):
            if slot in (2, 5):
                assert (pool.codes[name][0, 0, slot] & 127 == 127).all()
            else:
                np.testing.assert_array_equal(pool.codes[name][0, 0, slot], other.codes[name][0, 0, slot])


def test_a_raised_scale_rounds_what_is_there_and_a_new_block_begins_anew():
    rng = np.random.default_rng(3)
    pool, first = store_one(rng.normal(0, 1, (5, 64)))
    before = pool.codes["k"].copy()
    held = float(pool.scales["k"][0, 0, 0])
    pool, _ = store_one(rng.normal(0, 300, (2, 64)), position=5, pool=pool)
    scale = float(pool.scales["k"][0, 0, 0])
    assert scale > held
    np.testing.assert_array_equal(pool.codes["k"][0, 0, :5], plain.nearest_code(plain.VALUES[before[0, 0, :5]] * held / scale))
    # a small row does not lower it
    pool, _ = store_one(rng.normal(0, 1e-3, (1, 64)), position=7, pool=pool)
    assert float(pool.scales["k"][0, 0, 0]) == scale
    # the page again, for another request: from its first position on
    pool, rows = store_one(rng.normal(0, 1e-3, (3, 64)), position=0, pool=pool)
    fresh, _ = store_one(rows)
    assert pool.scales["k"][0, 0, 0] == fresh.scales["k"][0, 0, 0] < scale
    np.testing.assert_array_equal(pool.codes["k"][0, 0, :3], fresh.codes["k"][0, 0, :3])


def test_rows_without_a_place_are_stored_nowhere():
    from mini_llm_b200.kernels import ops
    rng = np.random.default_rng(4)
    pool = Pool(3, 2, 16, 32, 32)
    clean = [pool.codes["k"].copy(), pool.codes["v"].copy()]
    qkv = rows_of(rng, 5, 2 * 32 + 4 * 32, torch.bfloat16)
    table = ints([[-1, 7], [0, 3], [2, -1]])
    # a page that is none, one outside the pool, a negative position, a column outside the table, a page outside the pool
    ops.e4m3_store(None, qkv, 64, 128, 2, 2, 32, 32, 0, None, 1.0, ints([3, 20, -1, 32, 16]), ints([0, 0, 1, 1, 1]), table, *pool.operands)
    pool.down()
    np.testing.assert_array_equal(pool.codes["k"], clean[0])
    np.testing.assert_array_equal(pool.codes["v"], clean[1])
    assert np.isnan(pool.scales["k"]).all() and np.isnan(pool.scales["v"]).all()
    # queries alone
    q = torch.empty((5, 64), dtype=torch.bfloat16, device="cuda")
    ops.e4m3_store(q, qkv, 64, 128, 2, 2, 32, 32, 0, None, 1.0, ints([3, 20, -1, 32, 16]), ints([0, 0, 1, 1, 1]), None, None, None, None, None,
                   writes=False)
    np.testing.assert_array_equal(q.float().cpu().numpy(), qkv[:, :64].float().cpu().numpy())


def test_rows_that_fill_a_step_up_leave_the_others_alone():
    """Rows of one more request, all at position 0, as a step filled up to a round number of rows has them: what the other requests store is the same."""
    from mini_llm_b200.kernels import ops
    rng = np.random.default_rng(16)
    heads, dim, real, filler = 2, 64, 37, 27
    qkv = rows_of(rng, real + filler, 3 * heads * dim, torch.bfloat16)
    table = ints([[3, 1], [0, -1], [4, 4]])                                        # page 4: of no request
    items, positions = [0] * 30 + [1] * 7 + [2] * filler, list(range(11, 41)) + list(range(7)) + [0] * filler
    pages = []
    for n in (real, real + filler):
        pool = Pool(5, heads, 32, dim, dim)
        for tensor in pool.operands[2:]:
            tensor.fill_(2.0 ** -64)
        ops.e4m3_store(None, qkv[:n], heads * dim, 2 * heads * dim, heads, heads, dim, dim, 0, None, 1.0, ints(positions[:n]), ints(items[:n]),
                       table, *pool.operands)
        pages.append([tensor[:4].contiguous().view(torch.uint8) for tensor in pool.operands])
    for alone, beside in zip(*pages):
        assert torch.equal(alone, beside)


# ---- attention -----------------------------------------------------------------------------------

def filled_pool(rng, reaches, kv_heads, page, dim, vdim, spare=2):
    """Every position of every request stored, as an earlier step's rows; all else holds no number."""
    table, pages = scattered_table(reaches, page, rng, spare)
    pool = Pool(pages, kv_heads, page, dim, vdim)
    for item, reach in enumerate(reaches):
        for position in range(0, reach, 16):
            where, block = table[item, position // page], position % page // 16
            many = min(16, reach - position)
            for name, size in (("k", dim), ("v", vdim)):
                scale = 2.0 ** rng.integers(-12, -4, kv_heads)
                pool.scales[name][where, :, block] = scale
                rows = rng.normal(0, 1, (kv_heads, many, size)) / scale[:, None, None] * 2.0 ** rng.normal(0, 1, (kv_heads, 1, 1))
                pool.codes[name][where, :, block * 16:block * 16 + many] = plain.nearest_code(rows)
    pool.up()
    return pool, table


def attend(pool, table, entries, q, heads, vdim, scale, dtype=torch.bfloat16, out=None, workspace=None, **how):
    from mini_llm_b200.kernels import ops
    out = torch.full((q.shape[0], heads * vdim), 3.0, dtype=dtype, device="cuda") if out is None else out
    kv_heads = pool.codes["k"].shape[1]
    offsets, counts, starts = (ints([entry[i] for entry in entries]) for i in range(3))
    ops.e4m3_attention(out, q, *pool.operands, ints(table), offsets, counts, starts, heads, kv_heads, scale,
                       workspace=workspace or ops.e4m3_workspace("cuda", vdim), **how)
    return out


def check_attention(got, q, pool, table, entries, heads, scale, dtype, cap=0.0, window=0):
    want, spread, most, edge = plain.attention(q.float().cpu().numpy(), pool.codes["k"], pool.codes["v"], pool.scales["k"], pool.scales["v"], table,
                                         entries, heads, scale, cap, window)
    got = got.float().cpu().numpy().astype(np.float64)
    rows = np.zeros(got.shape[0], bool)
    for offset, count, _ in entries:
        rows[offset:offset + count] = True
    assert (got[~rows] == 3.0).all()
    got, want, spread, edge = got[rows], want[rows], spread[rows], edge[rows]
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    if dtype == torch.bfloat16:
        bound = np.abs(want) * 2.0 ** -8 + spread * (2.0 ** -11 + 2.0 ** -20 * (1 + most)) + edge * 2.0 ** -32
    else:
        n = max(start + count for _, count, start in entries)
        bound = np.abs(want) * 2.0 ** -24 + spread * 2.0 ** -24 * (n + 64 + 8 * (1 + most)) + edge * 2.0 ** -126
    off = np.abs(got - want)
    assert (off[~np.isnan(off)] <= bound[~np.isnan(off)]).all(), np.nanmax(off / np.maximum(bound, 1e-30))


SIZES = [
    # heads, kv_heads, dim, vdim, page
    (12, 12, 64, 64, 64), (4, 1, 128, 128, 16), (8, 2, 64, 128, 32), (6, 2, 96, 48, 48), (16, 1, 32, 16, 128), (20, 1, 128, 64, 16),
    (3, 3, 16, 112, 16), (34, 2, 80, 80, 64),
]
SINGLES = [[1], [16], [17, 33, 1], [300, 15, 16, 1000], [5, 128, 129, 2, 700, 63, 64, 65, 4000]]


@pytest.mark.parametrize("cap, window", [(0.0, 0), (20.0, 0), (0.0, 100), (5.0, 1), (0.0, 17)])
@pytest.mark.parametrize("lengths", SINGLES)
@pytest.mark.parametrize("heads, kv_heads, dim, vdim, page", SIZES)
def test_attention_of_single_tokens(heads, kv_heads, dim, vdim, page, lengths, cap, window):
    rng = np.random.default_rng(heads + dim + len(lengths))
    pool, table = filled_pool(rng, lengths, kv_heads, page, dim, vdim)
    entries = [(i, 1, length - 1) for i, length in enumerate(lengths)]
    q = rows_of(rng, len(lengths), heads * dim, torch.bfloat16)
    scale = 0.5 * dim ** -0.5
    got = attend(pool, table, entries, q, heads, vdim, scale, cap=cap, window=window, longest=1)
    check_attention(got, q, pool, table, entries, heads, scale, torch.bfloat16, cap, window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, dim, vdim, page", [(4, 2, 64, 64, 16), (3, 1, 256, 160, 32), (2, 2, 48, 256, 64)])
def test_plain_attention(heads, kv_heads, dim, vdim, page, dtype):
    rng = np.random.default_rng(dim)
    shapes = [(1, 0), (1, 40), (30, 100), (0, 5), (150, 0)]
    pool, table = filled_pool(rng, [max(1, count + start) for count, start in shapes], kv_heads, page, dim, vdim)
    entries = laid_out(shapes)
    q = rows_of(rng, entries[-1][0] + entries[-1][1] + 3, heads * dim, dtype)
    scale = 0.5 * dim ** -0.5
    for cap, window in ((0.0, 0), (10.0, 33)):
        got = attend(pool, table, entries, q, heads, vdim, scale, dtype, cap=cap, window=window, plain=True)
        check_attention(got, q, pool, table, entries, heads, scale, dtype, cap, window)


PORTIONS = [
    [(2, 0)], [(100, 0)], [(128, 0)], [(129, 3)], [(300, 57)], [(256, 1000), (5, 127)], [(1, 40), (17, 128), (0, 9), (1, 0), (260, 0), (2, 511)],
    [(600, 0), (1, 255), (257, 255)], [(33, 2000)],
]


@pytest.mark.parametrize("cap, window", [(0.0, 0), (20.0, 0), (0.0, 100), (5.0, 1), (0.0, 300)])
@pytest.mark.parametrize("shapes", PORTIONS)
@pytest.mark.parametrize("heads, kv_heads, dim, vdim, page", [(2, 2, 64, 64, 64), (4, 1, 128, 128, 16), (2, 1, 96, 48, 48), (3, 3, 16, 112, 128), (2, 1, 32, 16, 16)])
def test_attention_of_portions(heads, kv_heads, dim, vdim, page, shapes, cap, window):
    from mini_llm_b200.kernels import ops
    rng = np.random.default_rng(heads + dim + len(shapes))
    pool, table = filled_pool(rng, [max(1, count + start) for count, start in shapes], kv_heads, page, dim, vdim)
    entries = laid_out(shapes)
    q = rows_of(rng, entries[-1][0] + entries[-1][1] + 3, heads * dim, torch.bfloat16)
    scale = 0.5 * dim ** -0.5
    workspace = ops.e4m3_workspace("cuda", vdim)
    got = attend(pool, table, entries, q, heads, vdim, scale, cap=cap, window=window, workspace=workspace)
    check_attention(got, q, pool, table, entries, heads, scale, torch.bfloat16, cap, window)
    assert int(workspace.status) == 0 and int(workspace.counters.abs().sum()) == 0


# ---- what is no number, what lies elsewhere, and what the calls share ------------------------------

def test_values_that_are_no_numbers_reach_only_the_rows_that_see_them():
    """Position 70 of one request holds a key, position 150 a value that is none: queries before see numbers, queries from there on none, the
    other request nothing of it; within a window only those that still see them."""
    rng = np.random.default_rng(9)
    heads, dim = 4, 64
    for window in (0, 40):
        pool, table = filled_pool(rng, [300, 300], 2, 32, dim, dim)
        for name, position in (("k", 70), ("v", 150)):
            pool.codes[name][table[0, position // 32], :, position % 32] = 127
        pool.up()
        for shapes in ([(200, 60), (100, 130)], [(1, 69), (1, 200)], [(1, 70), (1, 200)], [(1, 100), (1, 1)], [(1, 149), (1, 1)], [(1, 250), (30, 100)]):
            entries = laid_out(shapes)
            q = rows_of(rng, entries[-1][0] + entries[-1][1], heads * dim, torch.bfloat16)
            got = attend(pool, table, entries, q, heads, dim, 0.05, window=window)
            check_attention(got, q, pool, table, entries, heads, 0.05, torch.bfloat16, 0.0, window)
            check_attention(attend(pool, table, entries, q, heads, dim, 0.05, window=window, plain=True), q, pool, table, entries, heads, 0.05,
                            torch.bfloat16, 0.0, window)


def test_queries_that_are_not_finite_stay_in_their_rows():
    rng = np.random.default_rng(10)
    pool, table = filled_pool(rng, [200], 1, 64, 64, 64)
    q = rows_of(rng, 150, 2 * 64, torch.bfloat16)
    bad = q.clone()
    for row, value in ((3, float("nan")), (17, float("inf")), (140, -float("inf"))):
        bad[row, 5] = value
    for entries in ([(0, 150, 50)], [(3, 1, 100)], [(17, 1, 100)]):
        clean, got = (attend(pool, table, entries, x, 2, 64, 0.1).float().cpu().numpy() for x in (q, bad))
        rows = np.ones(150, bool)
        rows[[3, 17, 140]] = False
        np.testing.assert_array_equal(got[rows], clean[rows])
        np.testing.assert_array_equal(got[:, 64:], clean[:, 64:])                 # (the other head)
        offset, count, _ = entries[0]
        assert np.isnan(got[[r for r in (3, 17, 140) if offset <= r < offset + count], :64]).all()


def test_entries_without_tokens_or_keys_and_pages_that_are_none():
    rng = np.random.default_rng(11)
    pool, table = filled_pool(rng, [100, 100, 100, 100], 2, 16, 64, 64)
    table[2, 1], table[3, 0] = -1, pool.codes["k"].shape[0] + 5                   # pages that the table does not name
    # no tokens; a position before the first; keys missing in the middle and at the start
    entries = [(0, 0, 50), (0, 1, -1), (1, 30, 40), (31, 1, 99), (32, 3, -2)]
    table = np.concatenate((table, table[:1]))
    q = rows_of(rng, 36, 4 * 64, torch.bfloat16)
    for plain_kernel in (False, True):
        got = attend(pool, table, entries, q, 4, 64, 0.1, plain=plain_kernel)
        check_attention(got, q, pool, table, entries, 4, 0.1, torch.bfloat16)
        assert (got[0] == 0).all() and (got[32:34] == 0).all() and not (got[34] == 0).all() and (got[35] == 3.0).all()
    # an entry that reaches past its row of the table sees what the table names
    entries = [(0, 1, 5000), (1, 40, 100), (41, 0, 0), (41, 0, 0), (41, 0, 0)]
    q = rows_of(rng, 41, 4 * 64, torch.bfloat16)
    check_attention(attend(pool, table, entries, q, 4, 64, 0.1), q, pool, table, entries, 4, 0.1, torch.bfloat16)


def test_scales_far_apart_and_scores_far_apart():
    """Blocks whose scales differ by 2^100, and queries that make scores of thousands: one block's values outweigh all others by far."""
    rng = np.random.default_rng(12)
    pool, table = filled_pool(rng, [400], 1, 16, 64, 64)
    for block in range(25):
        where = table[0, block]
        pool.scales["v"][where, 0, 0] = 2.0 ** int(rng.integers(-64, 40))
        pool.scales["k"][where, 0, 0] = 2.0 ** int(rng.integers(-12, -4))
    pool.up()
    q = rows_of(rng, 200, 3 * 64, torch.bfloat16)
    for scale in (0.01, 3.0):
        for entries in ([(0, 200, 200)], [(7, 1, 399)]):
            got = attend(pool, table, entries, q, 3, 64, scale)
            check_attention(got, q, pool, table, entries, 3, scale, torch.bfloat16)


@pytest.mark.parametrize("cap", [2.0 ** -100, 1e-3, 2.0, 10.0, 60.0, 8192.0])
def test_caps_at_their_borders(cap):
    """The least cap leaves all keys alike.  With the largest the hardware's approximations show: in cap * (1 - 2 r), r = 1 / (1 + e), the
    exponential's error of 2^-22 moves 2 r by 2^-23 (r' = -r^2, e = 1), the reciprocal's unit in the last place by 2^-23, the sum's rounding by
    2^-24: 1.25 * 2^-22 of the cap together.  (Scores up to a quarter of the cap, with a cap of 10 some, of 60 all, have less: the series that
    portions take for them ends 2^-23.5 of the cap early.)"""
    rng = np.random.default_rng(15)
    shapes = [(140, 60), (1, 150), (1, 0)]
    pool, table = filled_pool(rng, [count + start for count, start in shapes], 2, 32, 64, 48)
    entries = laid_out(shapes)
    q = rows_of(rng, entries[-1][0] + 1, 4 * 64, torch.bfloat16)
    want, spread, most, edge = plain.attention(q.float().cpu().numpy(), pool.codes["k"], pool.codes["v"], pool.scales["k"], pool.scales["v"], table,
                                               entries, 4, 0.1, cap)
    # the bound of other caps, and the capped scores' error: a weight is off by as much, their sum too, and so twice that of the sum of |v|
    bound = np.abs(want) * 2.0 ** -8 + spread * (2.0 ** -11 + 2.0 ** -20 * (1 + most) + 2 * 1.25 * 2.0 ** -22 * cap) + edge * 2.0 ** -32
    for plain_kernel in (False, True):
        got = attend(pool, table, entries, q, 4, 48, 0.1, cap=cap, plain=plain_kernel).float().cpu().numpy()
        assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("cap, window", [(0.0, 0), (7.0, 0), (0.0, 20)])
@pytest.mark.parametrize("power, scale", [(0, 0.0), (-100, 0.25), (-126, 2.0 ** -126), (-30, 2.0 ** -120)])
def test_scores_that_vanish(power, scale, cap, window):
    """No scale, and queries or a scale so small that a product of factors is below every 32-bit number: all visible keys weigh the same, and
    what is hidden stays hidden."""
    rng = np.random.default_rng(14)
    shapes = [(150, 70), (1, 99), (3, 0), (1, 0), (1, 300)]
    pool, table = filled_pool(rng, [count + start for count, start in shapes], 2, 32, 64, 48)
    entries = laid_out(shapes)
    q = (rows_of(rng, entries[-1][0] + 1, 4 * 64, torch.bfloat16).float() * 2.0 ** power).to(torch.bfloat16)
    for plain_kernel in (False, True):
        got = attend(pool, table, entries, q, 4, 48, scale, cap=cap, window=window, plain=plain_kernel)
        check_attention(got, q, pool, table, entries, 4, scale, torch.bfloat16, cap, window)


def test_results_do_not_depend_on_the_call_and_the_workspace_is_left_as_it_was():
    """Twice the same bits, whatever the workspace held; rows of wider matrices; parts of units among many CTAs (long requests, few heads)."""
    from mini_llm_b200.kernels import ops
    rng = np.random.default_rng(13)
    shapes = [(300, 3000), (1, 6000), (2, 0), (1, 17)]
    pool, table = filled_pool(rng, [count + start for count, start in shapes], 1, 64, 128, 64)
    entries = laid_out(shapes)
    wide_q = rows_of(rng, 304, 2 * 128 + 16, torch.bfloat16)
    q = wide_q[:, 8:8 + 256]
    workspace = ops.e4m3_workspace("cuda", 128)
    results = []
    for fill in (0.0, float("nan")):
        workspace.partial.fill_(fill)
        wide_out = torch.full((304, 2 * 64 + 24), 5.0, dtype=torch.bfloat16, device="cuda")
        attend(pool, table, entries, q, 2, 64, 0.05, out=wide_out[:, 16:16 + 128], workspace=workspace)
        assert (wide_out[:, :16] == 5.0).all() and (wide_out[:, 144:] == 5.0).all()
        results.append(wide_out[:, 16:144].clone())
        assert int(workspace.status) == 0 and int(workspace.counters.abs().sum()) == 0
    assert torch.equal(*results)
    check_attention(results[0], q, pool, table, entries, 2, 0.05, torch.bfloat16)


def test_another_stream_and_a_replayed_graph():
    from mini_llm_b200.kernels import ops
    rng = np.random.default_rng(14)
    pool, table = filled_pool(rng, [700, 300, 40], 2, 32, 64, 64)
    q = rows_of(rng, 300, 4 * 64, torch.bfloat16)
    qkv = rows_of(rng, 300, 8 * 64, torch.bfloat16)
    tables = ints(table)
    plans = [[(0, 200, 300), (200, 1, 200), (201, 20, 3)], [(0, 1, 650), (1, 250, 10), (251, 40, 0)]]
    offsets, counts, starts = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(3))
    positions, items = (torch.zeros(300, dtype=torch.int32, device="cuda") for _ in range(2))
    out, workspace = torch.zeros((300, 4 * 64), dtype=torch.bfloat16, device="cuda"), ops.e4m3_workspace("cuda", 64)

    def step():
        ops.e4m3_store(None, qkv, 4 * 64, 6 * 64, 4, 2, 64, 64, 0, None, 1.0, positions, items, tables, *pool.operands)
        ops.e4m3_attention(out, q, *pool.operands, tables, offsets, counts, starts, 4, 2, 0.1, workspace=workspace)

    def bring(plan):
        for i, t in enumerate((offsets, counts, starts)):
            t.copy_(ints([entry[i] for entry in plan]))
        at, item = steps_arrays(plan)
        positions.fill_(-1)
        positions[:len(at)], items[:len(at)] = ints(at), ints(item)
        out.fill_(3.0)

    wanted, stores = [], []
    first = [t.clone() for t in pool.operands]
    for plan in plans:
        bring(plan)
        for t, before in zip(pool.operands, first):
            t.copy_(before)
        step()
        wanted.append(out.clone())
        stores.append([t.clone() for t in pool.operands])
        pool.down()
        check_attention(out, q, pool, table, plan, 4, 0.1, torch.bfloat16)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for plan, want, store in list(zip(plans, wanted, stores)) * 2:
        for run in ("graph", "stream"):
            bring(plan)
            for t, before in zip(pool.operands, first):
                t.copy_(before)
            if run == "graph":
                graph.replay()
            else:
                stream.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(stream):
                    step()
                torch.cuda.current_stream().wait_stream(stream)
            torch.cuda.synchronize()
            assert torch.equal(out, want), run
            for t, kept in zip(pool.operands, store):
                assert torch.equal(t.view(torch.uint8), kept.view(torch.uint8))


def test_offsets_past_four_gigabytes():
    """Pages whose codes lie more than 2^32 bytes into the pool."""
    from mini_llm_b200.kernels import ops
    page, heads, dim = 128, 4, 128
    pages = (5 << 30) // (heads * page * dim)
    code = torch.float8_e4m3fn
    k_pages, v_pages = (torch.zeros((pages, heads, page, dim), dtype=torch.uint8, device="cuda").view(code) for _ in range(2))
    k_scales, v_scales = (torch.ones((pages, heads, page // 16), device="cuda") for _ in range(2))
    rng = np.random.default_rng(15)
    small = Pool(4, heads, page, dim, dim)
    table = np.array([[3, 1, 2]], np.int32)
    n = 300
    qkv = rows_of(rng, n, 3 * heads * dim, torch.bfloat16)
    inv_freq = torch.tensor(10000.0 ** (-np.arange(64) / 64), dtype=torch.float64, device="cuda")
    results = []
    for names, operands in ((table, small.operands), (table + pages - 4, (k_pages, v_pages, k_scales, v_scales))):
        q = torch.empty((n, heads * dim), dtype=torch.bfloat16, device="cuda")
        ops.e4m3_store(q, qkv, heads * dim, 2 * heads * dim, heads, heads, dim, dim, 128, inv_freq, 1.0, ints(np.arange(n)), ints([0] * n), ints(names), *operands)
        for entry in ((0, n, 0), (0, 1, n - 1)):
            out = torch.zeros((n, heads * dim), dtype=torch.bfloat16, device="cuda")
            ops.e4m3_attention(out, q, *operands, ints(names), ints([entry[0]]), ints([entry[1]]), ints([entry[2]]), heads, heads, 0.01,
                               workspace=ops.e4m3_workspace("cuda", dim))
            results.append(out)
    assert torch.equal(results[0], results[2]) and torch.equal(results[1], results[3]) and bool(results[0].abs().sum() > 0)


def test_refusals():
    from mini_llm_b200.kernels import ops
    from mini_llm_b200.kernels.lib import KernelError
    pool = Pool(3, 2, 32, 64, 64)
    kp, vp, ks, vs = pool.operands
    q, out = (torch.zeros((4, 4 * 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table, one, workspace = ints([[0, 1]]), ints([1]), ops.e4m3_workspace("cuda", 64)
    good = dict(out=out, q=q, k_pages=kp, v_pages=vp, k_scales=ks, v_scales=vs, block_table=table, item_offset=ints([0]), item_count=one,
                item_start=ints([0]), heads=4, kv_heads=2, scale=0.1, workspace=workspace)
    ops.e4m3_attention(**good)
    wide = torch.zeros((4, 4 * 64 + 4), dtype=torch.bfloat16, device="cuda")
    for change, text in ((dict(q=q.cpu()), "CUDA tensor"), (dict(q=q.half()), "element type"), (dict(out=out.float()), "bfloat16"), (dict(out=out[:3]), "columns"),
                         (dict(k_pages=kp.view(torch.uint8)), "float8"), (dict(k_pages=kp[:2]), "same pages"), (dict(v_pages=vp[:, :, :, ::2]), "contiguous"),
                         (dict(k_scales=ks[:, :1]), "scales"), (dict(k_scales=ks.half()), "float32"), (dict(block_table=table.long()), "int32"),
                         (dict(item_count=ints([1, 1])), "item_count"), (dict(item_start=ints([0]).long()), "int32"), (dict(heads=5), "heads over"),
                         (dict(kv_heads=4), "heads over"), (dict(window=-1), "window"), (dict(cap=-1.0), "cap"), (dict(scale=-0.1), "scale"),
                         (dict(cap=float("inf")), "cap"), (dict(cap=1e-40), "cap"), (dict(cap=float("nan")), "cap"), (dict(cap=8193.0), "cap"),
                         (dict(scale=float("inf")), "scale"), (dict(scale=1e39), "scale"), (dict(window=2 ** 31), "window"), (dict(item_count=[1]), "item_count"),
                         (dict(q=q[0]), "dimensions"), (dict(v_pages=vp[0]), "v_pages"),
                         (dict(scale=float("nan")), "scale"), (dict(workspace=None), "workspace"), (dict(q=wide[:, :256]), "16-byte"),
                         (dict(out=wide[:, 2:258]), "16-byte")):
        with pytest.raises(KernelError, match=text):
            ops.e4m3_attention(**{**good, **change})
    with pytest.raises(KernelError, match="workspace is for"):
        big = Pool(2, 2, 32, 64, 128)
        ops.e4m3_attention(**{**good, **dict(zip(("k_pages", "v_pages", "k_scales", "v_scales"), big.operands)),
                              "out": torch.zeros((4, 4 * 128), dtype=torch.bfloat16, device="cuda")})
    qkv = torch.zeros((4, 8 * 64), dtype=torch.bfloat16, device="cuda")
    good = dict(q_out=out, qkv=qkv, k_off=256, v_off=384, heads=4, kv_heads=2, dim=64, vdim=64, rot_dims=64,
                inv_freq=torch.ones(32, dtype=torch.float64, device="cuda"), amplitude=1.0, positions=ints([0, 1, 2, 3]), token_item=ints([0] * 4),
                block_table=table, k_pages=kp, v_pages=vp, k_scales=ks, v_scales=vs)
    ops.e4m3_store(**good)
    for change, text in ((dict(qkv=qkv.cpu()), "CUDA tensor"), (dict(qkv=qkv.half()), "element type"), (dict(dim=60), "multiples of 16"), (dict(vdim=512), "multiples of 16"),
                         (dict(amplitude=1e39), "amplitude"), (dict(amplitude=float("nan")), "amplitude"), (dict(positions=[0, 1, 2, 3]), "positions"),
                         (dict(rot_dims=63), "turned"), (dict(rot_dims=80), "turned"), (dict(v_off=400), "columns"), (dict(k_off=252), "multiples of 8"),
                         (dict(inv_freq=torch.ones(31, dtype=torch.float64, device="cuda")), "frequencies"), (dict(inv_freq=None), "expected a CUDA"),
                         (dict(inv_freq=torch.ones(32, device="cuda")), "float64"), (dict(positions=ints([0, 1])), "fewer positions"),
                         (dict(token_item=ints([0] * 4).long()), "int32"), (dict(q_out=out[:, :128]), "columns"), (dict(q_out=out.float()), "bfloat16"),
                         (dict(kv_heads=1), "another number"), (dict(k_pages=kp.view(torch.uint8)), "float8"), (dict(block_table=table[0]), "dimensions"),
                         (dict(q_out=wide[:, 2:258]), "16-byte")):
        with pytest.raises(KernelError, match=text):
            ops.e4m3_store(**{**good, **change})
    # nothing to do is no error
    ops.e4m3_store(**{**good, "qkv": qkv[:0], "q_out": out[:0], "positions": ints([]), "token_item": ints([])})
    none = torch.zeros((0, 2), dtype=torch.int32, device="cuda")
    ops.e4m3_attention(out[:0], q[:0], kp, vp, ks, vs, none, ints([]), ints([]), ints([]), 4, 2, 0.1, workspace=workspace)


# ---- units that stand behind one another in a CTA --------------------------------------------------

@pytest.mark.parametrize("heads, kv_heads, dim, page", [(12, 4, 64, 64), (12, 4, 128, 32)])
@pytest.mark.parametrize("shapes", [
    [(100, 90)] + [(700, 0)] * 16,                                        # few blocks of one tile, then units of two
    [(256 * 5 + 100, 300)] * 6,                                           # the remainder of every portion comes ahead of its full units
    [(count, 100 * i) for i in range(16) for count in (40, 500)],         # a short portion ahead of every long one
])
def test_units_of_one_tile_ahead_of_units_of_two(heads, kv_heads, dim, page, shapes):
    """The scales differ from block to block, so that a tile that meets another block's would show; against the kernel of every size.  Both results are
    rounded to bfloat16, 2^-8 each.  Of the sum of the weights times |v|, `top` at most, are off: the weights of 16 bits by 2^-11, sums of N terms
    in 32 bits by N 2^-24, and by scores as in ``check_attention``, of both kernels."""
    rng = np.random.default_rng(dim + len(shapes))
    pool, table = filled_pool(rng, [count + start for count, start in shapes], kv_heads, page, dim, dim)
    entries, scale, longest = laid_out(shapes), 0.1 * dim ** -0.5, max(count + start for count, start in shapes)
    q = torch.tensor(rng.normal(0, 1, (entries[-1][0] + entries[-1][1], heads * dim)), dtype=torch.float32, device="cuda").to(torch.bfloat16)
    k, v = (np.abs(plain.VALUES[pool.codes[name]]) * pool.scales[name].repeat(16, axis=2)[..., None] for name in ("k", "v"))
    top, edge = np.nanmax(v), longest * 448.0 * np.nanmax(pool.scales["v"])
    most = scale * np.sqrt(np.nanmax((k * k).sum(axis=3))) * float(q.float().view(-1, dim).norm(dim=1).max())
    for window in (0, 200):
        want = attend(pool, table, entries, q, heads, dim, scale, window=window, plain=True).float()
        first = attend(pool, table, entries, q, heads, dim, scale, window=window)
        for _ in range(4):
            assert torch.equal(attend(pool, table, entries, q, heads, dim, scale, window=window), first)
        got = first.float()
        bound = 2.0 ** -8 * (want.abs() + got.abs()) + top * (2.0 ** -11 + longest * 2.0 ** -24 + 2 * 2.0 ** -20 * (1 + most)) + edge * 2.0 ** -32
        assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


# ---- the ends of what 32 bits hold -----------------------------------------------------------------

@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("query, held, scale", [
    (126, -64, -60), (127, -64, -62), (126, -64, -62), (127, -64, -70), (111, -64, -47),       # the largest queries: scores of 4, 2, 1, 2^-7 and 1
    (100, -64, 60), (127, -64, 50), (100, 20, -110), (125, 0, -20),                            # products of factors beyond 32 bits
    (-100, 40, 127), (0, 40, 60), (-126, 55, 126), (-126, 55, 72),                             # the smallest queries, the largest scales
])
def test_queries_and_scales_of_all_sizes(query, held, scale, cap):
    """Queries of one entry, +-2^query, over keys that are zero but for one, 1 at a scale of 2^held: that key's score is +-2^(query + held + scale), all
    others' zero."""
    rng = np.random.default_rng(17)
    shapes = [(150, 70), (1, 99), (3, 60), (1, 40)]
    pool, table = filled_pool(rng, [count + start for count, start in shapes], 2, 32, 64, 48)
    stored = ~np.isnan(pool.scales["k"])
    pool.codes["k"][...] = 0
    pool.scales["k"][stored] = 2.0 ** held
    for item in range(len(shapes)):
        pool.codes["k"][table[item, 1], :, 5, 5] = 0x38                           # position 37
    pool.up()
    entries = laid_out(shapes)
    q = torch.zeros((entries[-1][0] + 1, 4, 64), device="cuda")
    q[:, 0::2, 5], q[:, 1::2, 5] = 2.0 ** query, -2.0 ** query
    q = q.flatten(1).to(torch.bfloat16)
    want, spread, most, edge = plain.attention(q.float().cpu().numpy(), pool.codes["k"], pool.codes["v"], pool.scales["k"], pool.scales["v"], table,
                                               entries, 4, 2.0 ** scale, cap)
    # (scores are powers of two or zero, so that but for a cap only the exponential, its argument's rounding and the weights' 16 bits are off)
    bound = np.abs(want) * 2.0 ** -8 + spread * (2.0 ** -11 + 2.0 ** -20 * (1 + (cap or min(most, 16.0)))) + edge * 2.0 ** -32
    for plain_kernel in (True, False):
        got = attend(pool, table, entries, q, 4, 48, 2.0 ** scale, cap=cap, plain=plain_kernel).float().cpu().numpy()
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rot", [0, 8, 32])
@pytest.mark.parametrize("power", [-100, -80, -70, 0, 40, 63, 64, 100, 127])
def test_amplitudes_of_all_sizes(power, rot, dtype):
    """Keys whose turned entries, times an amplitude of 2^power, are of any size and others of size 1; values, which no amplitude touches, are what
    they are without one, and so is a key of zeros."""
    from mini_llm_b200.kernels import ops
    rng = np.random.default_rng(18)
    n, dim = 21, 32
    amplitude = 2.0 ** power
    rows = rng.normal(0, 1, (n, 3 * dim))
    # (turned keys of size 2^-20 to 2^20: the largest amplitudes want small entries, the smallest large ones)
    rows[:, dim:dim + rot] *= 2.0 ** float(np.clip(-power + rng.integers(-20, 20), -120, 110))
    rows[4, dim:2 * dim] = 0.0
    qkv = torch.tensor(rows, dtype=torch.float32, device="cuda").to(dtype)
    inv_freq = 100.0 ** (-np.arange(max(rot // 2, 1)) / 16)
    pool, before = (Pool(2, 1, 32, dim, dim) for _ in range(2))
    table, positions, items = [[1]], np.arange(n), [0] * n
    ops.e4m3_store(None, qkv, dim, 2 * dim, 1, 1, dim, dim, rot, torch.tensor(inv_freq, dtype=torch.float64, device="cuda"), amplitude, ints(positions),
                   ints(items), ints(table), *pool.operands)
    pool.down()
    host = qkv.float().cpu().numpy()
    compare_append(pool, before, "v", host[:, None, 2 * dim:], 0, positions, items, np.array(table), inv_freq, 1.0)
    # the same numbers from entries that are multiplied already: a power of two leaves their digits
    already = host[:, None, dim:2 * dim].astype(np.float64)
    already[..., :rot] *= amplitude
    with np.errstate(over="ignore"):
        squares = already ** 2
    lengths = np.concatenate((squares[..., 0:rot:2] + squares[..., 1:rot:2], squares[..., rot:]), axis=-1).max(axis=-1)[:, 0]
    for block in (slice(0, 16), slice(16, n)):
        scale = float(pool.scales["k"][1, 0, block.start // 16])
        assert scale == plain.least_scale(float(lengths[block].max()))
        for t in range(n)[block]:
            exact = plain.turned(already[t, 0], rot, t, inv_freq) / scale
            got = plain.VALUES[pool.codes["k"][1, 0, t]]
            assert (np.abs(got - np.clip(exact, -448.0, 448.0)) <= np.maximum(np.abs(exact) * 2.0 ** -4, 2.0 ** -10) + 448 * 2.0 ** -21).all()


def test_amplitudes_that_are_refused():
    from mini_llm_b200.kernels import ops
    from mini_llm_b200.kernels.lib import KernelError
    pool, qkv = Pool(2, 1, 32, 32, 32), torch.ones((3, 96), device="cuda")
    for amplitude in (2.0 ** -101, -2.0 ** -140, 2.0 ** 127.5, -1e39, float("inf"), float("nan")):
        with pytest.raises(KernelError, match="amplitude"):
            ops.e4m3_store(None, qkv, 32, 64, 1, 1, 32, 32, 32, torch.ones(16, dtype=torch.float64, device="cuda"), amplitude, ints([0, 1, 2]),
                           ints([0] * 3), ints([[0]]), *pool.operands)
    # none at all leaves zeros, a negative one turns by half a turn more
    for amplitude in (0.0, -1.0):
        ops.e4m3_store(None, qkv, 32, 64, 1, 1, 32, 32, 32, torch.zeros(16, dtype=torch.float64, device="cuda"), amplitude, ints([0, 1, 2]),
                       ints([0] * 3), ints([[0]]), *pool.operands)
        pool.down()
        np.testing.assert_array_equal(plain.VALUES[pool.codes["k"][0, 0, :3]] * pool.scales["k"][0, 0, 0], np.full((3, 32), amplitude))
        np.testing.assert_array_equal(plain.VALUES[pool.codes["v"][0, 0, :3]] * pool.scales["v"][0, 0, 0], np.ones((3, 32)))


# ---- waits that run out ----------------------------------------------------------------------------

@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("away", [31, 33, 34, 35])                            # converters, products, softmax, schedule
def test_a_role_that_stays_away_is_reported_and_the_next_call_is_right(away, dim, cap):
    """Every wait of the portions' kernel is bounded.  Here one of its roles does nothing (a test's switch) and the limit is 2 ms: the others give up and
    the kernel returns with a code of one of them; after ``reset`` the workspace serves as a new one does."""
    from mini_llm_b200.kernels import ops
    rng = np.random.default_rng(19)
    shapes = [(100, 30), (700, 200), (1, 90), (300, 3000)]
    pool, table = filled_pool(rng, [count + start for count, start in shapes], 2, 32, dim, dim)
    entries = laid_out(shapes)
    q = rows_of(rng, entries[-1][0] + entries[-1][1], 4 * dim, torch.bfloat16)
    want = attend(pool, table, entries, q, 4, dim, 0.05, cap=cap)
    workspace = ops.e4m3_workspace("cuda", dim)
    for _ in range(2):
        workspace.wait_limit_ns, workspace.role_away = 2_000_000, away
        attend(pool, table, entries, q, 4, dim, 0.05, cap=cap, workspace=workspace)
        assert int(workspace.status) in {31, 33, 34, 35} - {away}
        workspace.wait_limit_ns = workspace.role_away = 0
        workspace.reset()
        assert int(workspace.status) == 0 and int(workspace.counters.abs().sum()) == 0
        assert torch.equal(attend(pool, table, entries, q, 4, dim, 0.05, cap=cap, workspace=workspace), want)
        assert int(workspace.status) == 0 and int(workspace.counters.abs().sum()) == 0


# ---- positions of all sizes ------------------------------------------------------------------------

@pytest.mark.parametrize("heads, kv_heads, dim, page", [(4, 2, 64, 16), (3, 1, 128, 48)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 1000])
def test_windows_longer_than_any_context(window, heads, kv_heads, dim, page):
    """Also with positions before the first: rows there are zero, the others see what they see without a window."""
    rng = np.random.default_rng(20)
    shapes = [(40, -5), (300, -200), (1, -3), (130, 20), (1, 77), (2, -1), (600, -300)]
    pool, table = filled_pool(rng, [max(1, count + start) for count, start in shapes], kv_heads, page, dim, dim)
    entries = laid_out(shapes)
    q = rows_of(rng, entries[-1][0] + entries[-1][1], heads * dim, torch.bfloat16)
    for plain_kernel in (False, True):
        got = attend(pool, table, entries, q, heads, dim, 0.05, window=window, plain=plain_kernel)
        check_attention(got, q, pool, table, entries, heads, 0.05, torch.bfloat16, 0.0, window)
        assert torch.equal(got, attend(pool, table, entries, q, heads, dim, 0.05, plain=plain_kernel))


@pytest.mark.parametrize("start", [129, 10 ** 6, 2 ** 31 - 40])
def test_walks_end_where_the_block_table_does(start):
    """Queries at positions behind the last that the table has a page for see all that it has, whatever their position, or, within a window that ends
    behind it, nothing."""
    rng = np.random.default_rng(21)
    heads, dim, page, reach = 4, 64, 16, 128
    pool, table = filled_pool(rng, [reach] * 3, 2, page, dim, dim)
    entries = [(0, 40, start), (40, 1, start + 39), (41, 2, start + 5)]
    q = rows_of(rng, 43, heads * dim, torch.bfloat16)
    at_its_end = [(row, 1, reach - 1) for row in range(43)]
    rows = np.array([0] * 40 + [1] + [2] * 2)
    for plain_kernel in (False, True):
        got = attend(pool, table, entries, q, heads, dim, 0.05, plain=plain_kernel)
        check_attention(got, q, pool, table[rows], at_its_end, heads, 0.05, torch.bfloat16)
        assert (attend(pool, table, entries, q, heads, dim, 0.05, window=1, plain=plain_kernel) == 0).all()


def test_first_calls_of_several_threads_at_once():
    """Heads of several sizes that share kernels, each thread on a stream and with a workspace of its own, in a process that has made no such call: what the
    calls set once must suffice for all of them."""
    code = '''
import threading
import torch
from mini_llm_b200.kernels import ops
SIZES = [(16, 16), (80, 16), (128, 112), (96, 96), (16, 64), (64, 64), (128, 128), (48, 48)]
work = []
for i, (dim, vdim) in enumerate(SIZES * 3):
    heads = (1, 12, 16)[i % 3]
    generator = torch.Generator(device="cuda").manual_seed(i)
    k, v = (torch.randint(0, 120, (60, 1, 32, size), generator=generator, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for size in (dim, vdim))
    scales = torch.full((60, 1, 2), 2.0 ** -7, device="cuda")
    q = torch.randn((201, heads * dim), generator=generator, device="cuda").bfloat16()
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [1, 200], [900, 700])]
    table = torch.randperm(60, generator=generator, device="cuda").to(torch.int32).view(2, 30)
    out = torch.zeros((201, heads * vdim), dtype=torch.bfloat16, device="cuda")
    work.append((out, q, k, v, scales, scales, table, *ints, heads, 1, 0.01))
spaces = [ops.e4m3_workspace("cuda", vdim) for _, vdim in SIZES * 3]
torch.cuda.synchronize()
start, errors = threading.Barrier(len(work)), []
def call(args, space):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            ops.e4m3_attention(*args, workspace=space)
            torch.cuda.current_stream().synchronize()
    except Exception as error:
        errors.append(error)
threads = [threading.Thread(target=call, args=pair) for pair in zip(work, spaces)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not errors, errors
for args, space in zip(work, spaces):
    got = args[0].clone()
    ops.e4m3_attention(*args, workspace=space)
    assert torch.equal(args[0], got) and int(space.status) == 0 and bool(got.abs().sum() > 0)
'''
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root)
    assert done.returncode == 0, done.stderr[-2000:]


# ---- what the calls ask of their operands ----------------------------------------------------------

def _changes(value):
    """Other operands in the place of one: other types, shapes, strides, devices, alignments and numbers."""
    if isinstance(value, torch.Tensor):
        yield from (value.cpu(), value[:-1], value[:0], value[None], value.reshape(-1), list(value.shape), None)
        for dtype in (torch.int32, torch.int64, torch.float32, torch.float64, torch.bfloat16, torch.float16, torch.uint8, torch.float8_e4m3fn):
            if dtype != value.dtype:
                yield torch.zeros(value.shape, dtype=torch.float32, device="cuda").to(dtype)
        for d in range(value.dim()):
            shape = list(value.shape)
            shape[d] *= 2
            longer = torch.zeros(shape, dtype=torch.float32, device="cuda").to(value.dtype)
            yield longer
            yield longer[tuple(slice(None, None, 2) if i == d else slice(None) for i in range(value.dim()))]           # every second
            shape[d] = value.shape[d] + 1
            yield torch.zeros(shape, dtype=torch.float32, device="cuda").to(value.dtype)[
                tuple(slice(1, None) if i == d else slice(None) for i in range(value.dim()))]                           # from the second on
    elif isinstance(value, int):
        yield from (0, 1, -1, 2, 3, 16, 17, 48, 256, 272, 10 ** 6, 2 ** 31)
    else:
        yield from (0, 1, -1, 0.5, -0.5, 2.0 ** 127, 2.0 ** -140, 1e39, float("inf"), -float("inf"), float("nan"))


@pytest.mark.parametrize("rows", [0, 1, 4])
def test_what_is_refused_is_refused_by_both_checks(rows, monkeypatch):
    """The calls ask everything in one expression, and again one by one for the error's text.  With one operand changed, a ``KernelError`` is raised, and
    nothing launched, where the second finds fault, and only there; but for a lone row's strides, which do not matter, the first finds it in the same cases."""
    from mini_llm_b200.kernels import ops
    from mini_llm_b200.kernels.lib import KernelError
    pool = Pool(3, 2, 32, 64, 48)
    kp, vp, ks, vs = pool.operands
    table, workspace = ints([[0, 1]]), ops.e4m3_workspace("cuda", 64)
    q, out = torch.zeros((rows, 4 * 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((rows, 4 * 48), dtype=torch.bfloat16, device="cuda")
    attention = dict(out=out, q=q, k_pages=kp, v_pages=vp, k_scales=ks, v_scales=vs, block_table=table, item_offset=ints([0]), item_count=ints([rows]),
                     item_start=ints([0]), heads=4, kv_heads=2, scale=0.1, cap=0.0, window=0)
    qkv = torch.zeros((rows, 4 * 64 + 2 * (64 + 48)), dtype=torch.bfloat16, device="cuda")
    store = dict(q_out=q, qkv=qkv, k_off=256, v_off=384, heads=4, kv_heads=2, dim=64, vdim=48, rot_dims=32,
                 inv_freq=torch.ones(16, dtype=torch.float64, device="cuda"), amplitude=1.0, positions=ints(range(rows)), token_item=ints([0] * rows),
                 block_table=table, k_pages=kp, v_pages=vp, k_scales=ks, v_scales=vs)
    launched, asked, cases = [], [], 0
    monkeypatch.setattr(ops, "_launch_on", lambda *args: launched.append(args))
    for call, check, good, more in ((ops.e4m3_attention, ops._check_e4m3_attention, attention, dict(workspace=workspace)),
                                    (ops.e4m3_store, lambda **o: check_store(**o, writes=True), store, {})):
        check_store = ops._check_e4m3_store
        of_call = getattr(ops, f"_check_{call.__name__}")
        monkeypatch.setattr(ops, f"_check_{call.__name__}", lambda *args, of_call=of_call: (asked.append(args), of_call(*args)))
        launched.clear(), asked.clear()
        call(**good, **more)
        assert launched and not asked
        for name, value in good.items():
            for other in _changes(value):
                if name == "q_out" and other is None:
                    continue                                    # (no queries wanted)
                operands, what = {**good, name: other}, (name, getattr(other, "shape", other), getattr(other, "dtype", None))
                launched.clear()
                try:
                    check(**operands)
                    fault = False
                except KernelError:
                    fault = True
                asked.clear()
                try:
                    call(**operands, **more)
                    refused = False
                except KernelError:
                    refused = True
                assert refused == fault and bool(launched) != refused, what
                assert bool(asked) == fault or (rows <= 1 and asked), what
                cases += 1
    assert cases > 300


def test_angles_are_those_of_64_bits():
    """Queries (1, 0) turn into the cosine and sine themselves.  Their final rounding is half a unit, 2^-25; of a sine's series 0.081 r-cubed terms are off by four
    roundings, 2^-25.6, and the angle by 2^-32 turns, 2^-29.3.  Nine in ten are the nearest 32-bit number (in a model of the series' arithmetic 96 of 100 are;
    a 32-bit angle would leave 84 of 100 whatever the functions' own rounding)."""
    from mini_llm_b200.kernels import ops
    rng = np.random.default_rng(22)
    n, half = 4000, 64
    positions = rng.integers(0, 2 ** 20, n).astype(np.int32)
    inv_freq = rng.uniform(0.1, 3.0, half)
    qkv = torch.zeros((n, 2 * half + 2 * 16), device="cuda")
    qkv[:, 0:2 * half:2] = 1.0
    q = torch.empty((n, 2 * half), device="cuda")
    ops.e4m3_store(q, qkv, 0, 2 * half, 1, 1, 2 * half, 16, 2 * half, torch.tensor(inv_freq, dtype=torch.float64, device="cuda"), 1.0, ints(positions),
                   ints([0] * n), None, None, None, None, None, writes=False)
    got = q.cpu().numpy().reshape(n, half, 2).astype(np.float64)
    angle = positions.astype(np.longdouble)[:, None] * inv_freq.astype(np.longdouble)[None, :]
    want = np.stack((np.cos(angle), np.sin(angle)), axis=-1)
    assert float(np.abs(got - want).max()) <= 2.0 ** -25 + 2.0 ** -25.6 + 2.0 ** -29
    assert (got.astype(np.float32) != want.astype(np.float32)).mean() <= 0.1
