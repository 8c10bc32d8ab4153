"""A cache in 8 bits against its definition in 64 bits (``plain_e4m3``): the store with the rotation on the way, and the attention
that reads it, for single tokens and portions of prompts.

Tolerances.  A code is half a step off at most: 2^-4 of its value, 2^-10 below the normal range.  Scales, and codes of rows that do
not turn (16-bit rows over a power of two are exact in 32 bits), are equal.  A turned entry comes from two products of 32-bit numbers and an
angle that is exact to 2^-24 turns: some 2^-21 of its pair, which is 448 scales at most.

Attention in bfloat16: 2^-8 of the result for its own rounding, and of the sum of the weights times |v| 2^-11 for the
weights, which are 16-bit floats, and 2^-20 (1 + size) for the scores: a score of products of sum `size` is some 8 sums cut off
at 2^-23, its 32-bit arithmetic and the exponential a few units of 2^-24 of it, and an error of a score is as
large a relative one of its weight.  With 32-bit queries sums of N terms, each rounded to 2^-24."""

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
    want, spread, most = plain.attention(q.float().cpu().numpy(), pool.codes["k"], pool.codes["v"], pool.scales["k"], pool.scales["v"], table,
                                         entries, heads, scale, cap, window)
    got = got.float().cpu().numpy().astype(np.float64)
    rows = np.zeros(got.shape[0], bool)
    for offset, count, _ in entries:
        rows[offset:offset + count] = True
    assert (got[~rows] == 3.0).all()
    got, want, spread = got[rows], want[rows], spread[rows]
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    if dtype == torch.bfloat16:
        bound = np.abs(want) * 2.0 ** -8 + spread * (2.0 ** -11 + 2.0 ** -20 * (1 + most))
    else:
        n = max(start + count for _, count, start in entries)
        bound = np.abs(want) * 2.0 ** -24 + spread * 2.0 ** -24 * (n + 64 + 8 * (1 + most))
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
