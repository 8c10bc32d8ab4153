"""Keys and values held in 8 bits: storing a step's tokens, and the attention that reads them.

The cache keeps a key or value as e4m3 codes (a byte each: sign, 4 bits of exponent, 3 of fraction) with one 32-bit
scale, a power of two, for each block of 16 positions and key/value head; what an entry stands for is code * scale.
Pages are ``[pages, kv_heads, page, size]``, scales ``[pages, kv_heads, page / 16]``; a request's row of the block table
names its pages in order.  A step brings entries: tokens of a request at positions start, start + 1, ...; a single token
while the request decodes, a portion of its prompt before.

``store``: the queries' and keys' first ``rot`` entries turn in interleaved pairs (2i, 2i + 1) by position * f_i, then keys
and values are appended to their blocks.  Rotation keeps a pair's length, so that a key's scale is known before any angle:
with n = x^2 + y^2 of a turned pair, x^2 of an entry that does not turn and of a value's, the scale is the least power of two
s >= 2^-64 with n <= (448 s)^2 for every row of the block so far (448 is the largest code).  Where new tokens raise the scale
of a block that holds tokens already, those codes are rounded again at the new scale (exact but for the smallest).

``attention``: softmax(q . k * scale) v over the keys at positions <= the query's, of those the last ``window`` if there is
one; with ``cap`` the score is cap * tanh(score / cap); query head h reads key/value head h // (heads / kv_heads).
"""

import math

import torch

own = False

BLOCK = 16
TOP = 448.0
LEAST_EXPONENT = -64


# ---- the cases -----------------------------------------------------------------------------------

def _spread(count, low, high, seed, tokens=1):
    """``count`` entries of ``tokens`` tokens at starts spread over low..high, as text."""
    state, parts = seed * 2654435761 % 2 ** 32, []
    for _ in range(count):
        state = (state * 1664525 + 1013904223) % 2 ** 32
        parts.append(f"{int(low * (high / low) ** (state / 2 ** 32))}:{tokens}")
    return " ".join(parts)


def listed():
    small = {"heads": 12, "kv_heads": 12, "dim": 64, "vdim": 64}          # the benchmark's GPT-2 stack
    shared = {"heads": 12, "kv_heads": 4, "dim": 64, "vdim": 64}          # the benchmark's stacks with shared heads
    large = {"heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128}         # heads as larger models have them
    return [
        # one request decodes: the least a step brings, where only the launch and its latency count
        {"name": "store_one_token", "op": "store", **shared, "rot": 64, "page": 64, "entries": "777:1"},
        # 64 requests decode
        {"name": "store_64_tokens", "op": "store", **large, "rot": 128, "page": 64, "entries": _spread(64, 40, 2000, 1)},
        # a full step: a long portion that goes on inside a block, short prompts, and requests that decode beside them
        {"name": "store_mixed_step", "op": "store", **small, "rot": 0, "page": 64,
         "entries": "345:1500 0:333 0:97 " + _spread(40, 30, 900, 2)},
        # a long prompt in one step
        {"name": "store_long_prompt", "op": "store", **large, "rot": 96, "page": 128, "entries": "0:8192"},
        # one request decodes near the end of a context of 1,024
        {"name": "attention_one_token", "op": "attention", **small, "page": 64, "window": 0, "cap": 0.0, "entries": "1000:1"},
        # 64 requests decode, contexts of all lengths
        {"name": "attention_64_tokens", "op": "attention", **large, "page": 64, "window": 0, "cap": 0.0, "entries": _spread(64, 100, 4000, 3)},
        # capped scores within a window
        {"name": "attention_window_cap", "op": "attention", **shared, "page": 16, "window": 1024, "cap": 50.0, "entries": _spread(31, 1, 4000, 4)},
        # one request decodes at the end of a long document
        {"name": "attention_long_context", "op": "attention", **large, "page": 128, "window": 0, "cap": 0.0, "entries": "131071:1"},
        # a short prompt alone
        {"name": "attention_short_prompt", "op": "attention", **small, "page": 64, "window": 0, "cap": 0.0, "entries": "0:100"},
        # a full step: a portion of a prompt behind what is cached, short prompts, and requests that decode beside them
        {"name": "attention_mixed_step", "op": "attention", **shared, "page": 64, "window": 0, "cap": 50.0,
         "entries": "1345:1024 0:333 0:97 " + _spread(40, 30, 2000, 5)},
        # a portion of a long document
        {"name": "attention_portion", "op": "attention", **large, "page": 64, "window": 0, "cap": 0.0, "entries": "14321:1999"},
        # a long prompt in one step
        {"name": "attention_long_prompt", "op": "attention", **small, "page": 64, "window": 0, "cap": 0.0, "entries": "0:16000"},
    ]


def draw(rng):
    def log(low, high):
        return int(round(low * (high / low) ** rng.random()))

    while True:
        dim = rng.choice((32, 64, 64, 96, 128, 128))
        kv_heads, group = rng.choice((1, 2, 3, 4, 5, 8, 12)), rng.choice((1, 1, 2, 3, 4, 8))
        case = {"op": rng.choice(("store", "attention", "attention")), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "vdim": dim if rng.random() < 0.8 else rng.choice((32, 64, 128)), "page": rng.choice((16, 32, 64, 128))}
        if case["op"] == "store":
            case["rot"] = rng.choice((0, dim, dim, dim // 2))
        else:
            case["window"] = rng.choice((0, 0, 0, log(1, 2000)))
            case["cap"] = rng.choice((0.0, 0.0, 50.0, 20.0))
        kind = rng.choice(("single", "portions", "mixed"))
        entries = []
        if kind != "portions":
            most = log(16, 40000 if case["op"] == "attention" else 4000)
            entries += [f"{log(1, most) - 1}:1" for _ in range(log(1, 64))]
        if kind != "single":
            entries += [f"{rng.choice((0, log(1, 8000)))}:{log(2, 4000)}" for _ in range(log(1, 6))]
        rng.shuffle(entries)
        case["entries"] = " ".join(entries)
        total, pairs = work(case), _entries(case)
        filled = len(pairs) * max(count for _, count in pairs) * max(start + count for start, count in pairs) * case["heads"]
        if total["flops"] <= 3e11 and total["bytes"] <= 1.8e8 and (case["op"] == "store" or filled <= 2e9):
            return case


def _entries(case):
    return [tuple(int(n) for n in entry.split(":")) for entry in case["entries"].split()]


def _seen(start, count, window):
    """Pairs of a query and a key that it sees, and the keys that any of them sees."""
    if not window:
        return count * start + count * (count + 1) // 2, start + count
    pairs = sum(min(window, start + i + 1) for i in range(count))
    return pairs, start + count - max(0, start - window + 1)


def work(case):
    heads, kv_heads, dim, vdim = case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    tokens = sum(count for _, count in _entries(case))
    if case["op"] == "store":
        columns = heads * dim + kv_heads * (dim + vdim)
        blocks = sum((start + count - 1) // BLOCK - start // BLOCK + 1 for start, count in _entries(case))
        held = tokens * (2 * columns + 2 * heads * dim + kv_heads * (dim + vdim)) + 8 * blocks * kv_heads
        return {"bytes": held, "flops": 6 * tokens * columns}
    seen = [_seen(start, count, case["window"]) for start, count in _entries(case)]
    pairs, keys = sum(p for p, _ in seen), sum(k for _, k in seen)
    held = kv_heads * keys * (dim + vdim) + 8 * kv_heads * (keys // BLOCK + 1) + 2 * tokens * heads * (dim + vdim)
    return {"bytes": held, "flops": 2 * pairs * heads * (dim + vdim)}


# ---- what a program has in hand ------------------------------------------------------------------

def _filled(generator, pages, kv_heads, page, size):
    """Pages of 8-bit rows as earlier steps have left them: rows of all sizes, each block with its scale."""
    blocks = page // BLOCK
    rows = torch.randn((pages, kv_heads, blocks, BLOCK, size), generator=generator, device="cuda", dtype=torch.float32)
    rows *= torch.exp2(2.0 * torch.randn((pages, kv_heads, blocks, 1, 1), generator=generator, device="cuda", dtype=torch.float32) - 1.0)
    exponent = _exponent(rows.square().amax(dim=(3, 4)))
    codes = (rows * torch.exp2(-exponent)[..., None, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return codes.view(pages, kv_heads, page, size), torch.exp2(exponent)


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    heads, kv_heads, dim, vdim, page = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["page"]
    entries = _entries(case)
    starts, counts = [start for start, _ in entries], [count for _, count in entries]
    tokens, blocks = sum(counts), [-(-(start + count) // page) for start, count in entries]
    pages = sum(blocks) + 1

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    # every request's pages lie anywhere in the pool; behind its last page a row of the block table names none
    places = torch.randperm(pages - 1, generator=generator, device="cuda").to(torch.int32)
    taken = torch.arange(max(blocks), device="cuda")[None, :] < ints(blocks)[:, None]
    table = torch.full((len(entries), max(blocks)), -1, dtype=torch.int32, device="cuda")
    table[taken] = places
    state = {"case": case, "block_table": table, "item_start": ints(starts), "item_count": ints(counts),
             "item_offset": ints([sum(counts[:i]) for i in range(len(counts))])}
    state["k_pages"], state["k_scales"] = _filled(generator, pages, kv_heads, page, dim)
    state["v_pages"], state["v_scales"] = _filled(generator, pages, kv_heads, page, vdim)
    item = torch.repeat_interleave(torch.arange(len(entries), device="cuda"), state["item_count"].long())
    state["token_item"] = item.to(torch.int32)
    state["positions"] = (state["item_start"][item] + torch.arange(tokens, device="cuda") - state["item_offset"][item]).to(torch.int32)
    if case["op"] == "store":
        columns = heads * dim + kv_heads * (dim + vdim)
        qkv = torch.randn((tokens, columns), generator=generator, device="cuda", dtype=torch.float32)
        # some entries of a head are larger than the rest in all tokens, as trained projections have them
        qkv *= torch.exp2(1.5 * torch.randn((1, columns), generator=generator, device="cuda", dtype=torch.float32))
        state["qkv"] = qkv.to(torch.bfloat16)
        half = case["rot"] // 2
        state["inv_freq"] = torch.tensor([10000.0 ** (-i / half) for i in range(half)] or [0.0], dtype=torch.float64, device="cuda")
        state["q"] = torch.empty((tokens, heads * dim), dtype=torch.bfloat16, device="cuda")
    else:
        state["q"] = torch.randn((tokens, heads * dim), generator=generator, device="cuda", dtype=torch.float32).to(torch.bfloat16)
        state["out"] = torch.empty((tokens, heads * vdim), dtype=torch.bfloat16, device="cuda")
    return state


# ---- one pass ------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "store":
        if own:
            _store_own(state)
        else:
            _store_plain(state)
        return {"q": state["q"], "k_pages": state["k_pages"], "v_pages": state["v_pages"], "k_scales": state["k_scales"],
                "v_scales": state["v_scales"]}
    if own:
        _attention_own(state)
        return state["out"]
    return _attention_plain(state)


def _store_own(state):
    from mini_llm_b200.kernels import ops
    c = state["case"]
    heads, kv_heads, dim, vdim = c["heads"], c["kv_heads"], c["dim"], c["vdim"]
    ops.e4m3_store(state["q"], state["qkv"], heads * dim, (heads + kv_heads) * dim, heads, kv_heads, dim, vdim, c["rot"], state["inv_freq"],
                   1.0, state["positions"], state["token_item"], state["block_table"], state["k_pages"], state["v_pages"],
                   state["k_scales"], state["v_scales"])


_workspaces = {}        # as a serving program keeps them: one for each size of a value


def _attention_own(state):
    from mini_llm_b200.kernels import ops
    c = state["case"]
    if c["vdim"] not in _workspaces:
        _workspaces[c["vdim"]] = ops.e4m3_workspace(state["q"].device, c["vdim"])
    counts = [count for _, count in _entries(c)]
    ops.e4m3_attention(state["out"], state["q"], state["k_pages"], state["v_pages"], state["k_scales"], state["v_scales"],
                       state["block_table"], state["item_offset"], state["item_count"], state["item_start"], c["heads"], c["kv_heads"],
                       c["dim"] ** -0.5, cap=c["cap"], window=c["window"], longest=max(counts), singles=min(counts) == 1,
                       workspace=_workspaces[c["vdim"]])


def _exponent(square):
    """The least whole e >= -64 with square <= (448 * 2^e)^2, in the type of ``square``: no rounding decides it."""
    e = torch.floor(0.5 * torch.log2((square.double() / TOP ** 2).clamp(min=2.0 ** -140)))
    e = torch.where(square.double() <= TOP ** 2 * torch.exp2(2.0 * e), e, e + 1.0)
    e = torch.where(square.double() <= TOP ** 2 * torch.exp2(2.0 * e), e, e + 1.0)
    return e.clamp(min=LEAST_EXPONENT).to(square.dtype)


def _turned(rows, rot, positions, inv_freq):
    """rows [T, heads, size] in 32 bits with their first ``rot`` entries turned; the angles are 64-bit."""
    if not rot:
        return rows
    angle = positions.double()[:, None] * inv_freq[None, :]
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    x, y = rows[..., 0:rot:2], rows[..., 1:rot:2]
    turned = torch.stack((x * cos - y * sin, x * sin + y * cos), dim=-1).flatten(-2)
    return torch.cat((turned, rows[..., rot:]), dim=-1)


def _append_plain(rows, squares, state, pages, scales):
    """Rows [T, kv_heads, size] into their blocks; squares [T, kv_heads]: what bounds each row's entries."""
    page, width = pages.shape[2], pages.shape[3]
    position, item = state["positions"].long(), state["token_item"].long()
    block = position // BLOCK
    # the tokens of one block stand side by side: their run's number, and its first token
    begins = torch.ones_like(block, dtype=torch.bool)
    begins[1:] = (block[1:] != block[:-1]) | (item[1:] != item[:-1])
    run_of = torch.cumsum(begins.long(), 0) - 1
    first = torch.nonzero(begins)[:, 0]
    where = state["block_table"].long()[item, position // page]
    top = torch.zeros((first.shape[0], rows.shape[1]), dtype=rows.dtype, device=rows.device)
    top = top.scatter_reduce(0, run_of[:, None].expand(-1, rows.shape[1]), squares, "amax")
    new = torch.exp2(_exponent(top))
    # what the block holds already: positions before the run's first
    spots, places = where[first], (position[first] % page) // BLOCK
    held = scales[spots, :, places]
    lead = position[first] % BLOCK
    new = torch.where((lead > 0)[:, None], torch.maximum(new, held), new)
    index = places[:, None] * BLOCK + torch.arange(BLOCK, device=rows.device)
    codes = pages.view(torch.uint8)[spots[:, None], :, index]                       # [runs, 16, kv_heads, size]
    again = (codes.view(torch.float8_e4m3fn).float() * (held / new)[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    older = (torch.arange(BLOCK, device=rows.device)[None, :] < lead[:, None])[..., None, None]
    pages.view(torch.uint8)[spots[:, None], :, index] = torch.where(older, again, codes)
    scales[spots, :, places] = new
    fresh = (rows / new[run_of][..., None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    pages.view(torch.uint8)[where, :, position % page] = fresh.view(torch.uint8)


def _store_plain(state):
    c = state["case"]
    heads, kv_heads, dim, vdim, rot = c["heads"], c["kv_heads"], c["dim"], c["vdim"], c["rot"]
    rows = state["qkv"].float()
    q = rows[:, :heads * dim].view(-1, heads, dim)
    k = rows[:, heads * dim:(heads + kv_heads) * dim].view(-1, kv_heads, dim)
    v = rows[:, (heads + kv_heads) * dim:].view(-1, kv_heads, vdim)
    state["q"].copy_(_turned(q, rot, state["positions"], state["inv_freq"]).flatten(1))
    square = k * k
    pairs = torch.cat((square[..., 0:rot:2] + square[..., 1:rot:2], square[..., rot:]), dim=-1)
    _append_plain(_turned(k, rot, state["positions"], state["inv_freq"]), pairs.amax(dim=-1), state, state["k_pages"], state["k_scales"])
    _append_plain(v, (v * v).amax(dim=-1), state, state["v_pages"], state["v_scales"])


def _attention_plain(state):
    c = state["case"]
    heads, kv_heads, dim, vdim, page = c["heads"], c["kv_heads"], c["dim"], c["vdim"], c["page"]
    table = state["block_table"].long().clamp(min=0)
    entries, reach, most = table.shape[0], table.shape[1] * page, max(count for _, count in _entries(c))
    # every entry's keys and values in order, and its queries, filled up to the longest
    k = state["k_pages"].float() * state["k_scales"].repeat_interleave(BLOCK, dim=2)[..., None]
    v = state["v_pages"].float() * state["v_scales"].repeat_interleave(BLOCK, dim=2)[..., None]
    k = k[table].transpose(1, 2).reshape(entries, kv_heads, reach, dim)
    v = v[table].transpose(1, 2).reshape(entries, kv_heads, reach, vdim)
    item = state["token_item"].long()
    row = state["positions"].long() - state["item_start"].long()[item]
    q = torch.zeros((entries, most, heads, dim), dtype=torch.float32, device="cuda")
    q[item, row] = state["q"].float().view(-1, heads, dim)
    q = q.view(entries, most, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).reshape(entries, kv_heads, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(dim ** -0.5)
    if c["cap"]:
        score = score.div_(c["cap"]).tanh_().mul_(c["cap"])
    at = state["item_start"].long()[:, None] + torch.arange(most, device="cuda")[None, :]
    key = torch.arange(reach, device="cuda")
    hidden = key[None, None, :] > at[..., None]
    if c["window"]:
        hidden |= key[None, None, :] <= at[..., None] - c["window"]
    score = score.view(entries, kv_heads, heads // kv_heads, most, reach).masked_fill_(hidden[:, None, None], -math.inf)
    # (a row filled up past its entry's tokens may see no key: it is left out below)
    weight = (score - score.amax(dim=-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = weight.sum(dim=-1, keepdim=True)
    out = torch.matmul(weight.view(entries, kv_heads, -1, reach), v).view(entries, kv_heads, heads // kv_heads, most, vdim) / total
    return out.permute(0, 3, 1, 2, 4).reshape(entries, most, heads * vdim)[item, row].to(torch.bfloat16)


# ---- the definition, in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return _store_exact(case, state) if case["op"] == "store" else _attention_exact(case, state)


def _nearest_code(x):
    """64-bit numbers rounded once to e4m3 (half to even; beyond 448 to 448)."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _store_exact(case, state):
    heads, kv_heads, dim, vdim, rot, page = (case[name] for name in ("heads", "kv_heads", "dim", "vdim", "rot", "page"))
    x = state["qkv"].double()
    angle = state["positions"].double()[:, None] * state["inv_freq"][None, :rot // 2]
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]

    def rotate(rows):
        if not rot:
            return rows
        pairs = torch.view_as_complex(rows[..., :rot].reshape(*rows.shape[:2], rot // 2, 2).contiguous())
        return torch.cat((torch.view_as_real(pairs * turn).flatten(-2), rows[..., rot:]), dim=-1)

    q, k, v = x.split([heads * dim, kv_heads * dim, kv_heads * vdim], dim=1)
    k, v = k.reshape(-1, kv_heads, dim), v.reshape(-1, kv_heads, vdim)
    result = {"q": rotate(q.reshape(-1, heads, dim)).flatten(1)}
    lengths = torch.cat((k[..., :rot].unflatten(-1, (-1, 2)).square().sum(-1), k[..., rot:].square()), dim=-1) if rot else k.square()
    table = state["block_table"].cpu()
    for name, rows, squares in (("k", rotate(k), lengths.amax(-1)), ("v", v, v.square().amax(-1))):
        pages, scales = state[name + "_pages"].double(), state[name + "_scales"].double()
        row = 0
        for item, (start, count) in enumerate(_entries(case)):
            position = start
            while position < start + count:
                block, place = position // BLOCK * BLOCK, int(table[item, position // page])
                many = min(block + BLOCK, start + count) - position
                part, slot = slice(row, row + many), block % page
                # square = m * 2^x with m in [1/2, 1), and 448^2 = 0.765625 * 2^18
                m, x = torch.frexp(squares[part].amax(0).clamp(min=2.0 ** -200))
                scale = torch.exp2(torch.ceil((x - 18 + (m > 0.765625)).double() / 2).clamp(min=-64.0))
                if position > block:
                    scale = torch.maximum(scale, scales[place, :, slot // BLOCK])
                    old = slice(slot, slot + position - block)
                    pages[place, :, old] = _nearest_code(pages[place, :, old] * (scales[place, :, slot // BLOCK] / scale)[:, None, None])
                scales[place, :, slot // BLOCK] = scale
                at = position % page
                pages[place, :, at:at + many] = _nearest_code(rows[part] / scale[None, :, None]).transpose(0, 1)
                row, position = row + many, position + many
        result[name + "_pages"], result[name + "_scales"] = pages, scales
    return result


def _attention_exact(case, state):
    heads, kv_heads, dim, vdim, page = (case[name] for name in ("heads", "kv_heads", "dim", "vdim", "page"))
    out, row = [], 0
    for item, (start, count) in enumerate(_entries(case)):
        pages = state["block_table"][item, :-(-(start + count) // page)].long()

        def rows(name, size):
            scaled = state[name + "_pages"][pages].double().unflatten(2, (-1, BLOCK)) * state[name + "_scales"][pages].double()[..., None, None]
            return scaled.flatten(2, 3).transpose(0, 1).reshape(kv_heads, -1, size)[:, :start + count]

        k, v = rows("k", dim), rows("v", vdim)
        for first in range(0, count, 1024):
            many = min(1024, count - first)
            q = state["q"][row + first:row + first + many].double().view(many, kv_heads, heads // kv_heads, dim)
            score = torch.einsum("tkgd,kld->kgtl", q, k) / math.sqrt(dim)
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            behind = (start + first + torch.arange(many, device="cuda"))[:, None] - torch.arange(start + count, device="cuda")[None, :]
            score[..., (behind < 0) | (behind >= (case["window"] or start + count))] = -math.inf
            out.append(torch.einsum("kgtl,kld->tkgd", torch.softmax(score, dim=-1), v).reshape(many, -1))
        row += count
    return torch.cat(out)
