"""The engine with its cache in 8 bits, under several ways of cutting requests into steps: what the cache holds against the plain keys and
values, and the logits against the plain implementation that attends over what the cache holds (a code that falls to the other side of
a tie is no error of the attention's).

Tolerances.  A cached entry is off by half a step of its code (2^-4 of it, 2^-10 of the scale below the normal range) and by what the key or
value it was made from is off (the logits' tolerances, of the largest entry).  A block's scale may have been raised after a query read it,
which moves the smallest codes by 2^-10 of the scale, 2^-19 of the block's largest entry: within the logits' tolerances."""

import math

import numpy as np
import pytest
import torch

import plain_gpt2
import plain_sumozen
import sumozen_helpers
from engine_helpers import bf16_atol, make_model, random_tokens, schedule_mixed, schedule_portions, schedule_tail_one_by_one, schedule_whole
from tiny_configs import RECIPES, TINY_A, TINY_C, TINY_D

pytestmark = pytest.mark.gpu

CONFIGS = {"A": (TINY_A, 16, 6.0), "C": (TINY_C, 48, 2.0), "D": (TINY_D, 64, 1.25)}         # configuration, page, sharpening
LENGTHS = {"A": {"a": 5, "b": 17, "c": 33, "d": 128}, "C": {"a": 300, "b": 45, "c": 131, "d": 2}, "D": {"a": 700, "b": 45, "c": 131, "d": 260}}
# 32-bit: the engine's bound for its logits, 1e-4, and as much again for the raised scales
F32_BOUND = 2e-4


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {}
    for key, (raw, _, sharpen) in CONFIGS.items():
        recipe, seed = RECIPES[key]
        out[key] = make_model(str(tmp_path_factory.mktemp(f"e4m3_{key}")), raw, recipe, seed, sharpen=sharpen)
    return out


def schedules(requests):
    prompts = {name: max(1, len(tokens) - 9) for name, tokens in requests.items()}
    return {"whole": schedule_whole(requests), "one_by_one": schedule_tail_one_by_one(requests, 12), "portions": schedule_portions(requests),
            "mixed": schedule_mixed(requests, prompts)}


def drive(engine, requests, steps, entries_with_pages):
    """As ``run_schedule``; also what the cache held of every request behind its last token: {name: [(k, v) of each run entry]}."""
    from mini_llm_b200.engine import StepEntry
    progress, slots, held = {n: 0 for n in requests}, {}, {}
    out = {n: np.full((len(t), engine.spec.vocab_size), np.nan, np.float32) for n, t in requests.items()}
    for step in steps:
        entries, places = [], []
        for name, n in step:
            if name not in slots:
                slots[name] = engine.open_request()
            start = progress[name]
            entries.append(StepEntry(slots[name], requests[name][start:start + n], list(range(n))))
            places += [(name, start + i) for i in range(n)]
            progress[name] += n
        logits = engine.step(entries).cpu().numpy()
        engine.check_status()
        for row, (name, position) in zip(logits, places):
            out[name][position] = row
        for name, _ in step:
            if progress[name] == len(requests[name]):
                held[name] = [tuple(x.double().cpu().numpy() for x in engine.read_kv(slots[name], entry)) for entry in entries_with_pages]
                engine.close_request(slots.pop(name))
    return out, held


def check_held(held, plain, atol):
    """What the cache holds [T, heads, size] against the plain rows."""
    got, want = np.concatenate([x.reshape(len(x), -1) for x in held], axis=1), np.concatenate([x.reshape(len(x), -1) for x in plain], axis=1)
    off = np.abs(got - want)
    # (half a step below the normal range, in scales: a scale is at most 2 / 448 of its block's largest entry)
    assert (off <= np.abs(want) * 2.0 ** -4 + np.abs(want).max() * 2.0 ** -9 / 448 + atol).all(), off.max()


def gpt2_over(folder, tokens, held, bf16):
    """The plain logits, every layer attending over what the cache holds; and the plain keys and values of each layer."""
    config, tensors = plain_gpt2.load_model(folder, round_matrices_to_bfloat16=bf16)
    rows, layers = iter(held), []
    real = plain_gpt2.multi_head_attention

    def attention(q, k, v, n_heads, scale, n_kv_heads=None, window=None):
        layers.append((k, v))
        k8, v8 = next(rows)
        return real(q, k8.reshape(k.shape), v8.reshape(v.shape), n_heads, scale, n_kv_heads, window)

    plain_gpt2.multi_head_attention = attention
    try:
        return plain_gpt2.forward(config, tensors, list(tokens)), layers
    finally:
        plain_gpt2.multi_head_attention = real


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("key", ["A", "C", "D"])
def test_gpt2_over_a_cache_in_8_bits(folders, key, dtype):
    from mini_llm_b200.engine import Engine
    raw, page, _ = CONFIGS[key]
    requests = {name: random_tokens(i + 3, n, raw["vocab_size"]) for i, (name, n) in enumerate(LENGTHS[key].items())}
    engine = Engine(folders[key], dtype=dtype, page_size=page, max_requests=4, cache_dtype="e4m3", debug_poison=True)
    assert engine.fused is None and engine.fused_reason == "the cache is held in 8 bits"
    for kind, steps in schedules(requests).items():
        got, held = drive(engine, requests, steps, range(raw["n_layer"]))
        for name, tokens in requests.items():
            want, layers = gpt2_over(folders[key], tokens, held[name], dtype == "bfloat16")
            atol = F32_BOUND if dtype == "float32" else bf16_atol(want)
            assert np.abs(got[name] - want).max() <= atol, (kind, name)
            for (k8, v8), (k, v) in zip(held[name], layers):
                for codes, rows in ((k8, k), (v8, v)):
                    check_held([codes.reshape(len(rows), -1)], [rows], 1e-4 if dtype == "float32" else 0.04 * np.abs(rows).max())
    engine.cache.check()
    chosen = {value for choice, value in engine.kernels.choices.items() if choice[0] == "e4m3_attention"}
    assert chosen == ({"e4m3_attention_plain"} if dtype == "float32"
                      else {"e4m3_attention_tiles", "e4m3_attention_step", "e4m3_attention_tiles+e4m3_attention_step"})


def sumozen_over(folder, tokens, held, monkeypatch):
    """The plain logits of a Sumozen stack whose softmax attentions read what the cache holds; and their plain keys and values."""
    config, tensors = plain_sumozen.load_model(folder)
    rows, layers = iter(held), []

    def attention(h, sizes, w, prefix):
        n, heads, groups, dim, vdim = h.shape[0], sizes["heads"], sizes["kv_heads"], sizes["dim"], sizes["vdim"]
        q, k, v = (plain_sumozen.causal_taps(h @ w[f"{prefix}.{x}"].T + w[f"{prefix}.{x}.b"], w[f"{prefix}.{x}.conv"]) for x in "qkv")
        q = plain_sumozen.rotate_interleaved(q.reshape(n, heads, dim), np.arange(n), sizes["rot"])
        layers.append((plain_sumozen.rotate_interleaved(k.reshape(n, groups, dim), np.arange(n), sizes["rot"]), v.reshape(n, groups, vdim)))
        k8, v8 = next(rows)
        out, cap = np.zeros((n, heads, vdim)), sizes.get("softcap")
        for head in range(heads):
            score = q[:, head] @ k8[:, head // (heads // groups)].T * sizes["scale"]
            score = cap * np.tanh(score / cap) if cap else score
            out[:, head] = plain_gpt2.causal_softmax(score) @ v8[:, head // (heads // groups)]
        return out.reshape(n, -1) @ w[f"{prefix}.o"].T + w[f"{prefix}.o.b"]

    with monkeypatch.context() as patch:
        patch.setattr(plain_sumozen, "capped_attention", attention)
        return plain_sumozen.forward(config, tensors, list(tokens), None), layers


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sumozen_over_a_cache_in_8_bits(tmp_path, dtype, monkeypatch):
    from mini_llm_b200.engine import Engine
    h = sumozen_helpers
    # (without experts: a token between two of them would go either way)
    raw = h.config([h.parallel(dim=16, vdim=32, scale=0.2, mlp=None), h.mamba(mlp=None),
                    h.parallel(heads=6, kv_heads=2, dim=64, vdim=64, rot_dims=64, scale=0.1, softcap=None, mlp=None)])
    folder = h.make_model(str(tmp_path / "model"), raw, seed=7, bfloat16_values=True)
    requests = {"a": random_tokens(1, 150, raw["vocab"]), "b": random_tokens(2, 40, raw["vocab"]), "c": random_tokens(3, 17, raw["vocab"])}
    engine = Engine(folder, dtype=dtype, page_size=32, cache_tokens=1024, max_requests=4, cache_dtype="e4m3", debug_poison=True)
    for kind, steps in schedules(requests).items():
        got, held = drive(engine, requests, steps, [0, 2])
        for name, tokens in requests.items():
            want, layers = sumozen_over(folder, tokens, held[name], monkeypatch)
            if dtype == "bfloat16":
                # (the bound of these stacks in bfloat16, whatever the cache holds: where a recurrence's read nearly cancels its write, the rounding of
                # its inputs shows many times over in that token and the later ones, so that no single token can be bounded)
                assert np.sqrt(((got[name] - want) ** 2).mean()) <= 0.04 * want.std(), (kind, name)
            else:
                assert np.abs(got[name] - want).max() <= F32_BOUND, (kind, name)
                for (k8, v8), (k, v) in zip(held[name], layers):
                    check_held([k8], [k], 1e-4)
                    check_held([v8], [v], 1e-4)


def test_replayed_steps_give_what_eager_ones_give(folders):
    from mini_llm_b200.engine import Engine
    raw, page, _ = CONFIGS["D"]
    requests = {name: random_tokens(i + 3, n, raw["vocab_size"]) for i, (name, n) in enumerate(LENGTHS["D"].items())}
    engine = Engine(folders["D"], page_size=page, max_requests=4, cache_dtype="e4m3")
    steps = schedules(requests)["mixed"]
    first, *others = [drive(engine, requests, steps, [0]) for _ in range(4)]
    # (the first time steps run one by one, then they are captured, then replayed)
    assert engine.step_kinds["eager"] > 0 and engine.step_kinds["replayed"] > 0
    for logits, held in others:
        for name in requests:
            np.testing.assert_array_equal(logits[name], first[0][name])
            for (k, v), (k0, v0) in zip(held[name], first[1][name]):
                np.testing.assert_array_equal(k, k0)
                np.testing.assert_array_equal(v, v0)


def test_generation_with_few_pages_and_the_bytes_of_the_cache(folders):
    from mini_llm_b200.engine import Engine
    from mini_llm_b200.generate import LLM
    prompts = [random_tokens(i, n, 1031) for i, n in enumerate((90, 33, 200, 7, 64, 150))]
    roomy = LLM(folders["D"], cache_dtype="e4m3", page_size=16).generate(prompts, max_new_tokens=24)
    # (pages for two of the requests at a time: the others wait, or are put back and their prompts run again)
    tight = LLM(folders["D"], cache_dtype="e4m3", page_size=16, cache_tokens=480, max_sessions=4).generate(prompts, max_new_tokens=24)
    assert [len(t) for t in roomy] == [len(t) for t in tight] == [24] * 6
    in_8, in_16 = (Engine(folders["D"], page_size=64, max_requests=2, cache_dtype=kind).storage.bytes() for kind in ("e4m3", None))
    assert in_8 < 0.51 * in_16


def test_what_a_cache_in_8_bits_refuses(folders, tmp_path):
    from mini_llm_b200.engine import Engine
    with pytest.raises(ValueError, match="cache_dtype"):
        Engine(folders["A"], cache_dtype="int8")
    with pytest.raises(ValueError, match="multiples of 16"):
        Engine(folders["A"], page_size=8, cache_dtype="e4m3")
    h = sumozen_helpers
    odd = h.make_model(str(tmp_path / "odd"), h.config([h.parallel(dim=16, vdim=24)]))
    with pytest.raises(ValueError, match="multiples of 16"):
        Engine(odd, page_size=16, cache_tokens=256, cache_dtype="e4m3")


def test_a_step_whose_kernel_gave_up_is_reported_and_later_steps_are_right(folders):
    from mini_llm_b200.engine import Engine, StepEntry
    from mini_llm_b200.kernels.lib import KernelError
    raw, page, _ = CONFIGS["D"]
    tokens = random_tokens(8, 400, raw["vocab_size"])
    engine = Engine(folders["D"], page_size=page, max_requests=2, cache_dtype="e4m3", cuda_graphs=False)

    def logits(check=True):
        slot = engine.open_request()
        try:
            first = engine.step([StepEntry(slot, tokens[:390], [389])])
            if check:
                engine.check_status()
            return [first.cpu().numpy()] + [engine.step([StepEntry(slot, [t], [0])]).cpu().numpy() for t in tokens[390:]]
        finally:
            engine.close_request(slot)

    want = logits()
    workspace = engine.kernels._e4m3_workspace
    workspace.wait_limit_ns, workspace.role_away = 2_000_000, 33
    with pytest.raises(KernelError, match="bounded wait"):
        logits()
    workspace.wait_limit_ns = workspace.role_away = 0
    for _ in range(2):
        for a, b in zip(logits(), want):
            np.testing.assert_array_equal(a, b)
    engine.check_status()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sumozen_with_experts_over_a_cache_in_8_bits(tmp_path, dtype, monkeypatch):
    """Every token takes all experts, so that no token lies between two of them; steps are filled up to round shapes with tokens of no request, which
    read pages of the poison and go through the router and the experts with what that makes of them."""
    from mini_llm_b200.engine import Engine
    h = sumozen_helpers
    raw = h.config([h.parallel(dim=16, vdim=32, scale=0.2, mlp=h.moe(experts=4, top=4)), h.mamba(mlp=None),
                    h.parallel(heads=6, kv_heads=2, dim=64, vdim=64, rot_dims=64, scale=0.1, softcap=None, mlp=h.moe(experts=3, top=3, shared=None))])
    folder = h.make_model(str(tmp_path / "model"), raw, seed=9, bfloat16_values=True)
    requests = {"a": random_tokens(1, 150, raw["vocab"]), "b": random_tokens(2, 40, raw["vocab"]), "c": random_tokens(3, 17, raw["vocab"])}
    engine = Engine(folder, dtype=dtype, page_size=32, cache_tokens=1024, max_requests=4, cache_dtype="e4m3", debug_poison=True)
    assert engine._can_pad
    for kind, steps in schedules(requests).items():
        for again in range(2):                                # (the second time captured steps are replayed)
            got, held = drive(engine, requests, steps, [0, 2])
            for name, tokens in requests.items():
                want, _ = sumozen_over(folder, tokens, held[name], monkeypatch)
                if dtype == "bfloat16":
                    # (the bound of these stacks in bfloat16, as above)
                    assert np.sqrt(((got[name] - want) ** 2).mean()) <= 0.04 * want.std(), (kind, name)
                else:
                    assert np.abs(got[name] - want).max() <= F32_BOUND, (kind, name)


def test_sizes_are_refused_before_weights_are_looked_for(folders, tmp_path):
    import json
    import os
    import shutil
    from mini_llm_b200.engine import Engine
    bare = str(tmp_path / "gpt2")
    os.makedirs(bare)
    shutil.copy(os.path.join(folders["A"], "config.json"), bare)                                       # (no weights)
    for page in (8, 24, 40):
        with pytest.raises(ValueError, match="multiples of 16"):
            Engine(bare, page_size=page, cache_dtype="e4m3")
    h = sumozen_helpers
    for i, mixer in enumerate((h.parallel(dim=16, vdim=24), h.parallel(dim=8, vdim=16, rot_dims=8))):
        folder = str(tmp_path / f"sumozen{i}")
        os.makedirs(folder)
        with open(os.path.join(folder, "config.json"), "w") as handle:
            json.dump(h.config([h.mamba(), mixer]), handle)
        with pytest.raises(ValueError, match="multiples of 16"):
            Engine(folder, page_size=16, cache_tokens=256, cache_dtype="e4m3")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_preempted_requests_are_right_over_what_the_cache_holds_each_time(folders, dtype):
    """So few pages that decoding requests are preempted and their tokens run again as a prompt, which stores them in other steps than before.  Whenever a
    request is closed, preempted or at its end, what the cache held of it is that of its tokens, and its logits are the plain ones over that;
    every token is the largest of its logits."""
    from mini_llm_b200.generate import LLM
    raw = CONFIGS["D"][0]
    prompts = [random_tokens(30 + i, n, raw["vocab_size"]) for i, n in enumerate((90, 60, 75))]
    llm = LLM(folders["D"], dtype=dtype, cache_dtype="e4m3", page_size=16, cache_tokens=272, max_sessions=3, run_ahead=False)
    engine, of_slot, closed = llm.engine, {}, []
    step, close = engine.step, engine.close_request

    def recorded_step(entries, *args, **how):
        logits = step(entries, *args, **how)
        rows = iter(logits.cpu().numpy() if logits is not None else ())
        for entry in entries:
            tokens, seen = of_slot.setdefault(entry.slot, ([], {}))
            for place in entry.want:
                seen[len(tokens) + place] = next(rows)
            tokens.extend(int(t) for t in entry.tokens)
        return logits

    def recorded_close(slot):
        if slot in of_slot:
            closed.append((*of_slot.pop(slot), [tuple(x.double().cpu().numpy() for x in engine.read_kv(slot, layer)) for layer in range(raw["n_layer"])]))
        close(slot)

    engine.step, engine.close_request = recorded_step, recorded_close
    got = llm.generate(prompts, max_new_tokens=40)
    preemptions = llm.scheduler.stats()["preemptions"]
    assert preemptions >= 1 and len(closed) == 3 + preemptions
    chosen = [{} for _ in prompts]
    for tokens, seen, held in closed:
        which = [i for i, prompt in enumerate(prompts) if tokens[:len(prompt)] == list(prompt)]
        assert len(which) == 1 and tokens == (list(prompts[which[0]]) + got[which[0]])[:len(tokens)]
        want, layers = gpt2_over(folders["D"], tokens, held, dtype == "bfloat16")
        atol = F32_BOUND if dtype == "float32" else bf16_atol(want)
        for position, logits in seen.items():
            assert np.abs(logits - want[position]).max() <= atol, position
            chosen[which[0]][position + 1 - len(prompts[which[0]])] = int(logits.argmax())
        for (k8, v8), (k, v) in zip(held, layers):
            for codes, rows in ((k8, k), (v8, v)):
                check_held([codes.reshape(len(rows), -1)], [rows], 1e-4 if dtype == "float32" else 0.04 * np.abs(rows).max())
    for tokens, of_request in zip(got, chosen):
        assert tokens == [of_request[i] for i in range(40)]
    assert engine.cache.pages_in_use() == [0]
    engine.cache.check()
