"""The engine with a cache in 8 bits, and its steps of drafted tokens: on the test double, and on the GPU."""

import numpy as np
import pytest
import torch

import plain_qwen2 as plain
from distie_amd import LLM, EngineConfig, SamplingParams, StepEntry
from distie_amd.cache import CacheManager
from distie_amd.config import load_model_config
from distie_amd.engine.batch import draw_tree
from distie_amd.engine.model import Model
from distie_amd.engine.runner import ModelRunner
from distie_amd.weights import load_into
from eight_bit_util import EightBitOps, quantised_keys_and_values
from engine_util import FP32_TOL, make_model_dir, oracle, random_ids

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module", params=["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
def ops(request):
    if request.param == "cpu":
        return EightBitOps()
    from distie_amd.kernels.hip_ops import HipOps

    return HipOps("cuda:0")


@pytest.fixture(scope="module", params=[("A", F32), ("B", F32), ("C", BF16)], ids=["A-fp32", "B-fp32", "C-bf16"])
def model(request, tmp_path_factory):
    name, dtype = request.param
    cfg = {"A": plain.TINY_A, "B": plain.TINY_B, "C": plain.TINY_C}[name]
    folder, weights = make_model_dir(tmp_path_factory.mktemp(f"trees{name}"), cfg, seed=23, dtype=dtype)
    return cfg, {"A": 4, "B": 8, "C": 16}[name], folder, weights, dtype


def runner_of(model, ops, cache_dtype=None, **options):
    cfg, block, folder, _, dtype = model
    built = Model(load_model_config(folder).model_spec())
    built.use_cache_dtype(cache_dtype)
    load_into(built, folder, ops.device, dtype)
    cache = CacheManager(built.cache_requirements(), block, options.get("pages", 64), 8, device=ops.device, dtype=dtype)
    return ModelRunner(built, cache, ops, dtype)


def near(got, want, dtype, eight=False):
    """Against the plain implementation. Float32 over a cache in float32: within FP32_TOL. Either bfloat16 or a cache in 8 bits: within
    the bounds that the engine's bfloat16 runs are held to (1/16 of the largest logit, 1/64 in the root mean square). Both: four times
    those. Rounding to bfloat16 moves a value x by up to 2^-8 |x|, and the codes are 2^-4 to 2^-3 |x| apart, so up to one value in 16
    falls to another code, which moves it by up to 2^-3 |x|: in the root mean square 2^-3.5 / 4 = 0.022 |x|, ten times the 2^-8 / sqrt(3) =
    0.0023 |x| of a rounding to bfloat16 alone. Keys and values are two of the about eight roundings of a layer, whose squares add
    up: (6 + 2 * 100) / 8 = 26, five times the error."""
    diff, scale = got.float().cpu() - want, float(want.abs().max())
    if dtype == F32 and not eight:
        assert float(diff.abs().max()) < FP32_TOL
        return
    more = 4 if eight and dtype == BF16 else 1
    assert float(diff.abs().max()) < more * scale / 16 and float(diff.pow(2).mean().sqrt()) < more * scale / 64


def plain_logits(model, ids, eight):
    if not eight:
        return oracle(model[3], model[0], ids)
    with quantised_keys_and_values():
        return oracle(model[3], model[0], ids)


@pytest.mark.parametrize("cuts", [[60], [1] * 60, [7, 1, 20, 2, 30]])
def test_a_cache_in_8_bits(model, ops, cuts):
    runner = runner_of(model, ops, "e4m3")
    ids = random_ids(model[0], 60, 5)
    out, at = [], 0
    for n in cuts:
        out.append(runner.step([StepEntry("a", ids[at:at + n], list(range(n)))]))
        at += n
    near(torch.cat(out), plain_logits(model, ids, True), model[4], True)
    runner.finish("a")
    runner.cache.check()
    page = sum(t.numel() * t.element_size() for t in runner.cache.groups[0].tensors.values())
    wide = sum(t.numel() * t.element_size() for t in runner_of(model, ops).cache.groups[0].tensors.values())
    dim = runner.model.blocks[0].mixer.head_dim
    assert page * dim * (4 if model[4] == F32 else 2) == wide * (dim + 1)            # a byte a value and one for each row


@pytest.mark.parametrize("eight", [False, True])
def test_a_tree_beside_chains(model, ops, eight):
    """Every drafted token's logits are those of its own path behind the context; what is kept is that path."""
    cfg = model[0]
    runner = runner_of(model, ops, "e4m3" if eight else None)
    prompts = {"a": random_ids(cfg, 21, 1), "b": random_ids(cfg, 3, 2), "c": random_ids(cfg, 34, 3)}
    runner.step([StepEntry(r, ids) for r, ids in prompts.items()])
    rng = np.random.default_rng(7)
    for turn in range(3):
        drafts = {"a": (random_ids(cfg, 9, 10 + turn), [-1, 0, 0, 1, 1, 2, 5, 6, -1]),
                  "b": (random_ids(cfg, 5, 20 + turn), None),
                  "c": (random_ids(cfg, 70, 30 + turn), [-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, 70)])}
        step = {r: d for r, d in drafts.items() if r != "c" or turn == 1}
        logits = runner.step([StepEntry(r, ids, list(range(len(ids))), parents) for r, (ids, parents) in step.items()])
        at, paths = 0, {}
        for r, (ids, parents) in step.items():
            parents = list(range(-1, len(ids) - 1)) if parents is None else parents
            cached = runner.cache.request(r).num_cached
            assert cached == len(prompts[r])                     # nothing counts before it is kept
            for i in sorted({0, len(ids) - 1, *rng.integers(0, len(ids), 4).tolist()}):
                path = [i]
                while parents[path[0]] >= 0:
                    path.insert(0, parents[path[0]])
                want = plain_logits(model, prompts[r] + [ids[j] for j in path], eight)[-1:]
                near(logits[at + i:at + i + 1], want, model[4], eight)
                if r not in paths or len(path) > len(paths[r]):
                    paths[r] = path[:6]
            at += len(ids)
        if turn == 2:
            paths["b"] = []
        runner.keep(paths)
        for r, path in paths.items():
            prompts[r] += [step[r][0][j] for j in path]
            assert runner.cache.request(r).num_cached == len(prompts[r])
    # what follows is attended over the kept paths
    last = {r: random_ids(cfg, 2, 40)[:1 + (r == "a")] for r in prompts}
    logits = runner.step([StepEntry(r, ids, [len(ids) - 1]) for r, ids in last.items()])
    for row, (r, ids) in zip(logits, last.items()):
        near(row[None], plain_logits(model, prompts[r] + ids, eight)[-1:], model[4], eight)
    for r in prompts:
        runner.finish(r)
    runner.cache.check()


def test_drafts_that_are_not_kept_are_written_over(model, ops):
    cfg = model[0]
    runner = runner_of(model, ops)
    prompt, ids = random_ids(cfg, 9, 1), random_ids(cfg, 6, 2)
    runner.step([StepEntry("a", prompt)])
    runner.step([StepEntry("a", ids, [], [-1, 0, 0, 1, 2, 2])])
    logits = runner.step([StepEntry("a", ids[:2], [0, 1])])
    near(logits, oracle(model[3], cfg, prompt + ids[:2])[-2:], model[4])
    with pytest.raises(ValueError, match="no drafted tokens"):
        runner.keep({"a": [0]})


def test_what_keep_and_trees_refuse(model, ops):
    cfg = model[0]
    runner = runner_of(model, ops)
    ids = random_ids(cfg, 6, 2)
    runner.step([StepEntry("a", ids)])
    for parents in ([-1, 1], [-2, 0], [0, -1], [-1], [-1, 0, 1]):
        with pytest.raises(ValueError):
            runner.step([StepEntry("a", ids[:2], [], parents)])
    runner.step([StepEntry("a", ids, [], [-1, 0, 0, 1, 2, -1])])
    for path in ([1], [0, 3], [0, 1, 4], [6], [-1], [0, 0], [2, 4]):
        with pytest.raises(ValueError, match="does not follow"):
            runner.keep({"a": path})
    with pytest.raises(ValueError, match="no drafted tokens"):
        runner.keep({"b": [0]})
    runner.keep({"a": [5]})
    assert runner.cache.request("a").num_cached == 7
    with pytest.raises(ValueError, match="no drafted tokens"):
        runner.keep({"a": [0]})
    runner.step([StepEntry("a", ids[:2], [], [-1, 0])])
    runner.cache.reset("a")
    with pytest.raises(ValueError, match="no drafted tokens"):
        runner.keep({"a": [0]})


@pytest.mark.parametrize("prompt", [0, 6])
@pytest.mark.parametrize("gone", ["reset", "released and added", "reset and cached again", "other request"])
def test_drafts_whose_pages_are_gone_are_not_kept(model, ops, prompt, gone):
    """Drafted entries are kept as long as the request has held on to their pages, with and without something cached in front of them."""
    cfg = model[0]
    runner = runner_of(model, ops)
    ids = random_ids(cfg, 6, 2)
    if prompt:
        runner.step([StepEntry("a", ids[:prompt])])
    runner.step([StepEntry("a", ids[:3], [], [-1, 0, 0])])
    if gone.startswith("re"):
        runner.cache.reset("a") if gone.startswith("reset") else runner.cache.release("a")
        if gone == "released and added":
            runner.cache.add("a")
        if gone == "reset and cached again" and prompt:             # by someone else's step than this runner's
            runner.cache.reserve("a", prompt)
            runner.cache.commit("a", prompt)
    else:
        runner.cache.release("a")
        runner.step([StepEntry("b", ids)])
    cached = runner.cache.request("a").num_cached if "a" in runner.cache else None
    for path in ([0], [0, 1], [0, 2], []):
        with pytest.raises(ValueError, match="no drafted tokens"):
            runner.keep({"a": path})
    assert (runner.cache.request("a").num_cached if "a" in runner.cache else None) == cached
    runner.cache.check()


def test_a_refused_step_leaves_drafts_to_be_kept(model, ops):
    cfg = model[0]
    runner = runner_of(model, ops)
    prompt, ids = random_ids(cfg, 9, 1), random_ids(cfg, 6, 2)
    runner.step([StepEntry("a", prompt)])
    runner.step([StepEntry("a", ids, [], [-1, 0, 0, 1, 2, 2])])
    for wrong in ([StepEntry("a", ids[:2], [], [-1, 1])], [StepEntry("a", ids[:2], [2])], [StepEntry("a", [cfg["vocab_size"]], [0])],
                  [StepEntry("a", [])], [StepEntry("a", ids[:1]), StepEntry("a", ids[:1])], [StepEntry("a", ids[:2], [], [-1])]):
        with pytest.raises(ValueError):
            runner.step(wrong)
    runner.keep({"a": [0, 2, 5]})
    kept = prompt + [ids[i] for i in (0, 2, 5)]
    logits = runner.step([StepEntry("a", ids[:2], [0, 1])])
    near(logits, oracle(model[3], cfg, kept + ids[:2])[-2:], model[4])


def test_draw_tree():
    depth, words = draw_tree([-1, 0, 0, 2, -1] + list(range(4, 130)))
    assert depth[:5].tolist() == [0, 1, 1, 2, 0] and depth[-1] == 126
    assert words.shape == (131, 3)
    sees = lambda i: [j for j in range(131) if int(words[i, j // 64]) >> (j % 64) & 1]
    assert sees(3) == [0, 2, 3] and sees(1) == [0, 1] and sees(130) == list(range(4, 131))


def test_generation_over_a_cache_in_8_bits(model, ops, tmp_path):
    """The whole engine: scheduler, captured steps where there are any, preemption. Greedy tokens are those with the largest
    logits of the plain implementation over quantised keys and values, or as good as these."""
    cfg, block, folder, weights, dtype = model
    llm = LLM(folder, ops=ops, engine=EngineConfig(dtype="float32" if dtype == F32 else "bfloat16", cache_dtype="e4m3", block_size=block, num_blocks=40,
                                                   token_budget=24, max_seqs=4))
    prompts = [random_ids(cfg, n, n) for n in (30, 3, 11, 1)]
    for prompt, out in zip(prompts, llm.generate(prompts, SamplingParams(max_new_tokens=8, ignore_eos=True))):
        assert len(out.token_ids) == 8
        want = plain_logits(model, prompt + out.token_ids, True)[len(prompt) - 1:-1]
        for logits, token in zip(want, out.token_ids):
            # (a token may win by rounding: both its logit and the largest are within `near` of the engine's)
            assert float(logits[token]) >= float(logits.max()) - 2 * (4 if dtype == BF16 else 1) * float(logits.abs().max()) / 16


@pytest.mark.gpu
def test_layers_ended_in_one_launch_over_a_cache_in_8_bits(tmp_path):
    """Captured steps of few rows at a width that the one-launch layer end takes: it ends in the next layer's q/k/v rows."""
    from distie_amd.kernels.hip_ops import HipOps, LayerTail

    cfg = dict(plain.TINY_C, hidden_size=1024, num_attention_heads=16, num_key_value_heads=2, intermediate_size=64, num_hidden_layers=3,
               layer_types=["full_attention"] * 3)
    cfg.pop("head_dim", None)
    folder, weights = make_model_dir(tmp_path / "wide", cfg, seed=5, dtype=BF16)
    ended, whole = [], LayerTail.finish_rows
    LayerTail.finish_rows = lambda self, *a: ended.append(1) or whole(self, *a)
    try:
        llm = LLM(folder, ops=HipOps("cuda:0"), engine=EngineConfig(dtype="bfloat16", cache_dtype="e4m3", block_size=16, num_blocks=64, max_seqs=8))
        prompts = [random_ids(cfg, n, n) for n in (30, 3, 11)]
        outs = llm.generate(prompts, SamplingParams(max_new_tokens=12, ignore_eos=True))
    finally:
        LayerTail.finish_rows = whole
    assert ended
    model = cfg, 16, folder, weights, BF16
    for prompt, out in zip(prompts, outs):
        want = plain_logits(model, prompt + out.token_ids, True)[len(prompt) - 1:-1]
        for logits, token in zip(want, out.token_ids):
            # (as above)
            assert float(logits[token]) >= float(logits.max()) - 2 * 4 * float(logits.abs().max()) / 16


WIDE = dict(plain.TINY_C, hidden_size=1024, num_attention_heads=16, num_key_value_heads=2, intermediate_size=64, num_hidden_layers=3,
            layer_types=["full_attention"] * 3)
WIDE.pop("head_dim", None)
PROMPTS, DECODED = (30, 3, 11), 24


class WrongPowers(EightBitOps):
    """The double with a mistake: one kv head's powers of keys (or of values) one too large, or the fourth entry of every request lost."""

    def __init__(self, mistake):
        super().__init__()
        self.mistake = mistake

    def rope_kv_write_e4m3(self, qkv, meta, group, cache, *more):
        out = super().rope_kv_write_e4m3(qkv, meta, group, cache, *more)
        page, at = (f(meta.groups[group].slots.long(), cache.k.shape[2]) for f in (torch.div, torch.remainder))
        page = page.long()
        if self.mistake == "lost":
            here = meta.positions == 3
            for scale in (cache.k_scale, cache.v_scale):
                scale[page[here], :, at[here]] = 1
        else:
            (cache.k_scale if self.mistake == "keys" else cache.v_scale)[page, 0, at] += 1
        return out


def away(cfg, block, folder, weights, ops):
    """How far (root mean square) the engine's logits over a cache in 8 bits are from the plain ones over codes: prompts, then single tokens
    together, in captured steps where there are any."""
    llm = LLM(folder, ops=ops, engine=EngineConfig(dtype="bfloat16", cache_dtype="e4m3", block_size=block, num_blocks=96, max_seqs=4, token_budget=64))
    ids = [random_ids(cfg, n + DECODED, n) for n in PROMPTS]
    got = [[llm.step([StepEntry(b, ids[b][:n], list(range(n)))]).float().cpu()] for b, n in enumerate(PROMPTS)]
    for i in range(DECODED):
        step = llm.step([StepEntry(b, [ids[b][n + i]], [0]) for b, n in enumerate(PROMPTS)]).float().cpu()
        for b in range(len(PROMPTS)):
            got[b].append(step[b:b + 1])
    with quantised_keys_and_values():
        off = torch.cat([torch.cat(rows) - oracle(weights, cfg, i) for rows, i in zip(got, ids)])
    return float(off.pow(2).mean().sqrt())


@pytest.mark.parametrize("cfg, block, caught", [(plain.TINY_A, 4, True), (plain.TINY_B, 8, True), (plain.TINY_C, 16, True), (WIDE, 16, False)],
                         ids=["A", "B", "C", "wide"])
def test_bfloat16_over_8_bits_is_off_by_what_its_roundings_move(ops, tmp_path, cfg, block, caught):
    """The same model with the same roundings on the CPU says how far that is. Another order of sums rounds other values, and of
    a rounding that falls the other way all behind it is another sample of the same error: twice the CPU's distance holds it, over thousands
    of logits in the root mean square. Wrong powers and a lost entry do not pass."""
    folder, weights = make_model_dir(tmp_path, cfg, seed=31, dtype=BF16)
    limit = 2 * away(cfg, block, folder, weights, EightBitOps())
    assert away(cfg, block, folder, weights, ops) <= limit
    if caught and ops.device.type == "cpu":
        for mistake in ("keys", "values", "lost"):
            assert away(cfg, block, folder, weights, WrongPowers(mistake)) > limit, mistake


def test_models_that_keep_more_than_pages_take_no_trees_and_no_8_bits(tmp_path, ops):
    import musutar_util

    config = musutar_util.make_config([musutar_util.attention_layer(), musutar_util.lightning_layer()])
    from distie_amd.config import config_from_dict

    model = Model(config_from_dict(config).model_spec())
    assert not model.takes_trees
    model.use_cache_dtype(None)
    with pytest.raises(ValueError, match="keeps no cache in e4m3"):
        model.use_cache_dtype("e4m3")
    with pytest.raises(ValueError, match="cache_dtype"):
        EngineConfig(cache_dtype="fp8")
