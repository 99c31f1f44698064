"""Models whose attention keeps keys and values in 8 bits, against the plain implementation with the same rounding of its keys and values.

The plain side rounds a whole sequence at its blocks' final scales, the engine block by block as tokens come; the two differ where a
token's earlier bytes moved to a larger scale, by at most 2^-10 of a block's largest value a move, and where a key that float32 has
to 1e-6 lies at a border between two bytes (2^-4 of that one number).  Of a sum over a hundred rows and more neither moves a logit by
1e-2 of the largest.  In bfloat16 keys and values are themselves known to some 2^-8 only, a good part of the distance between two
bytes (2^-3 of a value at most, 2^-4 at least): two runs round many of them to different bytes, so their roundings are as good as independent.  A rounding
is off by 2^-5.3 = 0.0255 of a value by root mean square (half a step at most, uniform, over mantissas that are uniform in their
logarithm); keys of norm sqrt(d) move a score of such queries by that much and so the weights' sums, values move them once more; two
sides, two causes: 0.0255 * 2 = 0.051 of an update, and no more of the logits, in 2-norm: bound 2^-4."""
from __future__ import annotations

import pytest
import torch

from conftest import OVERRIDES, TINY, require_gpu, token_ids
from plain import cache8_plain, dirozen_plain, qwen3_plain
from test_gpu_model import LENGTH, mixed_trace, run_alone, run_mixed

pytestmark = pytest.mark.gpu


def close(got, want, dtype, what):
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape, what
    if dtype == "bfloat16":
        off, most = float((got - want).norm() / want.norm()), 2.0 ** -4
    else:
        off, most = float((got - want).abs().max()) / max(1.0, float(want.abs().max())), 1e-2
    assert off <= most, f"{what}: {off:.3e}"


def rounded(x, page):
    """Keys or values [T, heads, d] of a sequence as the cache stands for them."""
    t, heads, d = x.shape
    cache = cache8_plain.Cache(-(-t // page), heads, page, d)
    n = cache.block
    cache.store(x, x, [[i, min(n, t - i), i // n, 0] for i in range(0, t, n)])
    return cache.rows(list(range(cache.x[0].shape[0])))[0].transpose(0, 1)[:t]


def runner_of(folder, dtype, page, tokens=256, overrides=None, requests=4, **options):
    from pulse_infer_amd.engine.runner import ModelRunner
    from pulse_infer_amd.models.factory import load_model

    graphs = options.pop("use_graphs", True)
    _, model = load_model(folder, mode=dtype, config_overrides=overrides, options=dict(cache_dtype="float8_e4m3", **options))
    return ModelRunner(model, page_size=page, num_pages=tokens // page, max_requests=requests, use_graphs=graphs)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,page", [("A", 4), ("A", 16), ("B", 16), ("B", 64), ("W", 8), ("W", 16)])
def test_whole_tail_and_portions(model_folders, plain_models, monkeypatch, name, page, dtype):
    require_gpu()
    plain = qwen3_plain.causal_attention
    monkeypatch.setattr(qwen3_plain, "causal_attention", lambda q, k, v, *a: plain(q, rounded(k, page), rounded(v, page), *a))
    ids = token_ids(TINY[name][0]["vocab_size"], LENGTH[name], seed=3)
    want = plain_models[name].logits(ids)
    runner = runner_of(model_folders[name], dtype, page, overrides=OVERRIDES[name])
    assert all(v.keys.dtype == torch.float8_e4m3fn for v in runner.views)
    close(run_alone(runner, ids, [len(ids)]), want, dtype, "whole")
    close(run_alone(runner, ids, [len(ids) - 32] + [1] * 32), want, dtype, "last 32 one by one")
    close(run_alone(runner, ids, [7, 2, 16, 3, 33, 5] + [len(ids) - 66]), want, dtype, "portions")
    close(run_alone(runner, ids[:3], [1, 1, 1]), want[:3], dtype, "first tokens")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_mixed_batches_with_page_reuse(model_folders, plain_models, monkeypatch, dtype):
    """Portions beside single tokens, requests that come and go, pages used again: each request as if it were alone."""
    require_gpu()
    plain = qwen3_plain.causal_attention
    monkeypatch.setattr(qwen3_plain, "causal_attention", lambda q, k, v, *a: plain(q, rounded(k, 16), rounded(v, 16), *a))
    ids, steps = mixed_trace(TINY["B"][0]["vocab_size"], seed=9)
    got, _, _ = run_mixed(runner_of(model_folders["B"], dtype, 16), steps)
    for k, mine in got.items():
        close(mine, plain_models["B"].logits(ids[k]), dtype, f"request {k}")


def test_recorded_steps_and_the_kernel_for_every_size(model_folders):
    """Decoding steps recorded and replayed against eager ones, and against the kernel that serves every size."""
    require_gpu()
    from pulse_infer_amd.engine.runner import StepEntry

    lengths, steps = [70, 5, 33], 24
    ids = [token_ids(TINY["B"][0]["vocab_size"], n + steps, seed=60 + i) for i, n in enumerate(lengths)]
    out = []
    for options in ({}, {"use_graphs": False}, {"use_graphs": False, "attention": "generic"}):
        runner = runner_of(model_folders["B"], "bfloat16", 16, **options)
        runner.GRAPH_AFTER_STEPS = 1
        for r, n in enumerate(lengths):
            runner.add_request(r)
            runner.reserve(r, n + steps)
            runner.step([StepEntry(r, ids[r][:n], [])])
        out.append(torch.stack([runner.step([StepEntry(r, [ids[r][n + s]], [0]) for r, n in enumerate(lengths)]) for s in range(steps)]))
        assert (runner.graph_replays > steps // 2) == (not options)
    close(out[0], out[1], "bfloat16", "recorded against eager")
    close(out[2], out[1], "bfloat16", "the kernel for every size")


def test_dirozen(tmp_path, monkeypatch):
    """Layers with caches of their own, values that are the raw keys, norms without weights, query temperatures, gates."""
    require_gpu()
    from pulse_infer_amd.config import DirozenConfig
    from pulse_infer_amd.weights import write_model_folder

    from test_gpu_dirozen import MIXED

    folder = write_model_folder(DirozenConfig.from_dict(MIXED), str(tmp_path / "d"), seed=70)
    plain = dirozen_plain.PlainDirozen.from_folder(folder)
    ids = token_ids(MIXED["vocab"], 90, seed=5)
    exact = plain.logits(ids)
    for dtype in ("float32", "bfloat16"):
        runner = runner_of(folder, dtype, 16)
        whole = run_alone(runner, ids, [90])
        parts = run_alone(runner, ids, [40, 1, 1, 20, 1, 27])
        close(parts, whole, dtype, "portions against whole")
        # keys and values off by 2^-4 of themselves at most, 2^-5.5 by root mean square, move the logits by far less than that
        off = (whole.double().cpu() - exact).norm() / exact.norm()
        assert 1e-4 < off < 2.0 ** -4, off


def test_generation_half_the_memory_and_the_command(model_folders, tmp_path, capsys):
    require_gpu()
    from pulse_infer_amd import LLM, cli

    prompts = [token_ids(TINY["B"][0]["vocab_size"], n, seed=n) for n in (3, 40, 17)]
    llm = LLM.from_pretrained(model_folders["B"], cache_dtype="float8_e4m3", num_pages=12, page_size=16, chunk_size=16, max_batch_size=3)
    got = llm.generate(prompts, max_new_tokens=12, ignore_eos=True)
    assert [len(g) for g in got] == [12] * 3 and got == llm.generate(prompts, max_new_tokens=12, ignore_eos=True)
    sizes = [sum(t.numel() * t.element_size() for g in e.runner.cache.groups for t in g.spec.tensors(g.storage))
             for e in (llm.engine, LLM.from_pretrained(model_folders["B"], num_pages=12, page_size=16).engine)]
    assert sizes[0] < 0.52 * sizes[1]
    assert cli.main([model_folders["B"], "--cache-dtype", "float8_e4m3", "--prompt-len", "20", "--max-new-tokens", "4", "--ignore-eos"]) == 0
    assert '"output_ids"' in capsys.readouterr().out


def test_refusals(model_folders, tmp_path):
    require_gpu()
    from pulse_infer_amd import LLM
    from pulse_infer_amd.config import TipidraConfig
    from pulse_infer_amd.models.factory import load_model
    from pulse_infer_amd.weights import write_model_folder

    from test_gpu_tipidra import CONFIGS

    with pytest.raises(ValueError, match="unknown cache dtype"):
        load_model(model_folders["A"], options={"cache_dtype": "int8"})
    folder = write_model_folder(TipidraConfig.from_dict(next(iter(CONFIGS.values()))), str(tmp_path / "t"), seed=1)
    with pytest.raises(ValueError, match="in 8 bits"):
        LLM.from_pretrained(folder, cache_dtype="float8_e4m3")


@pytest.mark.parametrize("changed", [False, True])
def test_alike_layers_are_launched_from_one_record(monkeypatch, changed):
    """The bits of the same steps through the layers' parts; a layer that is not alike goes through its own."""
    require_gpu()
    from pulse_infer_amd.config import Qwen3Config
    from pulse_infer_amd.models.causal_lm import expected_tensors
    from pulse_infer_amd.models.factory import build_model
    from pulse_infer_amd.weights.random_init import RandomSource

    from test_gpu_alike_runs import FEW_ROWS, SIZES, counted

    cfg = Qwen3Config.from_dict(SIZES)
    model = build_model(cfg, RandomSource(expected_tensors(cfg.model_spec()), seed=3), mode="bfloat16",
                        options={"cache_dtype": "float8_e4m3"})
    if changed:
        model.blocks[6].mixer.scale *= 2.0
    recorded, few = counted(monkeypatch, model, True, FEW_ROWS)
    through, many = counted(monkeypatch, model, False, FEW_ROWS)
    assert few < (0.9 if changed else 0.6) * many
    for a, b in zip(recorded, through):
        assert torch.equal(a, b)
