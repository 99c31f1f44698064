"""Models whose attention keeps keys and values in 8 bits, where runs, steps and recordings meet: a run that reads another's cache, tables made
on the device, recordings whose replays cut and join long contexts, projections that come in shares.  Bounds are those of
test_gpu_cache8_model.py; where both sides run the same kernels on the same bytes the results are the same bits."""
from __future__ import annotations

import pytest
import torch

from conftest import TINY, TINY_A, TINY_B, require_gpu, token_ids
from plain import qwen3_plain
from test_gpu_cache8_model import close, rounded, runner_of
from test_gpu_model import mixed_trace, run_alone, run_mixed

pytestmark = pytest.mark.gpu


def runner_on(spec, source, dtype, page=16, pages=16, **options):
    from pulse_infer_amd.engine.runner import ModelRunner
    from pulse_infer_amd.models.causal_lm import CausalLM

    return ModelRunner(CausalLM(spec, source, mode=dtype, options=dict(cache_dtype="float8_e4m3", **options)), page_size=page, num_pages=pages,
                       max_requests=4)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("head_dim,page", [(16, 16), (32, 16), (32, 8)])
def test_a_run_that_reads_another_runs_cache(tmp_path, monkeypatch, head_dim, page, dtype):
    """Run order [0, 1, 0, 2 reading run 1's cache] against the plain parts: the last run prepares queries alone."""
    require_gpu()
    from pulse_infer_amd.config import Qwen3Config
    from pulse_infer_amd.models.spec import RunSpec
    from pulse_infer_amd.weights import SafetensorsSource, write_model_folder

    P, T = qwen3_plain, 60
    exact = P.causal_attention
    monkeypatch.setattr(P, "causal_attention", lambda q, k, v, *a: exact(q, rounded(k, page), rounded(v, page), *a))
    cfg = Qwen3Config.from_dict(dict(TINY_A, num_hidden_layers=3, head_dim=head_dim))
    folder = write_model_folder(cfg, str(tmp_path / "m"), seed=31)
    spec = cfg.model_spec()
    spec.order = [RunSpec(0), RunSpec(1), RunSpec(0), RunSpec(2, cache_of=1)]
    runner = runner_on(spec, SafetensorsSource(folder), dtype, page, 128 // page)
    assert len(runner.cache.groups[0].runs) == 3 and [v.writable for v in runner.views] == [True, True, True, False]
    ids = token_ids(cfg.vocab_size, T, seed=9)

    plain = P.PlainQwen3.from_folder(folder)
    c, w, pos = plain.c, plain.w, list(range(T))
    nq, nkv, d, eps = c["num_attention_heads"], c["num_key_value_heads"], c["head_dim"], c["rms_norm_eps"]
    h = plain.layer(P.embedding(w["model.embed_tokens.weight"], ids), 0, pos)
    p = "model.layers.1."
    a = P.rms_norm(h, w[p + "input_layernorm.weight"], eps)
    k1 = P.rope(P.rms_norm(P.linear(a, w[p + "self_attn.k_proj.weight"]).view(T, nkv, d), w[p + "self_attn.k_norm.weight"], eps), pos, c["rope_theta"])
    v1 = P.linear(a, w[p + "self_attn.v_proj.weight"]).view(T, nkv, d)
    h = plain.layer(plain.layer(h, 1, pos), 0, pos)
    p = "model.layers.2."
    a = P.rms_norm(h, w[p + "input_layernorm.weight"], eps)
    q = P.rope(P.rms_norm(P.linear(a, w[p + "self_attn.q_proj.weight"]).view(T, nq, d), w[p + "self_attn.q_norm.weight"], eps), pos, c["rope_theta"])
    h = h + P.linear(P.causal_attention(q, k1, v1, d ** -0.5).reshape(T, nq * d), w[p + "self_attn.o_proj.weight"])
    m = P.rms_norm(h, w[p + "post_attention_layernorm.weight"], eps)
    h = h + P.gated_mlp(m, w[p + "mlp.gate_proj.weight"], w[p + "mlp.up_proj.weight"], w[p + "mlp.down_proj.weight"])
    want = P.linear(P.rms_norm(h, w["model.norm.weight"], eps), w["model.embed_tokens.weight"])
    for cuts in ([T], [11, 1, 1, 17, 1, 29], [40] + [1] * 20):      # (the last: recorded steps among them)
        close(run_alone(runner, ids, cuts), want, dtype, f"shared cache, portions of {cuts}")


def test_tables_made_on_the_device_change_nothing(model_folders):
    """Steps of requests that come and go, with windows on some layers: the same bits whether host or device makes rows and tables."""
    require_gpu()
    from conftest import OVERRIDES

    for name, page in (("B", 16), ("W", 16), ("W", 8)):
        _, steps = mixed_trace(TINY[name][0]["vocab_size"], seed=9)
        got = []
        for maps_from in (10 ** 9, 1):
            runner = runner_of(model_folders[name], "bfloat16", page, overrides=OVERRIDES[name], use_graphs=False)
            runner.MAPS_FROM = maps_from
            got.append(run_mixed(runner, steps)[0])
        assert got[0].keys() == got[1].keys()
        for k in got[0]:
            assert torch.equal(got[0][k], got[1][k]), (name, page, k)


def test_replays_that_cut_and_join_are_the_eager_steps():
    """Contexts of more than a thousand tokens that cross from one recording's range into the next one's, beside a short one: every replay, request
    by request, gives the eager step's bits, and keys, values and scales are the eager run's."""
    require_gpu()
    from pulse_infer_amd.config import Qwen3Config
    from pulse_infer_amd.engine.runner import ModelRunner, StepEntry
    from pulse_infer_amd.models.causal_lm import expected_tensors
    from pulse_infer_amd.models.factory import build_model
    from pulse_infer_amd.weights.random_init import RandomSource

    cfg = Qwen3Config.from_dict(dict(TINY_B, max_position_embeddings=4096, hidden_size=128, num_key_value_heads=2, head_dim=64, vocab_size=300))
    lengths, steps = [1010, 1300, 2030, 40], 30
    ids = [token_ids(300, n + steps, seed=80 + i) for i, n in enumerate(lengths)]
    outs, runners = [], []
    for graphs in (True, False):
        model = build_model(cfg, RandomSource(expected_tensors(cfg.model_spec()), seed=5), mode="bfloat16", options={"cache_dtype": "float8_e4m3"})
        runner = ModelRunner(model, page_size=16, num_pages=300, max_requests=4, use_graphs=graphs)
        runner.GRAPH_AFTER_STEPS = 1
        for r, n in enumerate(lengths):
            runner.add_request(r)
            runner.reserve(r, n + steps)
            runner.step([StepEntry(r, ids[r][:n], [])])
        got = []
        for s in range(steps):
            got.append(runner.step([StepEntry(r, [ids[r][n + s]], [0]) for r, n in enumerate(lengths)]))
            torch.cuda.synchronize()
        assert (runner.graph_replays, runner.graph_records) == ((steps - 2, 2) if graphs else (0, 0))      # (2,031 to 2,048, 2,049 to 2,060)
        outs.append(got)
        runners.append(runner)
    for s, (a, b) in enumerate(zip(*outs)):
        for r in range(len(lengths)):
            assert torch.isfinite(a[r]).all() and torch.equal(a[r], b[r]), (s, r)
    for a, b in zip(*(r.cache.groups[0].storage for r in runners)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_projections_in_shares(monkeypatch):
    """Rows of which the store takes the projection's float32 shares, against rows that the product has added up and rounded."""
    require_gpu()
    from pulse_infer_amd.config import Qwen3Config
    from pulse_infer_amd.engine.runner import ModelRunner, StepEntry
    from pulse_infer_amd.models.causal_lm import expected_tensors
    from pulse_infer_amd.models.factory import build_model
    from pulse_infer_amd.ops import cache8
    from pulse_infer_amd.parts.linear import Linear
    from pulse_infer_amd.weights.random_init import RandomSource

    cfg = Qwen3Config.from_dict(dict(TINY_B, hidden_size=4096, intermediate_size=512, num_hidden_layers=2, num_attention_heads=32,
                                     num_key_value_heads=8, head_dim=128, vocab_size=300, max_position_embeddings=512))
    model = build_model(cfg, RandomSource(expected_tensors(cfg.model_spec()), seed=5), mode="bfloat16", options={"cache_dtype": "float8_e4m3"})
    took, store = [], cache8.store
    monkeypatch.setattr(cache8, "store", lambda *a, **k: took.append((a[0].shape[0], k.get("parts") is not None)) or store(*a, **k))
    may_part = Linear.may_part
    outs = []
    for shares in (True, False):
        monkeypatch.setattr(Linear, "may_part", may_part if shares else lambda self, rows: False)
        runner = ModelRunner(model, page_size=16, num_pages=64, max_requests=4, use_graphs=False)
        fed, got = {}, []
        took.clear()
        for plan in ([("a", 70)], [("a", 1), ("b", 100)], [("a", 30), ("b", 1), ("c", 150)], [("a", 1), ("b", 1), ("c", 1)]):
            entries = []
            for name, n in plan:
                if name not in fed:
                    runner.add_request(name)
                at = fed.get(name, 0)
                fed[name] = at + n
                runner.reserve(name, at + n)
                entries.append(StepEntry(name, token_ids(300, 400, seed=ord(name))[at:at + n], list(range(n))))
            got.append(runner.step(entries))
        assert took == [(n, shares and n > 3) for n in (70, 70, 101, 101, 181, 181, 3, 3)]
        outs.append(got)
    for i, (a, b) in enumerate(zip(*outs)):
        close(a, b, "bfloat16", f"step {i}")


def test_who_reads_a_cache_must_take_it_as_it_is():
    """A run that would read a cache in 8 bits as if it were not, and the other way round; a model none of whose runs has one."""
    require_gpu()
    from types import SimpleNamespace

    from pulse_infer_amd.cache import Paged8KVSpec, PagedKVSpec, StateSpec
    from pulse_infer_amd.models.causal_lm import CausalLM
    from pulse_infer_amd.models.spec import RunSpec

    def specs_of(order, *specs):
        model = CausalLM.__new__(CausalLM)
        model.options = {"cache_dtype": "float8_e4m3"}
        model.spec = SimpleNamespace(order=order, architecture="toy")
        model.blocks = [SimpleNamespace(cache_spec=lambda s=s: s) for s in specs]
        return model.run_cache_specs()

    eight, plain, state = Paged8KVSpec(2, 32), PagedKVSpec(2, 32), StateSpec((4,))
    order = [RunSpec(0), RunSpec(1), RunSpec(2, cache_of=0)]
    assert specs_of(order, eight, state, eight) == [eight, state, None]
    assert specs_of(order, plain, eight, plain) == [plain, eight, None]
    for wrong in ((eight, state, plain), (plain, eight, eight)):
        with pytest.raises(ValueError, match="only one of the two"):
            specs_of(order, *wrong)
    with pytest.raises(ValueError, match="no layer"):
        specs_of(order, plain, state, plain)
