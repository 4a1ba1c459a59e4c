"""Models whose matrices are held in 4 bits, through replayer and engine, against the plain decoder with the same roundings."""
import functools
import json
import subprocess
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT, TINY
from helpers import Reference, assert_close, bulk_and_tail, collect, mixed, plain_model, portions, random_ids, whole
from plain import microscaled as px
from plain import model as pm

pytestmark = pytest.mark.gpu
LENGTHS = {"A": 100, "B": 150, "C": 190, "D": 300, "E": 60}


@functools.lru_cache(maxsize=None)
def _weights(model_dir):
    cfg, w = plain_model(model_dir)
    return cfg, px.matrices_rounded(w, cfg)


@functools.lru_cache(maxsize=64)
def _logits(model_dir, ids, rounded):
    cfg, w = _weights(model_dir)
    return px.forward_logits(w, cfg, list(ids), store=pm.to_bfloat16 if rounded else (lambda x: x))


def reference(model_dir, ids):
    ref = _logits(str(model_dir), tuple(ids), False).view(Reference)
    ref._rounded = lambda: _logits(str(model_dir), tuple(ids), True)
    return ref


def ids_of(name, seed=11, n=None):
    return random_ids(seed, n or LENGTHS[name], TINY[name]["vocab_size"])


@pytest.fixture(scope="module")
def replayers(tiny_dirs):
    from alofa_amd.replay import Replayer
    made = {}

    def get(name):
        if name not in made:
            made[name] = Replayer(tiny_dirs[name], "bfloat16", 512, matrices="mxfp4")
        assert not made[name].cache.requests, "a test left requests behind"
        return made[name]
    return get


@pytest.mark.parametrize("name", sorted(LENGTHS))
def test_whole_prompts(replayers, tiny_dirs, name):
    ids = ids_of(name)
    assert_close(collect(replayers(name), whole("w", ids))["w"], reference(tiny_dirs[name], ids), "bfloat16", f"{name} whole")


@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_bulk_then_one_by_one(replayers, tiny_dirs, name):
    ids = ids_of(name)
    r = replayers(name)
    got = collect(r, bulk_and_tail("t", ids))["t"]
    assert_close(got, reference(tiny_dirs[name], ids), "bfloat16", f"{name} bulk+tail")
    assert r.fn.graph_replays > 0      # (decode steps are captured and replayed)


@pytest.mark.parametrize("name", ["B", "C"])
def test_portions(replayers, tiny_dirs, name):
    ids = ids_of(name)
    assert_close(collect(replayers(name), portions("p", ids))["p"], reference(tiny_dirs[name], ids), "bfloat16", f"{name} portions")


@pytest.mark.parametrize("name", ["A", "C"])
def test_mixed_requests(tiny_dirs, name):
    from alofa_amd.replay import Replayer
    vocab, top = TINY[name]["vocab_size"], LENGTHS[name]
    requests = {f"r{i}": random_ids(100 + i, n, vocab) for i, n in enumerate([top, 41, top - 37, 64, 35])}
    steps, peak = mixed(requests, seed=5)
    got = collect(Replayer(tiny_dirs[name], "bfloat16", peak, matrices="mxfp4"), steps)
    for k, ids in requests.items():
        assert_close(got[k], reference(tiny_dirs[name], ids), "bfloat16", f"{name} mixed {k}")


def test_generation_and_memory(tiny_dirs):
    from alofa_amd import Engine
    cfg, w = _weights(str(tiny_dirs["D"]))
    prompts = [random_ids(s, n, cfg["V"]) for s, n in ((1, 5), (2, 17), (3, 40))]
    eng = Engine(tiny_dirs["D"], max_tokens=128, matrices="mxfp4")
    got = eng.generate(prompts, max_new=12)
    assert got == Engine(tiny_dirs["D"], max_tokens=128, matrices="mxfp4").generate(prompts, max_new=12)
    # every token is the plain decoder's choice on what came before it, or within what rounding activations to bfloat16 moves a logit
    for p, out in zip(prompts, got):
        ids = p + out
        ref = reference(tiny_dirs["D"], ids[:-1])
        room = 2.0 * np.abs(np.asarray(ref.rounded()) - np.asarray(ref)).max()
        for i, t in enumerate(out):
            row = np.asarray(ref)[len(p) - 1 + i]
            assert row.max() - row[t] <= 2 * room
    # the matrices take 4.25 bits a number (filled up to tiles of 16 x 128), where bfloat16 takes 16
    from alofa_amd.ops import MXRows
    h, i, kv = cfg["h"], cfg["I"], cfg["Hkv"] * cfg["d"]
    shapes = [(cfg["H"] * cfg["d"] + 2 * kv, h), (h, cfg["H"] * cfg["d"]), (i, h), (i, h), (h, i)]
    stored = Engine(tiny_dirs["D"], max_tokens=128)
    saved = cfg["L"] * sum(2 * n * k - MXRows.bytes(n, k, "e2m1") for n, k in shapes)
    assert stored.memory()["weights"] - eng.memory()["weights"] == saved


def test_matrices_that_are_in_the_format_already_stay_as_they_are(tiny_dirs, tmp_path):
    from safetensors.torch import save_file
    from alofa_amd.replay import Replayer
    cfg, w = _weights(str(tiny_dirs["A"]))
    (tmp_path / "config.json").write_text((tiny_dirs["A"] / "config.json").read_text())
    save_file({n: torch.from_numpy(np.ascontiguousarray(t)).bfloat16() for n, t in w.items()}, str(tmp_path / "model.safetensors"))
    ids = ids_of("A")
    a, b = (collect(Replayer(d, "bfloat16", 256, matrices="mxfp4"), whole("w", ids))["w"] for d in (tiny_dirs["A"], tmp_path))
    assert np.array_equal(a, b)


def test_programs(tiny_dirs, tmp_path):
    import os
    env = {**os.environ, "ALOFA_WEIGHTS": str(tiny_dirs["A"]), "ALOFA_PROMPT_IDS": "5,17,3;9,2", "ALOFA_MAX_NEW": "6", "ALOFA_MAX_TOKENS": "64", "ALOFA_MAX_PROMPT_TOKENS": "32", "ALOFA_MATRICES": "mxfp4"}
    r = subprocess.run([sys.executable, str(ROOT / "bin" / "generate")], env=env, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr
    from alofa_amd import Engine
    want = Engine(tiny_dirs["A"], max_tokens=64, seed=1234, matrices="mxfp4").generate([[5, 17, 3], [9, 2]], max_new=6)
    assert [[int(t) for t in line.split(",")] for line in r.stdout.split()] == want
    step = json.dumps({"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3], "want": [2]}], "end": ["a"]})
    r = subprocess.run([sys.executable, str(ROOT / "bin" / "trace_run"), "--model", str(tiny_dirs["A"]), "--dtype", "bfloat16", "--out", str(tmp_path), "--max-tokens", "64", "--matrices", "mxfp4"],
                       input=step + "\n", capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr
    assert int(np.fromfile(tmp_path / "0.f32", dtype=np.float32).argmax()) == want[0][0]


def test_shares_of_the_product_down_go_to_the_next_layers_norm(tmp_path):
    """A feed-forward so wide that its sum is shared out over K: the next layer's first norm adds the shares to the stream."""
    from alofa_amd import ops
    from alofa_amd.replay import Replayer
    from alofa_amd.weights import write_random_model
    cfg = dict(TINY["A"], num_hidden_layers=3, intermediate_size=8192)
    write_random_model(cfg, tmp_path, seed=77)
    ids = random_ids(5, 90, cfg["vocab_size"])
    replayer = Replayer(tmp_path, "bfloat16", 256, matrices="mxfp4")
    assert all(ops.mx_shares(n, cfg["hidden_size"], 8192) > 1 for n in (1, 17, 40, 90))
    ref = reference(tmp_path, ids)
    assert_close(collect(replayer, whole("w", ids))["w"], ref, "bfloat16", "whole")
    assert_close(collect(replayer, portions("p", ids, (40, 17, 23, 10)))["p"], ref, "bfloat16", "portions")
    assert_close(collect(replayer, bulk_and_tail("b", ids, 84))["b"], ref, "bfloat16", "bulk then one by one")


@pytest.mark.parametrize("T", [1, 23, 90])
def test_a_layer_whose_output_product_has_a_bias(T):
    """Layers of any registered design may have one. With a feed-forward that adds nothing the layer with it is the layer without it and the bias; and its second half reads that sum."""
    from alofa_amd import ops
    from alofa_amd.cache import CacheManager
    from alofa_amd.config import LayerSpec, ModelSpec, PartSpec, RunEntry
    from alofa_amd.engine import StepEntry, StepFunction
    from alofa_amd.model import Model, expected_tensors, runtime
    from alofa_amd.parts.microscaled import microscaled
    from alofa_amd.weights import random_tensors
    h, H, kv, d, inter, V = 160, 4, 2, 32, 352, 50
    rng = np.random.default_rng(T)
    stream = rng.standard_normal((T, h)).astype(np.float32)

    def run(bias, weights):
        layer = LayerSpec("l.", PartSpec("prenorm"), dict(
            mixer=PartSpec("gqa_attention", {"prefix": "l.att.", "hidden": h, "heads": H, "kv_heads": kv, "head_dim": d, "qkv_bias": True, "out_bias": bias, "window": None,
                                             "position": PartSpec("none", {"head_dim": d})}),
            feed_forward=PartSpec("swiglu", {"prefix": "l.ff.", "hidden": h, "intermediate": inter}),
            norms=(PartSpec("rmsnorm", {"name": "l.n0", "width": h, "eps": 1e-6}), PartSpec("rmsnorm", {"name": "l.n1", "width": h, "eps": 1e-6}))))
        spec = microscaled(ModelSpec(h, V, 128, PartSpec("token_embedding", {"name": "emb", "vocab": V, "width": h}), (layer,), (RunEntry(0),),
                                     PartSpec("rmsnorm", {"name": "nf", "width": h, "eps": 1e-6}), PartSpec("lm_head", {"name": "head", "tied_to": "emb", "vocab": V, "width": h})))
        expected = expected_tensors(spec)
        weights = weights or random_tensors(expected, 6, std=0.3, store_dtype="float32")
        model = Model(spec, {n: weights[n] for n in expected if n in weights}, runtime("bfloat16"))
        fn = StepFunction(model, CacheManager(model.cache_needs(), model.state_needs(), 8, 16, 2, device=model.rt.device, dtype=torch.bfloat16), 128)
        fn.cache.admit(0)
        ctx, _, _ = fn.begin([StepEntry(0, [1] * T, [])])
        out = torch.from_numpy(stream).cuda()
        model.blocks[0].forward(ctx, 0, out)
        return out.cpu().numpy(), weights
    got, weights = run(True, None)
    assert weights["l.att.o_proj.bias"].abs().max() > 0.1
    idle = dict(weights, **{"l.ff.down_proj.weight": torch.zeros(h, inter)})
    without, mixed_in = run(False, idle)[0], run(True, idle)[0]
    bias = weights["l.att.o_proj.bias"].numpy()
    # (one sum is rounded twice on the way, the other three times, half a unit of what is there each; the products themselves are the same up to the order of a sum of 128 numbers in shares of one)
    assert np.abs(mixed_in - (without + bias)).max() <= 8 * 2.0 ** -24 * (np.abs(without) + np.abs(bias) + np.abs(mixed_in) + np.abs(stream)).max()
    f64 = {n: t.double().numpy() for n, t in weights.items()}
    t = mixed_in.astype(np.float64)
    n = px.rounded(px.norm(t, f64["l.n1"], 1e-6), "e4m3")
    gate, up, down = (px.rounded(f64[f"l.ff.{m}_proj.weight"], "e2m1") for m in ("gate", "up", "down"))
    want = t + px.rounded(px.silu(n @ gate.T) * (n @ up.T), "e4m3") @ down.T
    # (an element here and there goes to its neighbour by a last bit: were a part in 256 of them all a whole step off)
    assert np.linalg.norm(got - want) / np.linalg.norm(want) <= 2.0 ** -24 + 2.0 ** -8
