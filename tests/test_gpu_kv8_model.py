"""A Galirax model served over the paged 8-bit cache: against its float64 reference with the cache of tests/kv8_ref.py in the attention's place, step by step as the engine
fed the tokens (what a page holds depends on the steps).

Tolerances: got and the reference quantise values that differ in the last bits of f32 (2^-20 of themselves after a projection, a norm and a rotation).  A value flips
to the neighbouring step with a probability of 2 127 2^-20 = 2.4e-4, by one step, where all values are off by 1 / sqrt(12) of a step anyway: sqrt(12 2.4e-4) = 5 % of what the
8 bits themselves do to the logits.  So with ONE attention layer the logits differ from the reference's by a quarter of that at most (and 1e-4 as over f32 caches).  Behind
a second attention layer the keys differ by a share of the quantisation itself, flips are no longer rare, and two independent quantisations are what is compared: sqrt(2) of
one's effect, 2 as a bound."""
from __future__ import annotations

import json

import numpy as np
import pytest

import galirax_ref as R
import kv8_ref as K
from koboldcpp_b200 import galirax as G
from koboldcpp_b200.engine import Engine, Request
from koboldcpp_b200.lib import B200Error

pytestmark = pytest.mark.gpu

ONE = lambda **kw: R.make_config([R.lightning_layer(heads=2, dim=16, vdim=32, mlp=None), R.attn_layer(heads=4, kv_heads=2, dim=32, vdim=48, rot_dims=16, mlp=None, **kw)], width=64, vocab=70)  # noqa: E731
CONFIGS = {
    "plain": (ONE(), 0.25),
    "window": (ONE(kind="attention_2", window=20, keep_first=3), 0.25),
    "wide heads": (R.make_config([R.attn_layer(heads=3, kv_heads=1, dim=128, vdim=128, rot_dims=64, mlp=None)], width=64, vocab=50, softcap=0.0), 0.25),
    "looped": (R.make_config([R.attn_layer(heads=4, kv_heads=4, dim=32, vdim=32, rot_dims=32, mlp=None), R.attn_layer("attention_2", heads=4, kv_heads=1, dim=64, vdim=32, window=30, mlp=None)],
                             width=128, vocab=96, loop=(1, 2, 2)), 2.0),
}


def forward8(monkeypatch, cfg, W, tokens, steps, page):
    """The reference's logits with keys and values stored in 8 bits, `steps` tokens at a time."""
    def attention(q, k, v, scale, sink, window=0, keep_first=0):
        T, H, _ = q.shape
        pool = K.Pool(-(-T // page), page, k.shape[1], k.shape[2], v.shape[2])
        entries, out, at = list(range(pool.n_pages)), [], 0
        for n in steps:
            pool.store(entries, k[at:at + n], v[at:at + n], at)
            out.append(pool.attend(entries, q[at:at + n], at, scale, window, keep_first, np.asarray(sink, np.float64))[0])
            at += n
        assert at == T
        return np.concatenate(out)
    with monkeypatch.context() as m:
        m.setattr(R, "sink_attention", attention)
        return R.forward(cfg, W, tokens)


def logits_err(got, want):
    d = got - want
    d = d - d.mean(-1, keepdims=True)
    return float((np.sqrt((d ** 2).mean(-1)) / want.std()).max())


def near(got, want8, want, factor):
    own = logits_err(want8, want)
    assert 1e-5 < own < 0.2  # the 8 bits do something, and not much
    assert logits_err(got, want8) <= factor * own + 1e-4


@pytest.mark.parametrize("name", CONFIGS)
@pytest.mark.parametrize("page", [16, 64])
def test_prompt_portions_and_decoding(monkeypatch, name, page):
    cfg, factor = CONFIGS[name]
    W = R.random_weights(cfg, seed=len(name))
    m = G.build(cfg, R.as_tensors(W), dtype="float32", n_ctx=512, n_seq_max=3, max_batch=200, kv8_page=page)
    toks = np.random.default_rng(1).integers(0, cfg["vocab"], 110).tolist()
    for steps in ([110], [70] + [1] * 40, [5, 40, 17, 1, 1, 30, 16]):
        eng, rows, at = Engine(m), [], 0
        for n in steps:
            rows.append(eng.step([("a", toks[at:at + n], range(n))]))
            at += n
        eng.finish("a")
        want, want8 = R.forward(cfg, W, toks[:at]), forward8(monkeypatch, cfg, W, toks[:at], steps, page)
        near(np.concatenate(rows), want8, want, factor)
    stats = m.stats()
    m.close()
    plain = G.build(cfg, R.as_tensors(W), dtype="float32", n_ctx=512, n_seq_max=3, max_batch=200)
    attn = [layer["mixer"] for layer in (cfg["layers"][i] for i in R.run_order(cfg)) if layer["type"] != "lightning"]
    tokens = 512 // page * page + 3 * page
    saved = sum(4 * 512 * x["kv_heads"] * (x["dim"] + x["vdim"]) for x in attn) - sum(K.Pool(1, page, x["kv_heads"], x["dim"], x["vdim"]).bytes * (tokens // page) for x in attn)
    assert plain.stats()["kv_bytes"] - stats["kv_bytes"] == saved and saved > 0
    plain.close()


def test_sequences_together_and_pages_that_are_used_again(monkeypatch):
    """Prompts beside decoding sequences; one ends, another takes its pages; as many tokens as there are cells always have room."""
    cfg, factor = CONFIGS["plain"]
    W = R.random_weights(cfg, seed=7)
    m = G.build(cfg, R.as_tensors(W), dtype="float32", n_ctx=256, n_seq_max=4, max_batch=256, kv8_page=32)
    rng = np.random.default_rng(2)
    eng = Engine(m)
    for _ in range(3):
        lens = {"a": 33, "b": 100, "c": 1, "d": 122 - 4}
        toks = {k: rng.integers(0, cfg["vocab"], n + 1).tolist() for k, n in lens.items()}
        first = eng.step([(k, toks[k][:n], [n - 1]) for k, n in lens.items()])
        second = eng.step([(k, toks[k][n:], [0]) for k, n in lens.items()])  # 256 cells: full
        with pytest.raises(B200Error, match="full"):
            eng.step([("a", [1], [0])])
        for i, (k, n) in enumerate(lens.items()):
            want, want8 = R.forward(cfg, W, toks[k]), forward8(monkeypatch, cfg, W, toks[k], [n, 1], 32)
            near(np.stack([first[i], second[i]]), want8[n - 1:], want[n - 1:], 2 * factor)  # (of two rows of logits the quantisation's effect is a rougher measure)
        eng.finish("b")
        more = rng.integers(0, cfg["vocab"], 90).tolist()
        got = eng.step([("e", more, range(90))])
        near(got, forward8(monkeypatch, cfg, W, more, [90], 32), R.forward(cfg, W, more), factor)
        for k in "acde":
            eng.finish(k)
    m.close()


def test_bfloat16_prompts(monkeypatch):
    """Served in bf16 a prompt's queries and weights are rounded to f16 as well; activations are rounded to bf16 in the projections, 2^-9 each: the logits agree with the
    float32 model's over the same cache to the bound of the bf16 tests (3 % of their deviation)."""
    cfg, _ = CONFIGS["plain"]
    W = R.random_weights(cfg, seed=3)
    toks = np.random.default_rng(5).integers(0, cfg["vocab"], 150).tolist()
    out = []
    for dtype in ("bfloat16", "float32"):
        m = G.build(cfg, R.as_tensors(W), dtype=dtype, n_ctx=256, n_seq_max=1, max_batch=150, kv8_page=16)
        eng = Engine(m)
        out.append(np.concatenate([eng.step([("x", toks[:120], range(120))])] + [eng.step([("x", [t], [0])]) for t in toks[120:]]))
        m.close()
    assert logits_err(out[0], out[1]) < 0.03


def test_generation_and_command_line(tmp_path, capsys):
    from test_gpu_galirax import write_model_folder
    from koboldcpp_b200 import __main__ as cli
    cfg, _ = CONFIGS["plain"]
    W = R.random_weights(cfg, seed=4)
    m = G.build(cfg, R.as_tensors(W), dtype="float32", n_ctx=256, n_seq_max=3, max_batch=64, kv8_page=16)
    prompts = [[5, 9, 2], [7] * 20, [1]]
    outs = Engine(m, max_step_tokens=12).generate([Request(p, 8) for p in prompts])
    m.close()
    for p, out in zip(prompts, outs):  # the reference's argmax over exact caches, or near it: the 8 bits move logits by less than a fifth of their deviation
        for i, tok in enumerate(out):
            lg = R.forward(cfg, W, p + out[:i])[-1]
            assert lg[tok] > lg.max() - 0.4 * lg.std()
    write_model_folder(tmp_path, cfg, W)
    assert cli.main(["generate", "--model", str(tmp_path), "--dtype", "float32", "--max-new-tokens", "8", "--kv8-page", "16", "--prompt", "5,9,2"]) == 0
    line = [json.loads(x) for x in capsys.readouterr().out.strip().splitlines() if x.startswith("{")][0]
    assert len(line["tokens"]) == 8


def test_refusals(tmp_path):
    cfg, _ = CONFIGS["plain"]
    W = R.as_tensors(R.random_weights(cfg, seed=4))
    with pytest.raises(B200Error, match="kv8_page 48"):
        G.build(cfg, W, n_ctx=256, n_seq_max=1, kv8_page=48)
    odd = R.make_config([R.attn_layer(heads=2, kv_heads=1, dim=24, vdim=24, mlp=None)], width=64, vocab=70)
    with pytest.raises(B200Error, match="multiples of 16"):
        G.build(odd, R.as_tensors(R.random_weights(odd, seed=1)), n_ctx=256, n_seq_max=1, kv8_page=16)
    with pytest.raises(B200Error, match="at most 1024"):
        G.build(cfg, W, n_ctx=256, n_seq_max=1025, kv8_page=16)
