"""Greedy generation with the paged 8-bit cache under a window with sinks,
against a forward in f64 whose attention has the same mask: the prompt's own
window (over its rows) and the decode steps' (over the cache) have to meet.

Teacher-forced as in test_gpu_generate_kv8.py, with its tolerances. The f64
forward is itself checked, without a window, against the oracle's. Greedy runs
of it under a window or a sink count that is one off fail the check at 5 to 21
of 36 tokens of the cases "narrow" and "qknorm_hd32".
"""
import numpy as np
import pytest

import ditch_b200
import test_gpu_generate as base
from oracle.model import OracleModel, flatten_batch
from synth import make_model, prompts

CASES = {
    # prompts shorter than the window, as long and longer; the decode steps move it over the prompt's end
    "hd64_bias": (dict(n_layers=3, hidden=256, heads=4, kv_heads=2, head_dim=64, inter=512, qkv_bias=True), [40, 1, 17, 64, 100], 24, 3),
    "qknorm_hd32": (dict(n_layers=2, hidden=256, heads=8, kv_heads=2, head_dim=32, inter=384, qk_norm=True), [33, 2, 90], 16, 0),
    "hd128_gqa8": (dict(n_layers=2, hidden=512, heads=8, kv_heads=1, head_dim=128, inter=512), [70, 130, 5], 33, 17),
    "narrow": (dict(n_layers=2, hidden=448, heads=7, kv_heads=1, head_dim=64, inter=384), [16, 15, 65], 5, 1),
}


class WindowedModel:
    """The dense decoder in f64 with a windowed causal mask, one sequence at a time."""

    def __init__(self, spec, weights, window=0, sinks=0):
        self.s, self.w, self.window, self.sinks = spec, {k: np.asarray(v, np.float64) for k, v in weights.items()}, window, sinks

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.s["eps"]) * w

    def forward(self, tokens, row_b, row_pos, capture_rows=(), logit_rows=()):
        s, w, n = self.s, self.w, len(tokens)
        hd, heads, kvh = s["head_dim"], s["heads"], s["kv_heads"]
        pos = np.asarray(row_pos, np.float64)
        assert not np.any(row_b) and np.array_equal(pos, np.arange(n))
        ang = pos[:, None] / s["rope_theta"] ** (np.arange(hd // 2) * 2.0 / hd)
        cos, sin = np.cos(ang)[:, None], np.sin(ang)[:, None]
        i, j = np.arange(n)[:, None], np.arange(n)[None]
        ok = j <= i
        if self.window:
            ok &= (j > i - self.window) | (j < self.sinks)

        def rope(x):
            a, b = x[..., :hd // 2], x[..., hd // 2:]
            return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)

        x = w["embed"][np.asarray(tokens, np.int64)]
        for l in range(s["n_layers"]):
            p = lambda name: w.get(f"L{l}.{name}")  # noqa: E731
            h = self.norm(x, p("input_norm"))
            q, k, v = ((h @ p(m).T + (p(b) if p(b) is not None else 0.0)).reshape(n, c, hd)
                       for m, b, c in (("q", "qb", heads), ("k", "kb", kvh), ("v", "vb", kvh)))
            if s.get("qk_norm"):
                q, k = self.norm(q, p("q_norm")), self.norm(k, p("k_norm"))
            q, k = rope(q), rope(k)
            out = np.empty_like(q)
            for a in range(heads):
                b = a // (heads // kvh)
                z = np.where(ok, q[:, a] @ k[:, b].T / np.sqrt(hd), -np.inf)
                z = np.exp(z - z.max(-1, keepdims=True))
                out[:, a] = z / z.sum(-1, keepdims=True) @ v[:, b]
            x = x + out.reshape(n, heads * hd) @ p("o").T
            h = self.norm(x, p("post_norm"))
            gate = h @ p("gate").T
            x = x + (gate / (1 + np.exp(-gate)) * (h @ p("up").T)) @ p("down").T
        return None, self.norm(x, w["final_norm"])[np.asarray(logit_rows, np.int64)] @ w["lm_head"].T


@pytest.mark.parametrize("name", sorted(CASES))
def test_the_f64_forward_is_the_oracles(name):
    kw, lens, _, _ = CASES[name]
    spec, f32, _ = make_model(970, **kw)
    for p in prompts(971, lens, spec["vocab"]):
        toks, rb, rp, _, _, _, _ = flatten_batch([p], 10 ** 6)
        rows = np.arange(len(p), dtype=np.uintp)
        want = OracleModel(spec, f32).forward(toks, rb, rp, logit_rows=rows)[1]
        for window in (0, 1000):
            got = WindowedModel(spec, f32, window, 4 if window else 0).forward(toks, rb, rp, logit_rows=rows)[1]
            assert np.abs(got - want).max() <= 1e-4 * np.abs(want).max()  # f32 sums of a few hundred terms, a few layers


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("name", sorted(CASES))
def test_windowed_generation(device, name, fmt, monkeypatch):
    kw, lens, window, sinks = CASES[name]
    spec, f32, tensors = make_model(980 + sorted(CASES).index(name), **kw)
    ps = prompts(990, lens, spec["vocab"])
    m = ditch_b200.Model(device, spec, tensors, max_seq=256)
    m.set_kv_cache(fmt, window=window, sinks=sinks)
    got = m.generate(ps, 48)
    m.close()
    monkeypatch.setattr(base, "FWD_RTOL", 4e-2 if fmt == "int8" else 8e-2)
    n, exact = base.check_generation(WindowedModel(spec, f32, window, sinks), ps, got, 48)
    assert n == 48 * len(ps)
    print(f"{name} {fmt}: {exact} of {n} tokens with a clear maximum")


@pytest.mark.gpu
def test_more_prompts_than_one_windowed_prefill_takes(device, request):
    """65,600 prompts, of which many are alike: those past one launch's 65,535
    sequences get the tokens of their likes before it."""
    spec, f32, tensors = make_model(995, n_layers=1, hidden=64, heads=1, kv_heads=1, head_dim=32, inter=64)
    m = ditch_b200.Model(device, spec, tensors, max_seq=16)
    device.set_deterministic(True)
    request.addfinalizer(lambda: device.set_deterministic(False))
    m.set_kv_cache("int8")
    ps = [np.array([i % 64, 7], np.uint32) for i in range(65600)]
    got = m.generate(ps, 3)
    m.close()
    assert len(got) == len(ps) and all(len(g) == 3 for g in got)
    assert all(got[i] == got[i % 64] for i in range(len(ps)))
    base.check_generation(OracleModel(spec, f32), ps[-8:], got[-8:], 3)
