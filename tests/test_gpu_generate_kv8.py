"""Greedy generation with the paged 8-bit cache (ditch_cuda_model_set_kv_cache):
append, windowed prefill attention and attention over the cache together.

Teacher-forced against the oracle as in test_gpu_generate.py: the device's
token must be the oracle's first maximum, or a logit within a tolerance of it
where the two best are closer than that. The tolerance is the forward bound
(2e-3 + 2e-2 max|row|) plus what 8-bit keys and values add: a block's scale is
its largest magnitude, about 3.5 standard deviations, so an int8 code is off by
at most 1/254 and 1/440 rms of that, under 1 % of a standard deviation, which
moves scores and values alike by under 1 % of their spread: 2e-2 max|row| more.
An E4M3 code is off by at most 2^-4 and 2.6 % rms: three times as much.
"""
import numpy as np
import pytest

import ditch_b200
import test_gpu_generate as base
from oracle.model import OracleModel
from synth import make_model, prompts

pytestmark = pytest.mark.gpu

CASES = {
    "hd64_bias": (dict(n_layers=3, hidden=256, heads=4, kv_heads=2, head_dim=64, inter=512, qkv_bias=True), [40, 1, 17, 64, 100]),
    "qknorm_hd32": (dict(n_layers=2, hidden=256, heads=8, kv_heads=2, head_dim=32, inter=384, qk_norm=True), [33, 2, 90]),
    "hd128_gqa8": (dict(n_layers=2, hidden=512, heads=8, kv_heads=1, head_dim=128, inter=512), [70, 130, 5]),
    "hd64_gqa7": (dict(n_layers=2, hidden=448, heads=7, kv_heads=1, head_dim=64, inter=384), [16, 15, 65]),
}


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("name", sorted(CASES))
def test_generation_with_the_8bit_cache(device, name, fmt, monkeypatch, request):
    kw, lens = CASES[name]
    spec, f32, tensors = make_model(900 + sorted(CASES).index(name), **kw)
    ps = prompts(910, lens, spec["vocab"])
    m = ditch_b200.Model(device, spec, tensors, max_seq=256)
    device.set_deterministic(True)  # split products in a fixed order, so that two runs can be compared
    request.addfinalizer(lambda: device.set_deterministic(False))
    m.set_kv_cache(fmt)
    got = m.generate(ps, 24)
    monkeypatch.setattr(base, "FWD_RTOL", 4e-2 if fmt == "int8" else 8e-2)
    n, exact = base.check_generation(OracleModel(spec, f32), ps, got, 24)
    assert n == 24 * len(ps)
    # a window over everything changes nothing; one that cuts is accepted and gives tokens
    m.set_kv_cache(fmt, window=1000, sinks=4)
    assert m.generate(ps, 24) == got
    m.set_kv_cache(fmt, window=16, sinks=2)
    cut = m.generate(ps, 24)
    assert [len(g) for g in cut] == [len(g) for g in got]
    assert all(0 <= t < spec["vocab"] for g in cut for t in g)
    m.set_kv_cache(None)  # the f32 cache again
    base.check_generation(OracleModel(spec, f32), ps, m.generate(ps, 24), 24)
    m.close()
    print(f"{name} {fmt}: {exact} of {n} tokens with a clear maximum")


def test_eos_and_window_against_masked_attention(device):
    """A window in the model's generation equals the cache attention's own
    definition: with one layer, a window of 1 leaves each token itself, so the
    continuation depends on the last token alone."""
    spec, f32, tensors = make_model(950, n_layers=1, hidden=128, heads=2, kv_heads=1, head_dim=64, inter=256)
    a, b = prompts(951, [30, 30], spec["vocab"])
    b = np.array(b)
    b[-1] = a[-1]
    m = ditch_b200.Model(device, spec, tensors, max_seq=128)
    m.set_kv_cache("int8", window=1)
    ga, gb = m.generate([a, b], 12)
    assert ga == gb
    g = m.generate([a], 12, eos_ids=[ga[3]])[0]
    assert g == ga[:ga.index(ga[3]) + 1]
    m.close()


def test_refusals(device):
    spec, f32, tensors = make_model(960, n_layers=1, hidden=128, heads=2, kv_heads=1, head_dim=40, inter=128)
    m = ditch_b200.Model(device, spec, tensors, max_seq=64)
    with pytest.raises(ditch_b200.Unsupported):
        m.set_kv_cache("int8")
    m.set_kv_cache(None)
    for args in (("int8", 0, 4), (None, 5, 0)):
        with pytest.raises(ditch_b200.DitchCudaError) as e:
            m.set_kv_cache(*args)
        assert e.value.code == 4
    m.close()
