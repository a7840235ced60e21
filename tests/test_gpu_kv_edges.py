"""The paged 8-bit cache and windowed attention where scales, magnitudes, pages
and offsets are out of the ordinary, against the definitions in f64.

Tolerance of an output element of 16 bits, from the formats: its own rounding,
u |out|, and the rounding of the softmax weights, u sum(p |v|) over the keys
that the row sees, with u = 2^-11 (f16) or 2^-8 (bf16) and |out| at most that
sum: 2 u sum(p max|v|) in all, and 5 % of it for the f32 sums, scores and
exponentials. What a row does not see has no part in it.
"""
import numpy as np
import pytest

import ditch_b200
from ditch_b200 import KvBatch, KvCache, Ragged, Rows
from test_gpu_kv import DT, STEP, TOP, Pool, gen, ints, randn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def reference(q, k, v, scale, window, sinks):
    """(out, sum of p max|v|) of f64 rows q [n, Hq, d] over k and v [len, Hkv, d], the queries the last of the tokens;
    NaN for a row that sees a key or value that is not finite."""
    n, hq, d = q.shape
    length, hkv = k.shape[:2]
    p, j = torch.arange(length - n, length, device=q.device), torch.arange(length, device=q.device)
    ok = j[None] <= p[:, None]
    if window:
        ok &= (j[None] > p[:, None] - window) | (j[None] < sinks)
    bad = ~(torch.isfinite(k).all(-1) & torch.isfinite(v).all(-1))
    k, v = (torch.where(bad[..., None], torch.zeros_like(x), x) for x in (k, v))
    out, bound = torch.zeros_like(q), torch.zeros_like(q[..., 0])
    for h in range(hq):
        kh = h // (hq // hkv)
        s = (q[:, h] @ k[:, kh].T * scale).masked_fill(~ok, -torch.inf)
        w = torch.softmax(s, -1)
        out[:, h], bound[:, h] = w @ v[:, kh], w @ v[:, kh].abs().amax(-1)
        out[(ok & bad[None, :, kh]).any(-1), h] = float("nan")
    return out, bound


def check(got, want, bound, dtype):
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    over = ((got - want).abs() / (2.1 * STEP[dtype] * bound + 1e-300)[..., None])[fine]
    assert not over.numel() or float(over.max()) <= 1.0, float(over.max())


def kernels_of(call):
    """The names of the kernels that `call` runs."""
    from torch.profiler import ProfilerActivity, profile

    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA], acc_events=True) as p:
        call()
        torch.cuda.synchronize()
    return [e.name for e in p.events()]


def attend(pool, q, new, scale, window=0, sinks=0, kernel=None, out=None):
    """The attention's rows; `kernel`: the kernel that the sizes are meant to reach."""
    out = torch.zeros_like(q) if out is None else out
    batch = pool.batch(new)
    size = pool.cache.attention_workspace(batch, q.shape[1])
    ws = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")

    def call():
        pool.cache.attention(batch, Rows.of(q), Rows.of(out), scale, window=window, sinks=sinks, workspace=ws, workspace_bytes=size)

    if kernel:
        assert any(kernel in n for n in kernels_of(call))
    else:
        call()
    torch.cuda.synchronize()
    pool.cache.dev.synchronize()
    return out


def check_all(pool, q, out, new, scale, window, sinks, dtype, values=None):
    at = 0
    for b, (a, t) in enumerate(zip(new, pool.lens)):
        k, v = (pool.values(w, b, t) for w in range(2)) if values is None else values[b]
        check(out[at:at + a], *reference(q[at:at + a].double(), k, v, scale, window, sinks), dtype)
        at += a


# 8 sequences of 300 rows in groups of 4 on 8 heads: what the tiled kernel takes
NEW = [300] * 8
LENS = [900 + 61 * i for i in range(8)]


@pytest.mark.parametrize("fmt,page,block", [("int8", 16, 16), ("fp8", 32, 16), ("int8", 32, 32)])
def test_tiled_pages_out_of_sight(device, fmt, page, block):
    """Tiles of 64 keys hold pages of which no row of the call sees a token:
    freed entries there, and pages of another owner with scales that are not
    finite, change nothing and are not reported."""
    g = gen(1)
    pool = Pool(device, g, fmt, LENS, 8, 128, page, block)
    q = randn(g, sum(NEW), 32, 128).to(torch.bfloat16)
    values = [[pool.values(w, b, t) for w in range(2)] for b, t in enumerate(LENS)]
    others = torch.isnan(pool.scales[0]).flatten(1).any(1).nonzero().flatten().tolist()
    for b, (a, t) in enumerate(zip(NEW, LENS)):
        for x in range(-(-4 // page), (t - a - 256 + 1) // page):
            pool.table[b, x] = (others[0], -1, 10 ** 6)[x % 3]
    out = attend(pool, q, NEW, 128 ** -0.5, 256, 4, kernel="k_tiled")
    check_all(pool, q, out, NEW, 128 ** -0.5, 256, 4, "bf16", values)


@pytest.mark.parametrize("layout", ["plain", "odd"])
def test_window_attention_nan_key_first(device, layout):
    """A NaN key that is the first, or the only one, that a row sees."""
    g = gen(2)
    pad = 0 if layout == "plain" else 3
    q, k, v = (randn(g, 400, h * 64 + pad).to(torch.bfloat16)[:, :h * 64].unflatten(1, (h, 64)) for h in (4, 2, 2))
    k[0, 1], k[150, 0] = float("nan"), float("nan")  # the first tokens of the two sequences
    k[230, 1] = float("nan")
    off = ints([0, 150, 400])
    out = torch.zeros_like(q)
    device.window_attention(Ragged(off, off, 2, 400, 400, 250, 250), Rows.of(q), Rows.of(k), Rows.of(v), Rows.of(out), 64, 0.125,
                            window=70)
    torch.cuda.synchronize()
    device.synchronize()
    for lo, hi in ((0, 150), (150, 400)):
        check(out[lo:hi], *reference(*(x[lo:hi].double() for x in (q, k, v)), 0.125, 70, 0), "bf16")


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("window", [0, 700])
def test_tiled_nan_key_scale_first(device, fmt, window):
    """A NaN scale of the first keys that rows see, in the tiled kernel."""
    g = gen(3)
    pool = Pool(device, g, fmt, LENS, 8, 128, 16, 16)
    pool.scales[0][int(pool.table[0, 0]), 3, 0] = float("nan")
    pool.scales[0][int(pool.table[2, 20]), 5, 0] = float("nan")
    q = randn(g, sum(NEW), 32, 128).to(torch.float16)
    out = attend(pool, q, NEW, 128 ** -0.5, window, 0, kernel="k_tiled")
    check_all(pool, q, out, NEW, 128 ** -0.5, window, 0, "f16")


@pytest.mark.parametrize("fmt,dtype,d,up,base", [
    ("int8", "bf16", 128, 12, 0), ("fp8", "bf16", 64, 20, 0), ("int8", "bf16", 64, 30, 0), ("fp8", "bf16", 128, 60, 0),
    ("int8", "bf16", 128, 70, -45), ("int8", "f16", 128, 14, -8), ("fp8", "f16", 64, 20, -10)])
def test_tiled_uneven_value_scales(device, fmt, dtype, d, up, base):
    """Blocks of values 2^up above the others: the rows that do not see them,
    or give them next to no weight, keep their precision."""
    g = gen(4)
    pool = Pool(device, g, fmt, LENS, 8, d, 16, 16)
    ks, vs = pool.scales
    vs *= 2.0 ** base

    def at(b, token):
        return int(pool.table[b, token // 16])

    vs[at(0, LENS[0] - 1)] *= 2.0 ** up    # the last tokens: most rows do not see them
    vs[at(1, LENS[1] - 150)] *= 2.0 ** up  # amid the new tokens
    vs[at(2, 17)] *= 2.0 ** up             # among the first tokens, with scores of -40
    pool.codes[0][at(2, 17)] = pool.encode(torch.full((8, 16, d), -TOP[fmt], device="cuda"))
    ks[at(2, 17)] = 1.0 / TOP[fmt]
    q = randn(g, sum(NEW), 32, d).to(DT[dtype])
    q[600:900] = (40 * d ** -0.5 + 0.1 * randn(g, 300, 32, d)).to(DT[dtype])
    vs[at(3, 40)] = 0.0                    # values of 0, and very small ones
    vs[at(4, 600)] *= 2.0 ** -50
    out = attend(pool, q, NEW, d ** -0.5, kernel="k_tiled")
    check_all(pool, q, out, NEW, d ** -0.5, 0, 0, dtype)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_tiled_values_all_zero(device, fmt):
    g = gen(5)
    pool = Pool(device, g, fmt, LENS, 8, 128, 16, 16)
    pool.scales[1][:] = 0.0
    q = randn(g, sum(NEW), 32, 128).to(torch.bfloat16)
    out = attend(pool, q, NEW, 128 ** -0.5, out=torch.ones_like(q), kernel="k_tiled")
    assert (out == 0).all()


def test_tiled_value_scale_not_finite_is_not_slow(device):
    """Rows that see a value scale that is not finite are NaN at once, and the
    others are not computed again one by one."""
    g = gen(6)
    pool = Pool(device, g, "int8", LENS, 8, 128, 16, 16)
    q = randn(g, sum(NEW), 32, 128).to(torch.bfloat16)

    def time():
        attend(pool, q, NEW, 128 ** -0.5)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        batch = pool.batch(NEW)
        size = pool.cache.attention_workspace(batch, 32)
        ws = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        a.record()
        pool.cache.attention(batch, Rows.of(q), Rows.of(out), 128 ** -0.5, workspace=ws, workspace_bytes=size)
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b)

    clean = time()
    pool.scales[1][int(pool.table[0, 45]), 2, 0] = float("nan")   # tokens 720..735: amid the new ones
    pool.scales[1][int(pool.table[1, 3]), :, 0] = float("inf")    # seen by all rows of the sequence
    pool.scales[0][int(pool.table[2, 5]), 7, 0] = float("nan")
    out = attend(pool, q, NEW, 128 ** -0.5, kernel="k_tiled")
    check_all(pool, q, out, NEW, 128 ** -0.5, 0, 0, "bf16")
    assert time() < 5 * clean


def test_append_offsets_that_begin_late_or_go_back(device):
    """Rows before the first sequence are left alone; offsets that decrease are
    reported. Several new tokens a sequence."""
    g = gen(7)
    lens, new = [70, 40, 33], [40, 8, 33]
    pool = Pool(device, g, "int8", lens, 2, 64, 16, 16)
    x = randn(g, 39 + sum(new), 2, 64)
    n = len(x)
    pool.cache.append(KvBatch(ints([39, 79, 87, 120]), ints(lens), pool.table, 3, n, 40, 70, pool.table.shape[1]), Rows.of(x), Rows.of(x))
    got = [y.clone() for y in pool.codes + pool.scales]
    torch.cuda.synchronize()
    device.synchronize()
    pool = Pool(device, gen(7), "int8", lens, 2, 64, 16, 16)
    y = x[39:].contiguous()
    pool.cache.append(pool.batch(new), Rows.of(y), Rows.of(y))
    torch.cuda.synchronize()
    device.synchronize()
    for a, b in zip(got, pool.codes + pool.scales):
        assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))
    # the second sequence ends before it begins; the third overlaps the first
    for first, offsets in ((0, [0, 40, 8, 48]), (60, [60, 100, 68, 108])):
        x = randn(g, first + 48, 2, 64)
        pool.cache.append(KvBatch(ints(offsets), ints([70, 40, 40]), pool.table, 3, len(x), 40, 70, pool.table.shape[1]), Rows.of(x),
                          Rows.of(x))
        torch.cuda.synchronize()
        with pytest.raises(ditch_b200.DitchCudaError):
            device.synchronize()
    device.synchronize()


@pytest.mark.parametrize("dtype,new", [("bf16", 1), ("f32", 1), ("bf16", 3), ("f32", 40)])
@pytest.mark.parametrize("power", [121, 122, 125, 127])
def test_int8_queries_near_the_largest_number(device, dtype, new, power):
    """Queries of up to 2^power, over keys as small: ordinary scores."""
    g = gen(8)
    pool = Pool(device, g, "int8", [100, 130], 2, 64, 16, 16)
    pool.scales[0] *= 2.0 ** -100
    q = (randn(g, 2 * new, 8, 64) / 6).clamp(-0.999, 0.999)
    q[:, :, 5] = 0.75
    q = (q * 2.0 ** power).to(DT[dtype])
    scale = 2.0 ** (100 - power + 2) / 8
    out = attend(pool, q, [new, new], scale)
    at = 0
    for b, t in enumerate(pool.lens):
        want, bound = reference(q[at:at + new].double(), pool.values(0, b, t), pool.values(1, b, t), scale, 0, 0)
        if dtype == "f32":  # 22 bits of the queries, f32 sums: as the tests of ordinary queries
            assert float((out[at:at + new].double() - want).abs().max()) <= 2e-5 * float(want.abs().max())
        else:
            check(out[at:at + new], want, bound, dtype)
        at += new


def sink_pool(device, fmt, lens, d):
    """Token 5 of each sequence takes nearly all weight and has a value of 0; the other keys are 0."""
    pool = Pool(device, gen(9), fmt, lens, 8, d, 16, 16)
    values = (1 + 0.2 * randn(gen(10), pool.n, 8, 16, d)) * (TOP[fmt] / 3)
    pool.codes[0][:] = pool.encode(torch.zeros_like(values))
    pool.codes[1][:] = pool.encode(values)
    pool.scales[0][:] = 1.0
    pool.scales[1][:] = 1.0 / 16
    first = pool.table[:, 0].long()
    pool.codes[0][first, :, 5] = pool.encode(torch.ones(len(lens), 8, d, device="cuda"))
    pool.codes[1][first, :, 5] = 0
    return pool


@pytest.mark.parametrize("fmt,dtype,bits", [
    ("int8", "f32", 12.3), ("int8", "f32", 16.6), ("fp8", "f32", 12.3), ("fp8", "f32", 16.6), ("fp8", "f16", 19.7), ("fp8", "bf16", 20.5)])
def test_small_weights_keep_their_bits(device, fmt, dtype, bits):
    """A sink with nearly all weight and no value: what is left of the row is
    made of weights of 2^-bits each, which keep their precision."""
    d = 64
    pool = sink_pool(device, fmt, [40, 33, 1000], d)
    q = torch.full((3, 8, d), bits * float(np.log(2.0)) / d, device="cuda").to(DT[dtype])
    out = attend(pool, q, [1, 1, 1], 1.0)
    for b, t in enumerate(pool.lens):
        want, bound = reference(q[b:b + 1].double(), pool.values(0, b, t), pool.values(1, b, t), 1.0, 0, 0)
        if dtype == "f32":  # two halves of a product 2^-22, scores and exponents up to 17 in f32, sums of up to 1000 terms
            assert float(((out[b:b + 1].double() - want).abs() / bound[..., None]).max()) <= 1e-5
        else:
            check(out[b:b + 1], want, bound, dtype)


@pytest.mark.parametrize("fmt,dtype,bits", [("int8", "bf16", 20.5), ("fp8", "f16", 18.2)])
def test_tiled_small_weights_keep_their_bits(device, fmt, dtype, bits):
    pool = sink_pool(device, fmt, LENS, 128)
    q = torch.full((sum(NEW), 32, 128), bits * float(np.log(2.0)) / 128, device="cuda").to(DT[dtype])
    out = attend(pool, q, NEW, 1.0, kernel="k_tiled")
    check_all(pool, q, out, NEW, 1.0, 0, 0, dtype)


@pytest.mark.parametrize("length", [500, 2500])
def test_window_attention_small_weights_keep_their_bits(device, length):
    q = torch.full((length, 4, 64), 18.2 * float(np.log(2.0)) / 64, device="cuda").half()
    k, v = torch.zeros(length, 2, 64, device="cuda").half(), (64 + 13 * randn(gen(11), length, 2, 64)).half()
    k[5], v[5] = 1.0, 0.0  # (outputs of 2^-12 and more: f16's normal numbers)
    off, out = ints([0, length]), torch.zeros_like(q)
    device.window_attention(Ragged(off, off, 1, length, length, length, length), Rows.of(q), Rows.of(k), Rows.of(v), Rows.of(out), 64, 1.0)
    torch.cuda.synchronize()
    device.synchronize()
    check(out, *reference(q.double(), k.double(), v.double(), 1.0, 0, 0), "f16")


@pytest.mark.parametrize("dtype,bits", [("f16", 19.7), ("bf16", 20.5), ("bf16", 17.1)])
def test_int8_values_of_0_leave_nothing(device, dtype, bits):
    """The same over int8 codes: a value of 0 with nearly all weight adds 0, also to f32 sums that are far smaller."""
    pool = sink_pool(device, "int8", [40, 33, 1000], 64)
    q = torch.full((3, 8, 64), bits * float(np.log(2.0)) / 64, device="cuda").to(DT[dtype])
    out = attend(pool, q, [1, 1, 1], 1.0)
    check_all(pool, q, out, [1, 1, 1], 1.0, 0, 0, dtype)


@pytest.mark.parametrize("dtype,length,window", [("f16", 700, 257), ("bf16", 2600, 0)])
def test_window_attention_repeats_itself(device, dtype, length, window):
    """Groups of 7 leave two rows of a tile of 128 without a query: what an
    earlier kernel left in shared memory there changes no row."""
    g = gen(12)

    def run(q, k, v):
        off, out = ints([0, len(q)]), torch.zeros_like(q)
        device.window_attention(Ragged(off, off, 1, len(q), len(q), len(q), len(q)), Rows.of(q), Rows.of(k), Rows.of(v), Rows.of(out), 64,
                                0.125, window=window)
        torch.cuda.synchronize()
        return out

    q, k, v = (randn(g, length, h, 64).to(DT[dtype]) for h in (14, 2, 2))
    k[:, :, ::9] *= 3
    first = run(q, k, v)
    for size in (1.0, 30.0, 300.0):
        run(*((size * randn(g, length, h, 64)).to(DT[dtype]) for h in (16, 2, 2)))  # 8 queries a group: all rows
        assert torch.equal(run(q, k, v), first)
    device.synchronize()
