"""The paged 8-bit key / value cache (append, read, attention) and windowed
attention over contiguous rows, against their definitions in f64.

Tolerances, from the formats alone:
  codes and scales    equal, bit for bit, to the formula evaluated in f32 (the
                      rotation's products and sums rounded one by one)
  f32 attention       2e-5 of the largest output: the products' inputs keep 22
                      bits or more, the sums are f32 (about 2^-22 for a sum of
                      hundreds of terms with cancellation), exp2 is within 2 ulp
  f16 / bf16 output   the output's rounding (2^-11 / 2^-8 relative) plus the
                      softmax weights' rounding, 2^-11 (f16) or 2^-8 (bf16) of
                      the sum of |p v|, at most the largest |v|: with s the
                      smallest step 2^-11 / 2^-8, at most 2 s max|v|
"""
import numpy as np
import pytest

import ditch_b200
from ditch_b200 import KvBatch, KvCache, Ragged, Rope, Rows

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TOP = {"int8": 127.0, "fp8": 448.0}
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


class Pool:
    """A pool with shuffled pages for sequences of `lens` tokens, random codes
    in it (junk everywhere, NaN scales in pages that nobody owns)."""

    def __init__(self, dev, g, fmt, lens, kv_heads, dim, page, block, spread=0.3):
        self.fmt, self.lens, self.heads, self.dim, self.page, self.block = fmt, lens, kv_heads, dim, page, block
        need = [-(-t // page) for t in lens]
        n = sum(need) + 2
        self.n = n
        order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = order[at:at + k]
            at += k
        self.codes, self.scales = [], []
        for _ in range(2):
            y = randn(g, n, kv_heads, page, dim) * (TOP[fmt] / 3)
            self.codes.append(self.encode(y))
            s = torch.exp(randn(g, n, kv_heads, page // block) * spread) / TOP[fmt] * 3
            s[order[at:].long()] = float("nan")
            self.scales.append(s)
        self.cache = KvCache(dev, fmt, self.codes[0], self.codes[1], self.scales[0], self.scales[1], kv_heads=kv_heads,
                             head_dim=dim, page_tokens=page, block_tokens=block, n_pages=n)

    def encode(self, y):
        y = y.clamp(-TOP[self.fmt], TOP[self.fmt])
        return (torch.round(y).to(torch.int8) if self.fmt == "int8" else y.to(torch.float8_e4m3fn)).view(torch.uint8)

    def decode(self, u):
        return (u.view(torch.int8) if self.fmt == "int8" else u.view(torch.float8_e4m3fn)).float()

    def rows(self, which, b, lo, hi):
        """(codes, scales) of tokens lo..hi-1 of sequence b."""
        t = torch.arange(lo, hi, device="cuda")
        page, off = self.table[b].long()[t // self.page], t % self.page
        return self.codes[which][page, :, off], self.scales[which][page, :, off // self.block]

    def values(self, which, b, hi):
        u, s = self.rows(which, b, 0, hi)
        return self.decode(u).double() * s.double()[..., None]

    def batch(self, new, lens=None):
        lens = self.lens if lens is None else lens
        offs = np.concatenate([[0], np.cumsum(new)]).tolist()
        return KvBatch(ints(offs), ints(lens), self.table, len(new), offs[-1], max(new), max(lens), self.table.shape[1])


def attention64(q, k, v, scale, window, sinks):
    """q [n, Hq, d], k and v [len, Hkv, d] in f64, the queries the last of the tokens."""
    n, hq, d = q.shape
    length, hkv = k.shape[:2]
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    p = torch.arange(length - n, length, device=q.device)
    j = torch.arange(length, device=q.device)
    ok = j[None] <= p[:, None]
    if window:
        ok &= (j[None] > p[:, None] - window) | (j[None] < sinks)
    for h in range(hq):
        kh = h // (hq // hkv)
        s = (q[:, h] @ k[:, kh].T) * scale
        s = torch.where(ok, s, torch.full_like(s, -torch.inf))
        top = s.amax(-1, keepdim=True) if length else s
        w = torch.where(ok, torch.exp(s - top), torch.zeros_like(s))
        total = w.sum(-1, keepdim=True)
        vv = v[:, kh]
        o = torch.zeros(n, d, dtype=torch.float64, device=q.device)
        seen = ok.any(-1)
        # what no row sees does not enter; what some row sees enters only there
        bad = ~torch.isfinite(vv).all(-1)
        o[seen] = (w[:, ~bad] @ vv[~bad])[seen] / total[seen]
        if bad.any():
            hit = (ok & bad[None]).any(-1)
            o[hit] = float("nan")
        out[:, h] = o
    return out


def close(got, want, kind, vmax):
    got, want = got.double(), want.double()
    if not want.numel():
        return
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    tol = 2e-5 * float(want[fine].abs().max()) if kind == "f32" else 2 * STEP[kind] * vmax
    err = float((got - want)[fine].abs().max()) if fine.any() else 0.0
    assert err <= tol, (err, tol)


# ---- append and read -----------------------------------------------------------
def rotate32(x, cos, sin, style):
    half = cos.shape[-1]
    r = x[..., :2 * half]
    a, b = (r[..., :half], r[..., half:]) if style == 0 else (r[..., 0::2], r[..., 1::2])
    c, s = cos[:, None], sin[:, None]
    a, b = a * c - b * s, b * c + a * s
    r = torch.cat([a, b], -1) if style == 0 else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([r, x[..., 2 * half:]], -1)


def over_top(x, fmt):
    """x / 127 or 448 as the f32 quotient (dividing by a Python number multiplies by its reciprocal)."""
    return x / torch.full_like(x, TOP[fmt])


def append32(pool, which, b, x, start):
    """The formula in f32: (codes, scales, per token) of the touched blocks' tokens lo..."""
    block = pool.block
    lo, end = start // block * block, start + len(x)
    codes, scales = [], []
    for f in range(lo, end, block):
        t = min(f + block, end)
        new = x[max(f, start) - start:t - start]
        fresh = over_top(new.abs().amax((0, 2)), pool.fmt)
        fresh = torch.where(fresh < 2.0 ** -126, torch.zeros_like(fresh), fresh)
        fresh = torch.where(torch.isfinite(new).all(-1).all(0), fresh, torch.full_like(fresh, float("nan")))
        s, old = fresh, None
        if f < start:
            u, sc = pool.rows(which, b, f, start)
            s = torch.maximum(fresh, sc[0])
            old = pool.decode(u) * torch.where(s > 0, sc[0] / s, torch.zeros_like(s))[:, None]
        inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
        y = new * inv[:, None]
        if old is not None:
            y = torch.cat([old, y])
        ok = torch.isfinite(s)[:, None]
        codes.append(pool.encode(torch.where(ok, y, torch.zeros_like(y))))
        scales.append(s[None].expand(t - f, -1))
    return lo, torch.cat(codes), torch.cat(scales)


APPENDS = [
    # fmt, dtype, q heads, kv heads, dim, page, block, (new, len) per sequence, half, style
    ("int8", "f32", 4, 2, 64, 16, 16, [(1, 1)], 32, 0),
    ("fp8", "bf16", 8, 8, 128, 64, 32, [(1, 33), (1, 32), (1, 1), (1, 100)], 64, 0),
    ("int8", "f16", 14, 2, 64, 32, 16, [(40, 40), (1, 77), (0, 9), (17, 32), (33, 50)], 32, 1),
    ("fp8", "f32", 4, 1, 128, 128, 64, [(130, 300), (1, 64), (65, 65)], 32, 0),
    ("int8", "bf16", 3, 3, 48, 64, 64, [(100, 163), (2, 65)], 16, 1),
    ("fp8", "f16", 6, 2, 112, 256, 16, [(19, 260), (300, 511)], 56, 0),
    ("int8", "f32", 2, 1, 16, 16, 16, [(5, 21), (31, 31)], 8, 0),
    ("int8", "bf16", 5, 5, 96, 32, 32, [(64, 70)], 0, 0),
    # more sequences than one step of the search takes, with and without several new tokens
    ("fp8", "bf16", 4, 2, 64, 16, 16, [(i % 4, 1 + i % 4 + i % 29) for i in range(150)], 32, 0),
    ("int8", "f16", 4, 2, 32, 64, 32, [(i % 3 != 1, 1 + i % 90) for i in range(1100)], 16, 1),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
@pytest.mark.parametrize("layout", ["columns", "odd"])
def test_append_and_read(device, case, layout):
    fmt, dtype, hq, hkv, d, page, block, seqs, half, style = APPENDS[case]
    g = gen(case)
    new, lens = [a for a, _ in seqs], [t for _, t in seqs]
    n = sum(new)
    pool = Pool(device, g, fmt, lens, hkv, d, page, block)
    width = (hq + 2 * hkv) * d + (0 if layout == "columns" else 3)  # odd: no head is 16-byte aligned
    flat = (randn(g, n, width) * torch.exp(randn(g, n, 1))).to(DT[dtype])
    col = lambda lo, h: flat.as_strided((n, h, d), (width, d, 1), lo)  # noqa: E731
    q, k, v = col(0, hq), col(hq * d, hkv), col((hq + hkv) * d, hkv)
    k[0, 0, 0] *= 50  # an outlier: a block's scale grows
    length = max(lens)
    ang = torch.rand(length, max(half, 1), generator=g, device="cuda") * 6.28
    cos, sin = torch.cos(ang), torch.sin(ang)
    rope = Rope(cos, sin, length, half, style) if half else None
    q_out, k_out, v_out = (torch.zeros(n, h, d, dtype=DT[t], device="cuda") for h, t in ((hq, dtype), (hkv, "bf16"), (hkv, "f32")))
    want, at = [], 0
    for b, (a, t) in enumerate(seqs):
        pos = torch.arange(t - a, t, device="cuda")
        turn = (lambda x: rotate32(x.float(), cos[pos], sin[pos], style)) if half else (lambda x: x.float())
        qq, kk, vv = turn(q[at:at + a]), turn(k[at:at + a]), v[at:at + a].float()
        want.append((qq, kk, vv, a and append32(pool, 0, b, kk, t - a), a and append32(pool, 1, b, vv, t - a)))
        at += a
    before = [x.clone() for x in pool.codes + pool.scales]
    batch = pool.batch(new)
    pool.cache.append(batch, Rows.of(k), Rows.of(v), q=Rows.of(q), q_out=Rows.of(q_out), rope=rope, k_out=Rows.of(k_out),
                      v_out=Rows.of(v_out))
    kb, vb = (torch.zeros(n, hkv, d, dtype=torch.float32, device="cuda") for _ in range(2))
    pool.cache.read(batch, Rows.of(kb), Rows.of(vb))
    torch.cuda.synchronize()
    device.synchronize()
    at = 0
    touched = [torch.zeros_like(x, dtype=torch.bool) for x in before]
    for b, (a, t) in enumerate(seqs):
        qq, kk, vv, wk, wv = want[b]
        assert torch.equal(q_out[at:at + a], qq.to(DT[dtype]))
        assert torch.equal(k_out[at:at + a], kk.to(torch.bfloat16)) and torch.equal(v_out[at:at + a], vv)
        for which, w, back in ((0, wk, kb), (1, wv, vb)):
            if not a:
                continue
            lo, codes, scales = w
            gc, gs = pool.rows(which, b, lo, t)
            assert torch.equal(gs, scales), which
            assert torch.equal(gc, codes), which
            vals = pool.decode(codes) * scales[..., None]
            assert torch.equal(back[at:at + a], vals[t - a - lo:])
            # within half a code of what was stored (half a step of e4m3's)
            x = kk if which == 0 else vv
            err = (vals[t - a - lo:] - x).abs()
            s = scales[t - a - lo:][..., None]
            step = s if fmt == "int8" else torch.maximum(x.abs() * 2.0 ** -3, s * 2.0 ** -9)
            assert (err <= 0.501 * step + 1e-30).all()
            tt = torch.arange(lo, t, device="cuda")
            pg, off = pool.table[b].long()[tt // page], tt % page
            touched[which][pg, :, off] = True
            touched[2 + which][pg, :, off // block] = True
        at += a
    for now, was, hit in zip(pool.codes + pool.scales, before, touched):  # nothing else was written
        same = (now == was) | (torch.isnan(now.float()) & torch.isnan(was.float()) if now.dtype == torch.float32 else False)
        assert bool((same | hit).all())


def test_append_token_by_token_and_in_place(device):
    """A sequence appended one token at a time: every block's values stay
    within one code of what was given (at most half a code when stored, and
    half a code each time its scale grew, shrinking in step with it)."""
    g = gen(77)
    for fmt in ("int8", "fp8"):
        pool = Pool(device, g, fmt, [40], 2, 64, 16, 16)
        k, v = randn(g, 40, 2, 64), randn(g, 40, 2, 64)
        for t in range(1, 41):
            pool.cache.append(pool.batch([1], [t]), Rows.of(k[t - 1:t]), Rows.of(v[t - 1:t]))
        torch.cuda.synchronize()
        for which, x in ((0, k), (1, v)):
            u, s = pool.rows(which, 0, 0, 40)
            got = pool.decode(u) * s[..., None]
            for f in range(0, 40, 16):
                part = x[f:f + 16]
                assert torch.equal(s[f], over_top(part.abs().amax((0, 2)), fmt))
            step = s[..., None] if fmt == "int8" else torch.maximum(x.abs() * 2.0 ** -3, s[..., None] * 2.0 ** -9)
            # int8: half a code of the last scale plus half a code of each smaller one before it
            grows = 16
            assert ((got - x).abs() <= 0.5 * grows * step).all() and ((got - x).abs().mean() <= 0.5 * step.mean())
    # queries and keys rotated in place
    q = randn(g, 3, 4, 64)
    want = q.clone()
    pool = Pool(device, g, "int8", [3], 2, 64, 16, 16)
    ang = torch.rand(3, 32, generator=g, device="cuda")
    k = randn(g, 3, 2, 64)
    pool.cache.append(pool.batch([3]), Rows.of(k), Rows.of(k), q=Rows.of(q), q_out=Rows.of(q),
                      rope=Rope(torch.cos(ang), torch.sin(ang), 3, 32))
    torch.cuda.synchronize()
    assert torch.equal(q, rotate32(want, torch.cos(ang), torch.sin(ang), 0))


def test_append_non_finite_zero_and_tiny(device):
    g = gen(5)
    pool = Pool(device, g, "int8", [48], 1, 32, 16, 16)
    x = randn(g, 48, 1, 32)
    x[3, 0, 5] = float("inf")
    x[20, 0, 1] = float("nan")
    x[32:] = 0.0
    y = torch.full((48, 1, 32), 1e-40, device="cuda")
    pool.cache.append(pool.batch([48]), Rows.of(x), Rows.of(y))
    torch.cuda.synchronize()
    u, s = pool.rows(0, 0, 0, 48)
    assert torch.isnan(s[:32]).all() and (s[32:] == 0).all() and (u == 0).all()
    u, s = pool.rows(1, 0, 0, 48)
    assert (s == 0).all() and (u == 0).all()


# ---- attention ---------------------------------------------------------------------
ATTENDS = [
    # fmt, dtype, q heads, kv heads, dim, page, block, (new, len), window, sinks
    ("int8", "f32", 4, 2, 64, 16, 16, [(1, 1)], 0, 0),
    ("int8", "bf16", 14, 2, 64, 16, 16, [(1, 201), (1, 16), (1, 17)], 0, 0),
    ("fp8", "f16", 8, 8, 128, 64, 32, [(1, 1000), (1, 3), (1, 64), (0, 5), (1, 65)], 0, 0),
    ("fp8", "f32", 32, 4, 128, 128, 64, [(1, 700), (1, 129)], 100, 4),
    ("int8", "bf16", 64, 8, 128, 32, 16, [(1, 3000), (1, 40)], 257, 17),
    ("int8", "f32", 16, 1, 96, 64, 64, [(3, 100), (1, 1), (2, 2)], 0, 0),
    ("fp8", "bf16", 12, 4, 80, 256, 16, [(5, 513), (4, 300)], 33, 1),
    ("int8", "f16", 6, 6, 128, 16, 16, [(70, 70), (1, 300), (33, 160)], 0, 0),
    ("int8", "bf16", 32, 8, 128, 64, 16, [(130, 700), (257, 257)], 0, 0),
    ("fp8", "bf16", 14, 2, 64, 64, 32, [(200, 1000), (90, 333), (1, 50)], 129, 5),
    ("fp8", "f32", 8, 2, 128, 64, 16, [(100, 400)], 64, 16),
    ("int8", "bf16", 40, 1, 112, 32, 32, [(7, 500)], 0, 0),
    ("int8", "f16", 4, 4, 16, 16, 16, [(40, 90), (1, 31)], 7, 3),
    ("fp8", "bf16", 2, 1, 32, 128, 64, [(1, 9000)], 0, 0),
    ("int8", "f32", 8, 1, 128, 64, 64, [(1, 12345), (1, 0x40)], 0, 0),
    ("int8", "bf16", 130, 1, 64, 64, 16, [(2, 100)], 1, 0),
    # many sequences: divided evenly over the CTAs, whole to a CTA, and tiled
    ("int8", "bf16", 8, 2, 64, 16, 16, [(1, 1 + 37 * i % 1500) for i in range(140)], 0, 0),
    ("fp8", "f16", 4, 2, 128, 64, 16, [(i % 2, 2 + i % 60) for i in range(200)], 0, 0),
    ("int8", "f16", 8, 2, 128, 32, 32, [(20 + i, 20 + i + 11 * i) for i in range(40)], 90, 3),
]


@pytest.mark.parametrize("case", range(len(ATTENDS)))
@pytest.mark.parametrize("layout", ["plain", "odd"])
def test_attention_over_the_cache(device, case, layout):
    fmt, dtype, hq, hkv, d, page, block, seqs, window, sinks = ATTENDS[case]
    g = gen(100 + case)
    new, lens = [a for a, _ in seqs], [t for _, t in seqs]
    n = sum(new)
    pool = Pool(device, g, fmt, lens, hkv, d, page, block)
    # the tokens past a sequence's end hold NaN codes and, in blocks of their own, NaN scales
    for b, t in enumerate(lens):
        last = -(-t // page) * page
        for x in range(t, last):
            pg, off = int(pool.table[b, x // page]), x % page
            for c, s in zip(pool.codes, pool.scales):
                c[pg, :, off] = 0x7f if fmt == "fp8" else 0x80
                if x // block * block >= t:
                    s[pg, :, off // block] = float("nan")
    pad = 0 if layout == "plain" else 5
    q = (randn(g, n, hq * d + pad)).to(DT[dtype])[:, :hq * d].unflatten(1, (hq, d))
    buf = torch.full((n, hq * d + pad), 7.0, dtype=DT[dtype], device="cuda")
    out = buf[:, :hq * d].unflatten(1, (hq, d))
    batch = pool.batch(new)
    size = pool.cache.attention_workspace(batch, hq)
    ws = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
    for _ in range(2):  # the workspace serves again
        pool.cache.attention(batch, Rows.of(q), Rows.of(out), d ** -0.5, window=window, sinks=sinks, workspace=ws,
                             workspace_bytes=size)
    torch.cuda.synchronize()
    device.synchronize()
    at = 0
    for b, (a, t) in enumerate(seqs):
        k, v = pool.values(0, b, t), pool.values(1, b, t)
        want = attention64(q[at:at + a].double(), k, v, d ** -0.5, window, sinks)
        close(out[at:at + a], want, dtype, float(v.abs().max()) if t else 0.0)
        at += a
    if pad:
        assert (buf[:, hq * d:] == 7.0).all()


def test_attention_pages_outside_the_window_may_be_gone(device):
    """With a window, the pages between the sinks and the window are not
    looked at: their numbers may be anything."""
    g = gen(9)
    for new, q_heads in ((1, 8), (150, 4)):
        pool = Pool(device, g, "int8", [2000], 2, 128, 16, 16)
        q = randn(g, new, q_heads, 128).to(torch.bfloat16)
        k, v = pool.values(0, 0, 2000), pool.values(1, 0, 2000)
        want = attention64(q.double(), k, v, 0.1, 256, 4)
        first = (2000 - new - 256 + 1) // 16  # the first page that the first row's window reaches
        pool.table[0, 1:first] = -1
        out = torch.zeros_like(q)
        batch = pool.batch([new])
        size = pool.cache.attention_workspace(batch, q_heads)
        ws = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
        pool.cache.attention(batch, Rows.of(q), Rows.of(out), 0.1, window=256, sinks=4, workspace=ws, workspace_bytes=size)
        torch.cuda.synchronize()
        device.synchronize()
        close(out, want, "bf16", float(v.abs().max()))


def test_attention_scale_not_finite(device):
    """A NaN scale reaches the rows that see its block, and no others."""
    g = gen(10)
    for new in (1, 40, 200):
        pool = Pool(device, g, "fp8", [200, 200], 1, 64, 16, 16)
        pool.scales[1][int(pool.table[0, 5]), 0, 0] = float("nan")  # tokens 80..95
        q = randn(g, 2 * new, 4, 64).to(torch.bfloat16)
        out = torch.zeros_like(q)
        batch = pool.batch([new, new])
        size = pool.cache.attention_workspace(batch, 4)
        ws = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
        pool.cache.attention(batch, Rows.of(q), Rows.of(out), 0.125, window=110, sinks=2, workspace=ws, workspace_bytes=size)
        torch.cuda.synchronize()
        for b in range(2):
            k, v = pool.values(0, b, 200), pool.values(1, b, 200)
            want = attention64(q[b * new:(b + 1) * new].double(), k, v, 0.125, 110, 2)
            vmax = float(v[torch.isfinite(v)].abs().max())
            close(out[b * new:(b + 1) * new], want, "bf16", vmax)


WINDOWS = [
    # dtype, q heads, kv heads, dim, (queries, keys), window, sinks
    ("bf16", 4, 2, 64, [(1, 1)], 0, 0),
    ("bf16", 32, 8, 128, [(64, 64), (33, 33), (1, 1), (50, 50)], 0, 0),
    ("f16", 14, 2, 64, [(101, 101), (300, 700), (1, 400), (0, 10), (129, 129)], 57, 4),
    ("bf16", 8, 1, 128, [(513, 513), (128, 1000)], 0, 0),
    ("f16", 3, 3, 96, [(200, 260)], 100, 17),
    ("bf16", 5, 1, 40, [(77, 77), (3, 2)], 0, 0),  # three queries, two keys: the first row sees nothing
    ("bf16", 12, 4, 128, [(700, 900)], 130, 0),
    ("f16", 6, 2, 112, [(5, 0), (31, 64)], 1, 0),
    ("bf16", 64, 8, 128, [(1000, 1000)], 256, 4),
    ("bf16", 130, 1, 64, [(9, 50)], 0, 0),
    ("f16", 4, 4, 8, [(300, 300)], 200, 150),
    ("bf16", 28, 4, 128, [(1, 2000), (2, 1999)], 0, 0),
    # runs of 2048 keys and more: the shape for long runs, with ragged ends (one row tile, few keys)
    ("bf16", 8, 2, 128, [(300, 2500), (33, 70), (1, 1), (40, 2049)], 0, 0),
    ("f16", 14, 2, 64, [(95, 3001), (18, 18), (19, 500)], 2500, 4),
    ("bf16", 4, 4, 80, [(129, 129), (2100, 2100)], 0, 0),
    ("bf16", 8, 2, 128, [(1 + i % 37, 1 + i % 37 + i % 5) for i in range(45)], 0, 0),
]


@pytest.mark.parametrize("case", range(len(WINDOWS)))
@pytest.mark.parametrize("layout", ["plain", "columns", "odd"])
def test_window_attention(device, case, layout):
    dtype, hq, hkv, d, seqs, window, sinks = WINDOWS[case]
    g = gen(200 + case)
    nq, nk = sum(a for a, _ in seqs), sum(t for _, t in seqs)
    pad = {"plain": 0, "columns": 64, "odd": 3}[layout]

    def rows(n, h):
        return randn(g, n, h * d + pad).to(DT[dtype])[:, :h * d].unflatten(1, (h, d))

    q, k, v = rows(nq, hq), rows(nk, hkv), rows(nk, hkv)
    buf = torch.full((nq, hq * d + pad), 7.0, dtype=DT[dtype], device="cuda")
    out = buf[:, :hq * d].unflatten(1, (hq, d))
    qo = np.concatenate([[0], np.cumsum([a for a, _ in seqs])]).tolist()
    ko = np.concatenate([[0], np.cumsum([t for _, t in seqs])]).tolist()
    ragged = Ragged(ints(qo), ints(ko), len(seqs), nq, nk, max(a for a, _ in seqs), max(t for _, t in seqs))
    device.window_attention(ragged, Rows.of(q), Rows.of(k), Rows.of(v), Rows.of(out), d, d ** -0.5, window=window, sinks=sinks)
    torch.cuda.synchronize()
    device.synchronize()
    for b, (a, t) in enumerate(seqs):
        kk, vv = k[ko[b]:ko[b + 1]].double(), v[ko[b]:ko[b + 1]].double()
        want = attention64(q[qo[b]:qo[b + 1]].double(), kk, vv, d ** -0.5, window, sinks)
        close(out[qo[b]:qo[b + 1]], want, dtype, float(vv.abs().max()) if t else 0.0)
    if pad:
        assert (buf[:, hq * d:] == 7.0).all()


def test_window_attention_non_finite_out_of_sight(device):
    """Infinities and NaN that a row does not see (later tokens, tokens before
    its window, the next sequence's) leave it as it is; rows that see them get
    what the formula gives."""
    g = gen(300)
    q, k, v = (randn(g, 300, 4, 64).to(torch.bfloat16) for _ in range(3))
    v[250] = float("nan")      # second sequence's token 50
    v[20, 1] = float("nan")    # first sequence's token 20, head 1
    k[251, 2] = float("-inf")  # scores of that token are infinite or NaN
    qo = ints([0, 200, 300])
    out = torch.zeros_like(q)
    device.window_attention(Ragged(qo, qo, 2, 300, 300, 200, 200), Rows.of(q), Rows.of(k), Rows.of(v), Rows.of(out), 64,
                            0.125, window=70, sinks=3)
    torch.cuda.synchronize()
    for lo, hi in ((0, 200), (200, 300)):
        for h in range(4):
            kk, vv = k[lo:hi, h:h + 1].double(), v[lo:hi, h:h + 1].double()
            if lo == 200 and h == 2:
                continue
            want = attention64(q[lo:hi, h:h + 1].double(), kk, vv, 0.125, 70, 3)
            close(out[lo:hi, h:h + 1], want, "bf16", float(vv[torch.isfinite(vv)].abs().max()))
    # head 2 of the second sequence: rows before token 50 do not see either
    want = attention64(q[200:250, 2:3].double(), k[200:250, 2:3].double(), v[200:250, 2:3].double(), 0.125, 70, 3)
    close(out[200:250, 2:3], want, "bf16", float(v[200:250, 2].abs().max()))


def test_streams_and_graph(device):
    """The calls run on the caller's stream and can be captured in a graph."""
    g = gen(400)
    pool = Pool(device, g, "int8", [100, 300], 2, 64, 16, 16)
    q = randn(g, 2, 8, 64).to(torch.bfloat16)
    out, kv = torch.zeros_like(q), randn(g, 2, 2, 64).to(torch.bfloat16)
    batch = pool.batch([1, 1])
    size = pool.cache.attention_workspace(batch, 8)
    ws = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
    qr, orow, kvr = Rows.of(q), Rows.of(out), Rows.of(kv)

    def step(stream):
        pool.cache.append(batch, kvr, kvr, stream=stream)
        pool.cache.attention(batch, qr, orow, 0.125, workspace=ws, workspace_bytes=size, stream=stream)

    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step(s.cuda_stream)
    s.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    want = torch.cat([attention64(q[b:b + 1].double(), pool.values(0, b, t), pool.values(1, b, t), 0.125, 0, 0)
                      for b, t in enumerate((100, 300))])
    close(out, want, "bf16", 12.0)


def test_device_side_numbers_out_of_bounds(device):
    """Offsets, lengths and pages outside their bounds are left out and
    reported by the next synchronize; the device stays usable."""
    g = gen(500)
    pool = Pool(device, g, "int8", [20, 20], 1, 32, 16, 16)
    x = randn(g, 2, 1, 32)
    keep = [c.clone() for c in pool.codes]
    for offsets, lens, pages in (([0, 1, 2], [21, 20], None), ([0, 5, 2], [20, 20], None), ([0, 1, 2], [20, 20], 10 ** 6)):
        table = pool.table.clone()
        if pages:
            table[:, 1] = pages
            table[0, 1] = -5
        b = KvBatch(ints(offsets), ints(lens), table, 2, 2, 1, 20, 2)
        out = torch.zeros(2, 1, 32, device="cuda")
        size = pool.cache.attention_workspace(b, 1)
        ws = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
        pool.cache.append(b, Rows.of(x), Rows.of(x))
        pool.cache.attention(b, Rows.of(x), Rows.of(out), 1.0, workspace=ws, workspace_bytes=size)
        torch.cuda.synchronize()
        with pytest.raises(ditch_b200.DitchCudaError):
            device.synchronize()
    device.synchronize()
    assert torch.equal(pool.codes[0][int(pool.table[0, 0])], keep[0][int(pool.table[0, 0])])


def test_refusals(device):
    g = gen(600)
    pool = Pool(device, g, "int8", [20], 2, 64, 16, 16)
    b = pool.batch([1])
    q, kv, x3 = randn(g, 1, 4, 64), randn(g, 1, 2, 64), randn(g, 1, 3, 64)
    bad = ditch_b200.DitchCudaError

    def cache(**kw):
        a = dict(kv_heads=2, head_dim=64, page_tokens=16, block_tokens=16, n_pages=pool.n)
        a.update(kw)
        return KvCache(device, "int8", pool.codes[0], pool.codes[1], pool.scales[0], pool.scales[1], **a)

    for kw in (dict(page_tokens=24), dict(page_tokens=512), dict(block_tokens=32), dict(block_tokens=8), dict(kv_heads=0),
               dict(n_pages=0), dict(head_dim=0)):
        with pytest.raises(bad) as e:
            cache(**kw).append(b, Rows.of(kv), Rows.of(kv))
        assert e.value.code == 4, kw
    for dim in (24, 144):
        with pytest.raises(ditch_b200.Unsupported):
            cache(head_dim=dim).append(b, Rows.of(kv), Rows.of(kv))
    tab = torch.zeros(20, 32, device="cuda")
    for rope in (Rope(tab, tab, 19, 32), Rope(tab, tab, 20, 40), Rope(tab, tab, 20, 32, 2), Rope(None, tab, 20, 32)):
        with pytest.raises(bad):
            pool.cache.append(b, Rows.of(kv), Rows.of(kv), rope=rope)
    with pytest.raises(ditch_b200.Unsupported):
        pool.cache.append(b, Rows.of(kv), Rows.of(kv), rope=Rope(tab, tab, 20, 12))
    for args in ((Rows.of(x3), Rows.of(kv)), (Rows.of(kv), Rows.of(kv.half()))):
        with pytest.raises(bad):
            pool.cache.append(b, *args)
    with pytest.raises(bad):
        pool.cache.append(b, Rows.of(kv), Rows.of(kv), q=Rows.of(q))
    with pytest.raises(bad):
        pool.cache.read(b, Rows.of(kv), Rows.of(x3))
    for args, kw in (((Rows.of(x3), Rows.of(x3), 1.0), {}), ((Rows.of(q), Rows.of(kv), 1.0), {}), ((Rows.of(q), Rows.of(q), 0.0), {}),
                     ((Rows.of(q), Rows.of(q), float("nan")), {}), ((Rows.of(q), Rows.of(q), 1.0), dict(sinks=4))):
        with pytest.raises(bad):
            pool.cache.attention(b, *args, **kw)
    h = q.half()
    off = ints([0, 1])
    rg = Ragged(off, off, 1, 1, 1, 1, 1)
    with pytest.raises(ditch_b200.Unsupported):
        device.window_attention(rg, Rows.of(q), Rows.of(q), Rows.of(q), Rows.of(q), 64, 1.0)
    with pytest.raises(ditch_b200.Unsupported):
        device.window_attention(rg, Rows.of(h), Rows.of(h), Rows.of(h), Rows.of(h), 60, 1.0)
    with pytest.raises(bad):
        device.window_attention(rg, Rows.of(h), Rows.of(x3.half()), Rows.of(x3.half()), Rows.of(h), 64, 1.0)
    with pytest.raises(bad):
        device.window_attention(rg, Rows.of(h), Rows.of(h), Rows.of(h), Rows.of(q.bfloat16()), 64, 1.0)
    with pytest.raises(bad):
        device.window_attention(Ragged(off, None, 1, 1, 1, 1, 1), Rows.of(h), Rows.of(h), Rows.of(h), Rows.of(h), 64, 1.0)
    with pytest.raises(ValueError):
        Rows.of(q[0])
    # an empty batch is fine and does nothing
    empty = KvBatch(ints([0]), None, None, 0, 0, 0, 0, 0)
    pool.cache.append(empty, Rows.of(kv), Rows.of(kv))
    pool.cache.attention(empty, Rows.of(q), Rows.of(q), 1.0)
    device.window_attention(Ragged(None, None, 0, 0, 0, 0, 0), Rows.of(h), Rows.of(h), Rows.of(h), Rows.of(h), 64, 1.0)
