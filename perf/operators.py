"""The operators of the paged 8-bit key / value cache and of windowed attention: the cases they are measured on, their
plain forms, and their values in 64 bits.

  append   rotary embedding of new queries and keys; the keys and values rounded to 8-bit codes with one scale for each
           block of tokens and head, and written to a paged cache. The rows written are read back as values.
  attend   attention of each sequence's newest tokens over that cache (single tokens and chunks), causal, with an optional
           sliding window and first tokens (sinks) that stay visible.
  window   the same attention over contiguous keys and values of 16 bits (a prompt's own rows).
"""
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TOP = {"int8": 127.0, "fp8": 448.0}  # the largest code of each cache format
TINY = 2.0 ** -126                   # scales below the smallest normal f32 are stored as 0


# ---- cases -------------------------------------------------------------------
def listed():
    return [
        # one token of one short sequence, small heads: the latency of a lone decode step
        dict(name="append-one", op="append", format="int8", type="bf16", q_heads=14, kv_heads=2, head_dim=64, page=16, block=16,
             seqs=1, new_lo=1, new_hi=1, len_lo=101, len_hi=101, rot=64, style=0, at=1),
        # a batched decode step: one token for each of 128 sequences
        dict(name="append-step", op="append", format="fp8", type="bf16", q_heads=32, kv_heads=8, head_dim=128, page=64, block=32,
             seqs=128, new_lo=1, new_hi=1, len_lo=65, len_hi=1000, rot=128, style=0, at=2),
        # the prefill of 128 prompts of 64 tokens from the f32 rows of a QKV product
        dict(name="append-prompts", op="append", format="int8", type="f32", q_heads=32, kv_heads=8, head_dim=128, page=64, block=16,
             seqs=128, new_lo=64, new_hi=64, len_lo=64, len_hi=64, rot=128, style=0, at=3),
        # ragged chunks of long prompts, interleaved rotation of half of each head
        dict(name="append-chunks", op="append", format="fp8", type="f16", q_heads=64, kv_heads=8, head_dim=128, page=128, block=64,
             seqs=7, new_lo=200, new_hi=1500, len_lo=1500, len_hi=4500, rot=64, style=1, at=4),
        # a lone decode step over a short context
        dict(name="attend-one", op="attend", format="int8", type="bf16", q_heads=14, kv_heads=2, head_dim=64, page=16, block=16,
             seqs=1, new_lo=1, new_hi=1, len_lo=201, len_hi=201, window=0, sinks=0, at=5),
        # decode steps of 128 prompts of 64 tokens and up to 100 generated ones, at f32
        dict(name="attend-step", op="attend", format="int8", type="f32", q_heads=32, kv_heads=8, head_dim=128, page=64, block=16,
             seqs=128, new_lo=1, new_hi=1, len_lo=65, len_hi=164, window=0, sinks=0, at=6),
        # decode over long ragged contexts: the cache's bytes are all that counts
        dict(name="attend-long", op="attend", format="fp8", type="bf16", q_heads=32, kv_heads=8, head_dim=128, page=64, block=32,
             seqs=32, new_lo=1, new_hi=1, len_lo=4000, len_hi=32000, window=0, sinks=0, at=7),
        # decode with a sliding window and four sinks: most of each context is out of sight
        dict(name="attend-window", op="attend", format="int8", type="bf16", q_heads=64, kv_heads=8, head_dim=128, page=32, block=16,
             seqs=64, new_lo=1, new_hi=1, len_lo=500, len_hi=8000, window=1024, sinks=4, at=8),
        # a chunk of new tokens for each of four sequences over what they have cached
        dict(name="attend-chunk", op="attend", format="int8", type="bf16", q_heads=32, kv_heads=8, head_dim=128, page=64, block=16,
             seqs=4, new_lo=512, new_hi=512, len_lo=1000, len_hi=8000, window=0, sinks=0, at=9),
        # the prefill of 128 ragged prompts of at most 64 tokens
        dict(name="window-prompts", op="window", type="bf16", q_heads=32, kv_heads=8, head_dim=128, seqs=128, new_lo=33, new_hi=64,
             past_lo=0, past_hi=0, window=0, sinks=0, at=10),
        # ragged prompts of odd lengths after prefixes of their own, small heads in groups of seven
        dict(name="window-odd", op="window", type="f16", q_heads=14, kv_heads=2, head_dim=64, seqs=5, new_lo=101, new_hi=1901,
             past_lo=0, past_hi=701, window=257, sinks=4, at=11),
        # one long prompt under a window of half its length
        dict(name="window-long", op="window", type="bf16", q_heads=64, kv_heads=8, head_dim=128, seqs=1, new_lo=8192, new_hi=8192,
             past_lo=0, past_hi=0, window=4096, sinks=4, at=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "window"])
    q_heads, kv_heads = rng.choice([(14, 2), (32, 8), (64, 8), (16, 16), (8, 1), (12, 4)])
    c = dict(op=op, type=rng.choice(["bf16", "bf16", "f16"]), q_heads=q_heads, kv_heads=kv_heads, head_dim=rng.choice([64, 128]),
             at=rng.randrange(1 << 20))
    if op == "window":
        seqs = _log(rng, 1, 64)
        top = _log(rng, 16, max(16, 6000 // seqs))
        c.update(seqs=seqs, new_lo=max(1, top // 3), new_hi=top, past_lo=0, past_hi=rng.choice([0, 333]),
                 window=rng.choice([0, _log(rng, 16, 4096)]))
        c["sinks"] = rng.choice([0, 4, 17]) if c["window"] else 0
        return c
    c["format"] = rng.choice(["int8", "fp8"])
    c["type"] = rng.choice(["bf16", "f16", "f32"])
    c["page"] = rng.choice([16, 32, 64, 128])
    c["block"] = rng.choice([b for b in (16, 32, 64) if b <= c["page"]])
    if op == "append":
        seqs = _log(rng, 1, 128)
        new = rng.choice([1, 1, _log(rng, 2, max(2, 8192 // seqs))])
        c.update(seqs=seqs, new_lo=max(1, new // 2), new_hi=new, len_lo=new, len_hi=new + _log(rng, 1, 2000), style=rng.choice([0, 1]))
        c["rot"] = rng.choice([c["head_dim"], c["head_dim"], c["head_dim"] // 2])
        return c
    if rng.random() < 0.65:  # a decode step
        seqs = _log(rng, 1, 128)
        top = _log(rng, 60, min(32000, max(60, 400000 // seqs)))
        c.update(seqs=seqs, new_lo=1, new_hi=1, len_lo=max(1, top // 4), len_hi=top)
    else:  # a few tokens at once, or a chunk
        seqs = _log(rng, 1, 8)
        new = _log(rng, 2, 600)
        c.update(seqs=seqs, new_lo=max(1, new // 2), new_hi=new, len_lo=new, len_hi=new + _log(rng, 1, 4000))
    c["window"] = rng.choice([0, 0, _log(rng, 16, 4096)])
    c["sinks"] = rng.choice([0, 4, 17]) if c["window"] else 0
    return c


def _lengths(c):
    """(new tokens, length with them) of each sequence: fixed by the case alone."""
    r = random.Random(c["at"])
    got = []
    for _ in range(c["seqs"]):
        new = r.randint(c["new_lo"], c["new_hi"])
        total = new + r.randint(c["past_lo"], c["past_hi"]) if c["op"] == "window" else max(new, r.randint(c["len_lo"], c["len_hi"]))
        got.append((new, total))
    return got


def _pairs(c):
    """Visible (query, key) pairs, and keys that some query sees, over all sequences."""
    pairs = seen = 0
    w, s = c["window"], c["sinks"]
    for new, total in _lengths(c):
        first = total - new
        if not w:
            pairs += sum(range(first + 1, total + 1))
            seen += total
            continue
        for p in range(first, total):
            low = max(0, p - w + 1)
            pairs += p + 1 - low + min(s, low)
        low = max(0, first - w + 1)
        seen += total - low + min(s, low)
    return pairs, seen


def work(c):
    size = {"f32": 4, "bf16": 2, "f16": 2}[c["type"]]
    hq, hkv, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    n = sum(a for a, _ in _lengths(c))
    if c["op"] == "append":
        out = 4 if c["type"] == "f32" else 2
        back = sum(t - (t - a) // c["block"] * c["block"] for a, t in _lengths(c))
        # rows in, rotated queries out, codes out, then the written blocks' codes in and their values out
        return {"bytes": n * d * ((hq + 2 * hkv) * size + hq * out + 2 * hkv) + back * 2 * hkv * d * 3, "flops": 6 * n * d * (hq + hkv)}
    pairs, seen = _pairs(c)
    if c["op"] == "attend":
        return {"bytes": seen * hkv * (2 * d + 8 / c["block"]) + 2 * n * hq * d * size, "flops": 4 * pairs * d * hq}
    return {"bytes": (seen * hkv * 2 + 2 * n * hq) * d * size, "flops": 4 * pairs * d * hq}


# ---- inputs --------------------------------------------------------------------
def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _keys(g, *shape):
    """Keys as models make them: a few of a head's dimensions are several times the others."""
    x = _randn(g, *shape)
    x[..., ::19] *= 4.0
    return x


def _pool(c, g, st):
    """A pool of pages in which the sequences' pages lie in no order, full of codes as the quantiser makes them."""
    page, hkv, d = c["page"], c["kv_heads"], c["head_dim"]
    need = [-(-t // page) for _, t in st["lengths"]]
    n = sum(need) + 3
    order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(c["seqs"], max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    st.update(table=table, n_pages=n, max_pages=max(need))
    for name in ("k", "v"):
        x = torch.empty(n, hkv, page, d, dtype=torch.uint8, device="cuda")
        for lo in range(0, n, 4096):
            hi = min(n, lo + 4096)
            y = torch.randn(hi - lo, hkv, page, d, generator=g, device="cuda")
            if c["format"] == "int8":
                x[lo:hi] = torch.round(y * 40).clamp(-127, 127).to(torch.int8).view(torch.uint8)
            else:
                x[lo:hi] = (y * 140).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        st[name + "_pool"] = x
        mid = (3.0 if name == "k" else 2.0) / TOP[c["format"]]
        st[name + "_scale"] = torch.exp(_randn(g, n, hkv, page // c["block"], std=0.3)) * mid


def _touched(c, st):
    """For the plain append: every token of the blocks that the new tokens reach, sequence by sequence."""
    page, block = c["page"], c["block"]
    seq, pos, src, blk, first = [], [], [], [], []
    blocks = at = 0
    for b, (new, total) in enumerate(st["lengths"]):
        start = total - new
        lo = start // block * block
        for f in range(lo, total, block):
            first.append((b, f, 1 if f < start else 0))
        for p in range(lo, total):
            seq.append(b)
            pos.append(p)
            src.append(at + p - start if p >= start else -1)
            blk.append(blocks + (p - lo) // block)
        blocks += -(-(total - lo) // block)
        at += new
    seq, pos, src, blk, first = (torch.tensor(v, device="cuda") for v in (seq, pos, src, blk, first))
    new = torch.nonzero(src >= 0).flatten()
    old = torch.nonzero(src < 0).flatten()
    st["plan"] = dict(page=st["table"][seq, pos // page].long(), off=pos % page, pos=pos, blk=blk, new=new, old=old, n_blocks=blocks,
                      block_page=st["table"][first[:, 0], first[:, 1] // page].long(), block_off=first[:, 1] % page // block,
                      keep=first[:, 2].bool())


def _index(c, st, keys):
    """For the plain attentions: where each (sequence, query) and (sequence, key) lies in the flat rows, padded."""
    new = torch.tensor([a for a, _ in st["lengths"]], device="cuda")
    total = torch.tensor([t for _, t in st["lengths"]], device="cuda")
    i = torch.arange(int(max(a for a, _ in st["lengths"])), device="cuda")
    q_at = (st["offsets"][:-1].long()[:, None] + i).clamp(max=st["n_new"] - 1)
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), new)
    st["plan"] = dict(new=new, total=total, q_at=q_at, seq=seq, row=torch.arange(st["n_new"], device="cuda") - st["offsets"][:-1].long()[seq])
    if keys:
        j = torch.arange(int(max(t for _, t in st["lengths"])), device="cuda")
        st["plan"]["k_at"] = (st["kv_offsets"][:-1].long()[:, None] + j).clamp(max=st["n_kv"] - 1)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, hq, hkv, d = TYPES[c["type"]], c["q_heads"], c["kv_heads"], c["head_dim"]
    lengths = _lengths(c)
    offsets = [0]
    for a, _ in lengths:
        offsets.append(offsets[-1] + a)
    n = offsets[-1]
    st = dict(case=c, lengths=lengths, n_new=n, offsets=_ints(offsets), lens=_ints([t for _, t in lengths]),
              max_new=max(a for a, _ in lengths), max_len=max(t for _, t in lengths))
    if c["op"] == "append":
        # the rows of one QKV product: queries, keys and values are its columns
        rows = torch.cat([_randn(g, n, hq, d), _keys(g, n, hkv, d), _randn(g, n, hkv, d, std=0.7)], 1).to(dt)
        st.update(q=rows[:, :hq], k=rows[:, hq:hq + hkv], v=rows[:, hq + hkv:], q_out=torch.empty(n, hq, d, dtype=dt, device="cuda"))
        angle = torch.arange(st["max_len"], device="cuda")[:, None] * 10000.0 ** (-torch.arange(c["rot"] // 2, device="cuda") * 2.0 / c["rot"])
        st.update(cos=torch.cos(angle).float(), sin=torch.sin(angle).float())
        _pool(c, g, st)
        _touched(c, st)
        m = len(st["plan"]["pos"])
        st.update(k_back=torch.empty(m, hkv, d, dtype=torch.bfloat16, device="cuda"), v_back=torch.empty(m, hkv, d, dtype=torch.bfloat16, device="cuda"))
        back = [0]
        for a, t in lengths:
            back.append(back[-1] + t - (t - a) // c["block"] * c["block"])
        st["back_offsets"] = _ints(back)
    elif c["op"] == "attend":
        st.update(q=_randn(g, n, hq, d, std=0.5, dtype=dt), out=torch.empty(n, hq, d, dtype=dt, device="cuda"))
        _pool(c, g, st)
        _index(c, st, False)
    else:
        kv = [0]
        for _, t in lengths:
            kv.append(kv[-1] + t)
        st.update(n_kv=kv[-1], kv_offsets=_ints(kv), q=_randn(g, n, hq, d, dtype=dt), k=_keys(g, kv[-1], hkv, d).to(dt),
                  v=_randn(g, kv[-1], hkv, d, std=0.7, dtype=dt), out=torch.empty(n, hq, d, dtype=dt, device="cuda"))
        _index(c, st, True)
    if own:
        import ditch_b200 as db
        global _device
        _device = _device or db.Device(0)
        if c["op"] == "window":
            st["ragged"] = db.Ragged(st["offsets"], st["kv_offsets"], c["seqs"], n, st["n_kv"], st["max_new"], st["max_len"])
            st["rows"] = [db.Rows.of(st[x]) for x in ("q", "k", "v", "out")]
            return st
        st["cache"] = db.KvCache(_device, c["format"], st["k_pool"], st["v_pool"], st["k_scale"], st["v_scale"], kv_heads=hkv,
                                 head_dim=d, page_tokens=c["page"], block_tokens=c["block"], n_pages=st["n_pages"])
        st["batch"] = db.KvBatch(st["offsets"], st["lens"], st["table"], c["seqs"], n, st["max_new"], st["max_len"], st["max_pages"])
        if c["op"] == "append":
            st["rows"] = [db.Rows.of(st[x]) for x in ("q", "k", "v", "q_out")]
            st["rope"] = db.Rope(st["cos"], st["sin"], st["max_len"], c["rot"] // 2, c["style"])
            st["back_rows"] = [db.Rows.of(st[x]) for x in ("k_back", "v_back")]
            st["back"] = db.KvBatch(st["back_offsets"], st["lens"], st["table"], c["seqs"], back[-1], max(b - a for a, b in zip(back, back[1:])),
                                    st["max_len"], st["max_pages"])
        else:
            st["rows"] = [db.Rows.of(st[x]) for x in ("q", "out")]
            st["bytes"] = st["cache"].attention_workspace(st["batch"], hq)
            st["workspace"] = torch.zeros(max(1, st["bytes"]), dtype=torch.uint8, device="cuda")
    return st


_device = None


# ---- one pass ------------------------------------------------------------------
def run(st):
    c = st["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "window": _plain_window}[c["op"]](st)
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        q, k, v, q_out = st["rows"]
        st["cache"].append(st["batch"], k, v, q=q, q_out=q_out, rope=st["rope"], stream=stream)
        st["cache"].read(st["back"], *st["back_rows"], stream=stream)
        return {"q": st["q_out"], "k": st["k_back"], "v": st["v_back"]}
    scale = c["head_dim"] ** -0.5
    if c["op"] == "attend":
        q, out = st["rows"]
        st["cache"].attention(st["batch"], q, out, scale, window=c["window"], sinks=c["sinks"], workspace=st["workspace"],
                              workspace_bytes=st["bytes"], stream=stream)
        return st["out"]
    q, k, v, out = st["rows"]
    _device.window_attention(st["ragged"], q, k, v, out, c["head_dim"], scale, window=c["window"], sinks=c["sinks"], stream=stream)
    return st["out"]


def _rotate(x, cos, sin, style):
    """x [n, heads, d] f32; the first 2 * half dimensions rotate, in halves (0) or in neighbours (1)."""
    half = cos.shape[-1]
    r = x[..., :2 * half]
    a, b = (r[..., :half], r[..., half:]) if style == 0 else (r[..., 0::2], r[..., 1::2])
    co, si = cos[:, None], sin[:, None]
    a, b = a * co - b * si, b * co + a * si
    r = torch.cat([a, b], -1) if style == 0 else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([r, x[..., 2 * half:]], -1)


def _code_values(c, u8):
    return (u8.view(torch.int8) if c["format"] == "int8" else u8.view(torch.float8_e4m3fn)).float()


def _encode(c, x):
    top = TOP[c["format"]]
    x = x.clamp(-top, top)
    return (torch.round(x).to(torch.int8) if c["format"] == "int8" else x.to(torch.float8_e4m3fn)).view(torch.uint8)


def _plain_append(st):
    c, p = st["case"], st["plan"]
    hkv, d = c["kv_heads"], c["head_dim"]
    cos, sin = st["cos"][p["pos"][p["new"]]], st["sin"][p["pos"][p["new"]]]
    st["q_out"].copy_(_rotate(st["q"].float(), cos, sin, c["style"]))
    got = {"q": st["q_out"]}
    for name, x in (("k", _rotate(st["k"].float(), cos, sin, c["style"])), ("v", st["v"].float())):
        pool, scales = st[name + "_pool"], st[name + "_scale"]
        blk = p["blk"][p["new"]]
        top = torch.zeros(p["n_blocks"], hkv, device="cuda").index_reduce_(0, blk, x.abs().amax(-1), "amax")
        fresh = top / TOP[c["format"]]
        fresh = torch.where(fresh < TINY, torch.zeros_like(fresh), fresh)
        was = scales[p["block_page"], :, p["block_off"]]
        kept = torch.where(p["keep"][:, None], was, torch.zeros_like(was))
        s = torch.maximum(kept, fresh)
        nil = s == 0
        inverse = torch.where(nil, torch.zeros_like(s), 1.0 / s)
        ratio = torch.where(nil, torch.zeros_like(s), kept / s)
        codes = torch.empty(len(p["pos"]), hkv, d, dtype=torch.uint8, device="cuda")
        codes[p["new"]] = _encode(c, x * inverse[blk][..., None])
        old = p["old"]
        codes[old] = _encode(c, _code_values(c, pool[p["page"][old], :, p["off"][old]]) * ratio[p["blk"][old]][..., None])
        pool[p["page"], :, p["off"]] = codes
        scales[p["block_page"], :, p["block_off"]] = s
        got[name] = (_code_values(c, codes) * s[p["blk"]][..., None]).to(torch.bfloat16)
    return got


def _attention(c, q, k, v, new, total):
    """q [B, T, Hq, d], k and v [B, S, Hkv, d], all f32 and padded: f32 [B, T, Hq, d], zero where a row sees nothing."""
    b, t, hq, d = q.shape
    s, hkv = k.shape[1], k.shape[2]
    g = hq // hkv
    x = torch.matmul(q.view(b, t, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * t, d), k.permute(0, 2, 3, 1)).view(b, hkv, g, t, s)
    x *= d ** -0.5
    i = torch.arange(t, device="cuda")
    j = torch.arange(s, device="cuda")
    at = (total - new)[:, None] + i
    hidden = (j > at[:, :, None]) | (i >= new[:, None])[:, :, None]
    if c["window"]:
        hidden |= (j <= at[:, :, None] - c["window"]) & (j >= c["sinks"])
    x.masked_fill_(hidden[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x -= torch.where(torch.isinf(top), torch.zeros_like(top), top)
    x = torch.exp_(x)
    total_p = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, hkv, g * t, s), v.permute(0, 2, 1, 3)).view(b, hkv, g, t, d)
    o = o / torch.where(total_p > 0, total_p, torch.ones_like(total_p))
    return o.permute(0, 3, 1, 2, 4).reshape(b, t, hq, d)


def _plain_attend(st):
    c, p = st["case"], st["plan"]
    page = c["page"]
    pos = torch.arange(st["max_len"], device="cuda")
    pages = st["table"].long()[:, pos // page]
    rows = []
    for name in ("k", "v"):
        codes = _code_values(c, st[name + "_pool"][pages, :, pos % page])
        rows.append(codes * st[name + "_scale"][pages, :, pos % page // c["block"]][..., None])
    o = _attention(c, st["q"].float()[p["q_at"]], *rows, p["new"], p["total"])
    return o[p["seq"], p["row"]].to(st["q"].dtype)


def _plain_window(st):
    c, p = st["case"], st["plan"]
    o = _attention(c, st["q"].float()[p["q_at"]], st["k"].float()[p["k_at"]], st["v"].float()[p["k_at"]], p["new"], p["total"])
    return o[p["seq"], p["row"]].to(st["q"].dtype)


# ---- the definitions in 64 bits --------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_append(st) if case["op"] == "append" else _exact_attention(st)


def _exact_values(c, st, name, b, lo, hi):
    """Values of tokens lo..hi-1 of sequence b in the cache, [hi - lo, Hkv, d]."""
    at = torch.arange(lo, hi, device="cuda")
    page = st["table"][b].long()[at // c["page"]]
    off = at % c["page"]
    u8 = st[name + "_pool"][page, :, off]
    x = (u8.view(torch.int8).double() if c["format"] == "int8" else u8.view(torch.float8_e4m3fn).double())
    return x, st[name + "_scale"][page, :, off // c["block"]].double()


def _exact_attention(st):
    c = st["case"]
    hq, hkv, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    g = hq // hkv
    result = torch.zeros(st["n_new"], hq, d, dtype=torch.float64, device="cuda")
    q_start = kv_start = 0
    for b, (new, total) in enumerate(st["lengths"]):
        if c["op"] == "attend":
            (kc, ks), (vc, vs) = _exact_values(c, st, "k", b, 0, total), _exact_values(c, st, "v", b, 0, total)
            keys, values = kc * ks[..., None], vc * vs[..., None]
        else:
            keys, values = st["k"][kv_start:kv_start + total].double(), st["v"][kv_start:kv_start + total].double()
        for lo in range(0, new, 512):
            hi = min(new, lo + 512)
            p = torch.arange(total - new + lo, total - new + hi, device="cuda")
            reach = 0 if not c["window"] else max(0, total - new + lo - c["window"] + 1)
            seen = torch.arange(reach, total - new + hi, device="cuda")
            if reach:
                seen = torch.cat([torch.arange(0, min(c["sinks"], reach), device="cuda"), seen])
            ok = seen[None] <= p[:, None]
            if c["window"]:
                ok &= (p[:, None] - seen[None] < c["window"]) | (seen[None] < c["sinks"])
            for h in range(hkv):
                kk, vv = keys[seen, h], values[seen, h]
                qq = st["q"][q_start + lo:q_start + hi, h * g:(h + 1) * g].double()
                logits = torch.einsum("tgd,sd->tgs", qq, kk) / d ** 0.5
                logits = torch.where(ok[:, None], logits, torch.full_like(logits, -torch.inf))
                w = torch.softmax(logits, -1)
                result[q_start + lo:q_start + hi, h * g:(h + 1) * g] = torch.einsum("tgs,sd->tgd", w, vv)
        q_start += new
        kv_start += total
    return result


def _exact_append(st):
    c = st["case"]
    hkv, d, block, half = c["kv_heads"], c["head_dim"], c["block"], c["rot"] // 2
    top = TOP[c["format"]]

    def turned(x, lo, n):
        z = x.double().clone()
        for i in range(half):
            a, b = (i, i + half) if c["style"] == 0 else (2 * i, 2 * i + 1)
            co, si = st["cos"][lo:lo + n, i].double()[:, None], st["sin"][lo:lo + n, i].double()[:, None]
            u, w = z[:, :, a].clone(), z[:, :, b].clone()
            z[:, :, a], z[:, :, b] = u * co - w * si, w * co + u * si
        return z

    def rounded(x):
        if c["format"] == "int8":
            return torch.round(x).clamp(-top, top)
        m = x.abs().clamp(max=top)  # e4m3: 3 bits after the leading one, the exponent not below -6
        step = torch.exp2(torch.floor(torch.log2(m.clamp(min=2.0 ** -6))) - 3)
        return torch.sign(x) * torch.round(m / step) * step

    qs, kept = [], {"k": [], "v": []}
    at = 0
    for b, (new, total) in enumerate(st["lengths"]):
        start = total - new
        qs.append(turned(st["q"][at:at + new], start, new))
        for name in ("k", "v"):
            x = st[name][at:at + new]
            x = turned(x, start, new) if name == "k" else x.double()
            lo = start // block * block
            n = -(-(total - lo) // block)
            fresh = torch.zeros(n * block, hkv, d, dtype=torch.float64, device="cuda")
            fresh[start - lo:total - lo] = x
            fresh = fresh.view(n, block, hkv, d)
            scale = fresh.abs().amax((1, 3)) / top
            if start > lo:
                codes, s = _exact_values(c, st, name, b, lo, start)
                scale[0] = torch.maximum(scale[0], s[0])
            part = torch.where(scale > 0, scale, torch.ones_like(scale))[:, None, :, None]
            y = rounded(fresh / part)
            if start > lo:
                y[0, :start - lo] = rounded(codes * (s[0] / part[0, 0, :, 0])[None, :, None])
            kept[name].append((y * scale[:, None, :, None]).reshape(n * block, hkv, d)[:total - lo])
        at += new
    return {"q": torch.cat(qs), "k": torch.cat(kept["k"]), "v": torch.cat(kept["v"])}
