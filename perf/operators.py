"""Cases of the decoder operators: rotary positions, the 8-bit paged key/value cache (append, gather) and the
attention that reads it.

A case is a dict of plain values. prepare(case, seed) makes what a serving or training program holds before the call;
run(state) is one pass, by elementary torch operations (own = False) or by the framework's entry points (own = True).
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_TYPES = {"f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # one step of 16 sequences: the 32 query and 8 key heads of a fused projection's rows, latency counts
        dict(name="rope_step", op="rope", type="f16", tokens=16, heads=40, more=8, dim=128, rot=128, pairs="half",
             base=10000.0, scaling="none", positions=4096, back=False),
        # prompts packed into one call, frequencies blended for contexts 32 times the trained length
        dict(name="rope_prompt", op="rope", type="f16", tokens=16384, heads=40, more=8, dim=128, rot=128, pairs="half",
             base=500000.0, scaling="ramp", positions=131072, back=False),
        # a training step's gradient, 32 bits, interleaved pairs in part of an 80-wide head, an odd token count
        dict(name="rope_gradient", op="rope", type="f32", tokens=24001, heads=12, more=0, dim=80, rot=32,
             pairs="interleaved", base=10000.0, scaling="linear", positions=8000, back=True),
        # one new token of each of 48 sequences: tail pages take one token and may have to be scaled again
        dict(name="append_step", op="append", type="f16", seqs=48, new_lo=1, new_hi=1, ctx_lo=0, ctx_hi=4000, heads=8,
             more=32, dim=128, page=16, layout="heads", sizes=1),
        # prompts of six sequences going into a cache laid out by tokens
        dict(name="append_prompt", op="append", type="f16", seqs=6, new_lo=700, new_hi=4000, ctx_lo=0, ctx_hi=2000,
             heads=8, more=32, dim=128, page=64, layout="tokens", sizes=2),
        # odd head counts and widths, 32-bit activations, a few to a few hundred tokens each
        dict(name="append_odd", op="append", type="f32", seqs=9, new_lo=1, new_hi=300, ctx_lo=0, ctx_hi=700, heads=5,
             more=5, dim=80, page=32, layout="heads", sizes=3),
        # one token of one sequence, the framework's own head layout (8 heads of 64, 256 positions): pure latency
        dict(name="attend_token", op="attend", type="f32", seqs=1, new_lo=1, new_hi=1, prompts=0, prompt_hi=1,
             len_lo=256, len_hi=256, idle=0, heads=8, kv_heads=8, dim=64, page=16, layout="heads", window=0, sizes=4),
        # a full serving batch of ragged lengths, some slots idle
        dict(name="attend_batch", op="attend", type="f16", seqs=64, new_lo=1, new_hi=1, prompts=0, prompt_hi=1,
             len_lo=1, len_hi=8192, idle=4, heads=32, kv_heads=8, dim=128, page=64, layout="heads", window=0, sizes=5),
        # two very long contexts, few rows
        dict(name="attend_long", op="attend", type="f16", seqs=2, new_lo=1, new_hi=1, prompts=0, prompt_hi=1,
             len_lo=150001, len_hi=200003, idle=0, heads=32, kv_heads=4, dim=128, page=16, layout="heads", window=0,
             sizes=6),
        # checking a few drafted tokens at a time, windowed, 32 bits, a 96-wide head, laid out by tokens
        dict(name="attend_check", op="attend", type="f32", seqs=24, new_lo=1, new_hi=6, prompts=0, prompt_hi=1,
             len_lo=20, len_hi=3000, idle=1, heads=24, kv_heads=8, dim=96, page=32, layout="tokens", window=1024,
             sizes=7),
        # prompts over cached prefixes: the largest products
        dict(name="attend_prompt", op="attend", type="f16", seqs=3, new_lo=1000, new_hi=2048, prompts=0, prompt_hi=1,
             len_lo=2048, len_hi=6144, idle=0, heads=32, kv_heads=8, dim=128, page=64, layout="heads", window=0,
             sizes=8),
        # two prompts among running sequences, eight query heads to a key head, 256-wide heads
        dict(name="attend_mixed", op="attend", type="f16", seqs=20, new_lo=1, new_hi=1, prompts=2, prompt_hi=700,
             len_lo=100, len_hi=4000, idle=1, heads=16, kv_heads=2, dim=256, page=128, layout="heads", window=0,
             sizes=9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend"])
    kind = rng.choice(["f16", "f16", "f32"])
    if op == "rope":
        dim = rng.choice([64, 72, 80, 96, 128, 192, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        heads = _log(rng, 1, 64)
        tokens = _log(rng, 1, 80_000_000 // (heads * dim * (2 if kind == "f32" else 1)) if heads * dim > 640 else 60000)
        return dict(op=op, type=kind, tokens=tokens, heads=heads, more=rng.choice([0, 0, 1, 8]), dim=dim,
                    rot=rot - rot % 2, pairs=rng.choice(["half", "interleaved"]),
                    base=rng.choice([10000.0, 500000.0, 1000000.0]), scaling=rng.choice(["none", "linear", "ramp"]),
                    positions=_log(rng, 16, 1000000), back=rng.random() < 0.4)
    if op == "append":
        heads, dim = _log(rng, 1, 16), 16 * rng.randint(2, 16)
        seqs = _log(rng, 1, 64)
        most = max(1, min(4000, 12_000_000 // (heads * dim * seqs)))
        hi = _log(rng, 1, most)
        return dict(op=op, type=kind, seqs=seqs, new_lo=rng.choice([1, hi]), new_hi=hi, ctx_lo=0,
                    ctx_hi=_log(rng, 1, 4000), heads=heads, more=rng.choice([0, 1, 16]), dim=dim,
                    page=rng.choice([16, 32, 64, 128, 256]), layout=rng.choice(["heads", "tokens"]),
                    sizes=rng.randint(1, 1 << 30))
    kv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 192, 256])
    what = rng.choice(["step", "step", "check", "prompt", "mixed"])
    seqs = _log(rng, 1, 64) if what in ("step", "check", "mixed") else _log(rng, 1, 4)
    len_hi = _log(rng, 16, max(16, min(200000, 200_000_000 // (seqs * kv * dim))))
    hi = {"step": 1, "check": rng.randint(2, 8), "prompt": _log(rng, 16, 2048), "mixed": 1}[what]
    prompts = rng.randint(1, 2) if what == "mixed" else 0
    rows = _log(rng, 16, 700) if what == "mixed" else 1
    while seqs * kv * group * max(hi, rows) * max(hi, rows, len_hi) > 800_000_000:
        len_hi, hi, rows = max(16, len_hi // 2), max(1, hi * 3 // 4), max(1, rows * 3 // 4)
    return dict(op=op, type=kind, seqs=seqs, new_lo=rng.choice([1, hi]), new_hi=hi, prompts=min(prompts, seqs),
                prompt_hi=rows, len_lo=1, len_hi=len_hi, idle=rng.choice([0, 0, 1]) if seqs > 1 else 0,
                heads=kv * group, kv_heads=kv, dim=dim, page=rng.choice([16, 32, 64, 128, 256]),
                layout=rng.choice(["heads", "tokens"]), window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]),
                sizes=rng.randint(1, 1 << 30))


def _append_sizes(case):
    """Of each sequence: tokens in the cache before, and new ones."""
    r = random.Random(case["sizes"])
    return [(r.randint(case["ctx_lo"], case["ctx_hi"]), r.randint(case["new_lo"], case["new_hi"]))
            for _ in range(case["seqs"])]


def _attend_sizes(case):
    """Of each sequence: tokens in the cache (the new ones among them), and new ones."""
    r = random.Random(case["sizes"])
    got = []
    for b in range(case["seqs"]):
        n = r.randint(case["new_lo"], case["new_hi"])
        if b < case["prompts"]:
            n = r.randint(max(1, case["prompt_hi"] // 2), case["prompt_hi"])
        length = max(n, r.randint(case["len_lo"], case["len_hi"]))
        got.append((length, n))
    for b in range(case["idle"]):  # a slot of a padded batch that holds no sequence: a row, and nothing to see
        got[case["seqs"] - 1 - b] = (0, 1)
    r.shuffle(got)
    return got


def _pages(tokens, page):
    return -(-tokens // page)


# ---------------------------------------------------------------- prepare ----

def _frequencies(case):
    """The angle a position turns each pair by, in radians, in 64 bits; and the factor on the result."""
    i = np.arange(case["rot"] // 2, dtype=np.float64)
    f = case["base"] ** (-2.0 * i / case["rot"])
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "ramp":  # fast pairs kept, slow ones divided by 32, a ramp between (4096 trained positions)
        at = lambda turns: case["rot"] * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(case["base"]))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), case["rot"] - 1)
        keep = 1.0 - np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        return f / 32.0 * (1.0 - keep) + f * keep, 0.1 * math.log(32.0) + 1.0
    return f, 1.0


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _values(shape, g):
    """int8 values as quantised activations have them: near a bell, up to the ends of the range."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 26):
        n = min(1 << 26, flat.numel() - at)
        flat[at:at + n] = (torch.randn(n, device="cuda", generator=g) * 36.0).clamp_(-127, 127).to(torch.int8)
    return out


def _pool(case, pages, g):
    """The cache: values as [page, head, token, dim] whatever the order in memory, and a scale of each page and head."""
    h, p, d = case.get("kv_heads", case["heads"]), case["page"], case["dim"]
    kv = []
    for _ in range(2):
        if case["layout"] == "tokens":
            kv.append(_values((pages, p, h, d), g).transpose(1, 2))
        else:
            kv.append(_values((pages, h, p, d), g))
    scales = [torch.rand(pages, h, device="cuda", generator=g) * 0.03 + 0.015 for _ in range(2)]
    return kv + scales


def _tables(lengths, page, spare, g):
    """Each sequence's pages in a random order over the pool; -1 where it has none."""
    need = [_pages(n, page) for n in lengths]
    order = torch.randperm(sum(need) + spare, device="cuda", generator=g).to(torch.int32)
    tables = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables


def _starts(news):
    return _i32(np.concatenate([[0], np.cumsum(news)]).astype(np.int32).tolist())


def prepare(case, seed):
    g = _generator(seed)
    dt = _TYPES[case["type"]]
    s = {"op": case["op"], "case": case}
    if case["op"] == "rope":
        t, h = case["tokens"], case["heads"]
        rows = torch.randn(t, h + case["more"], case["dim"], device="cuda", generator=g).to(dt)
        s["x"] = rows[:, :h]
        # runs of successive positions from random beginnings, as packed prompts have them
        run = max(1, t // 8)
        first = torch.randint(0, max(1, case["positions"] - run), (t // run + 1,), device="cuda", generator=g)
        at = torch.arange(t, device="cuda")
        s["pos"] = (first[at // run] + at % run).to(torch.int32)
        f, s["factor"] = _frequencies(case)
        s["phases"] = torch.from_numpy(np.rint(f / (2 * math.pi) * 2.0 ** 64).astype(np.int64)).cuda()
        return s
    if case["op"] == "append":
        sizes = _append_sizes(case)
        old, news = [c for c, _ in sizes], [n for _, n in sizes]
        lens = [c + n for c, n in sizes]
        t, h, p = sum(news), case["heads"], case["page"]
        s["pool"] = _pool(case, sum(_pages(n, p) for n in lens) + 8, g)
        s["tables"] = _tables(lens, p, 8, g)
        # a projection's rows: queries, keys, values
        rows = torch.randn(t, case["more"] + 2 * h, case["dim"], device="cuda", generator=g)
        rows *= torch.rand(t, 1, 1, device="cuda", generator=g) * 2.0 + 0.2
        rows = rows.to(dt)
        s["k"], s["v"] = rows[:, case["more"]:case["more"] + h], rows[:, case["more"] + h:]
        s["starts"], s["lens"] = _starts(news), _i32(lens)
        # what the call changes: the new positions, and the older ones of the page that the first of them falls in
        first = [c - c % p for c in old]
        s["seq"] = _i32(np.repeat(np.arange(len(lens)), [n - f for n, f in zip(lens, first)]).tolist())
        s["at"] = _i32(np.concatenate([np.arange(f, n) for n, f in zip(lens, first)]).tolist())
        return s
    sizes = _attend_sizes(case)
    lens, news = [n for n, _ in sizes], [n for _, n in sizes]
    s["pool"] = _pool(case, sum(_pages(n, case["page"]) for n in lens) + 4, g)
    s["tables"] = _tables(lens, case["page"], 4, g)
    s["q"] = torch.randn(sum(news), case["heads"], case["dim"], device="cuda", generator=g).to(dt)
    s["starts"], s["lens"], s["most"] = _starts(news), _i32(lens), max(news)
    s["scale"] = 1.0 / math.sqrt(case["dim"])
    s["work"] = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")  # the workspace such a program keeps
    return s


# -------------------------------------------------------------------- run ----

def run(state):
    if own:
        return _OWN[state["op"]](state)
    return _PLAIN[state["op"]](state)


def _plain_rope(s):
    c = s["case"]
    r = c["rot"]
    # the product of position and phase wraps at whole turns; its upper half is the turn's fraction, signed
    turns = (s["pos"].to(torch.int64)[:, None] * s["phases"][None, :]) >> 32
    angle = turns.to(torch.float32) * (2.0 * math.pi / 2.0 ** 32)
    cos, sin = (angle.cos() * s["factor"])[:, None, :], (angle.sin() * s["factor"])[:, None, :]
    if c["back"]:
        sin = -sin
    x = s["x"].to(torch.float32)
    out = x.clone()
    if c["pairs"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        out[..., :r // 2] = a * cos - b * sin
        out[..., r // 2:r] = b * cos + a * sin
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2] = a * cos - b * sin
        out[..., 1:r:2] = b * cos + a * sin
    return out.to(s["x"].dtype)


def _token_places(s, tokens):
    """Of each new token: its sequence, and its position."""
    at = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(s["starts"][1:].to(torch.int64), at, right=True)
    news = s["starts"][1:] - s["starts"][:-1]
    return seq, (s["lens"] - news)[seq] + at - s["starts"][seq]


def _quantised(x, scale):
    q = torch.round(x / scale)
    return torch.where(scale > 0, q, torch.zeros_like(q)).clamp(-127, 127).to(torch.int8)


def _plain_append_one(s, x, pool, scales, seq, at, page, slot):
    p = s["case"]["page"]
    x = x.to(torch.float32)
    pages, heads = scales.shape
    # the largest magnitude of the new values of each page and head
    most = torch.full((pages, heads), -1.0, device="cuda")
    most.scatter_reduce_(0, page[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    # the page that a sequence's older tokens end in keeps their scale where that is larger
    news = s["starts"][1:] - s["starts"][:-1]
    old = s["lens"] - news
    tail = s["tables"].gather(1, (old // p).clamp(max=s["tables"].shape[1] - 1).long()[:, None])[:, 0]
    kept = (old % p > 0) & (news > 0) & (tail >= 0)
    tail = tail[kept].long()
    filled = (old % p)[kept]
    before = scales[tail]
    now = torch.where(most >= 0, most * (1.0 / 127.0), scales)
    now[tail] = torch.maximum(now[tail], before)
    scales.copy_(now)
    ratio = torch.where(now[tail] > 0, before / now[tail], torch.zeros_like(before))
    again = torch.round(pool[tail].to(torch.float32) * ratio[:, :, None, None]).to(torch.int8)
    older = torch.arange(p, device="cuda")[None, :] < filled[:, None]
    pool[tail] = torch.where(older[:, None, :, None], again, pool[tail])
    pool[page, :, slot] = _quantised(x, now[page][:, :, None])


def _plain_gather(s, seq, at, pool, scales, dtype):
    p = s["case"]["page"]
    page = s["tables"][seq, at // p].long()
    return (pool[page, :, at % p].to(torch.float32) * scales[page][:, :, None]).to(dtype)


def _plain_append(s):
    k, v, ks, vs = s["pool"]
    seq, at = _token_places(s, s["k"].shape[0])
    page = s["tables"][seq, at // s["case"]["page"]].long()
    slot = at % s["case"]["page"]
    _plain_append_one(s, s["k"], k, ks, seq, at, page, slot)
    _plain_append_one(s, s["v"], v, vs, seq, at, page, slot)
    seq, at = s["seq"].long(), s["at"].long()
    return {"k": _plain_gather(s, seq, at, k, ks, s["k"].dtype), "v": _plain_gather(s, seq, at, v, vs, s["k"].dtype),
            "k_scale": ks, "v_scale": vs}


def _plain_attend(s):
    c = s["case"]
    k, v, ks, vs = s["pool"]
    q = s["q"].to(torch.float32)
    tokens, heads, d = q.shape
    hk, n, seqs = c["kv_heads"], s["most"], s["lens"].shape[0]
    group = heads // hk
    ids = s["tables"].clamp(min=0).long()
    length = ids.shape[1] * c["page"]
    # every sequence's keys and values, side by side and padded: [seq, kv head, position, dim]
    spread = lambda pool, scales: (pool[ids].to(torch.float32) * scales[ids][..., None, None]).transpose(1, 2).reshape(seqs, hk, length, d)  # noqa: E731
    news = s["starts"][1:] - s["starts"][:-1]
    row = (s["starts"][:-1, None] + torch.arange(n, device="cuda")[None, :]).clamp(max=tokens - 1).long()
    rows = q[row].view(seqs, n, hk, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hk, group * n, d)
    scores = torch.matmul(rows, spread(k, ks).transpose(2, 3)).mul_(s["scale"]).view(seqs, hk, group, n, length)
    at = torch.arange(length, device="cuda")[None, None, :]
    mine = ((s["lens"] - news)[:, None] + torch.arange(n, device="cuda")[None, :])[:, :, None]
    seen = (at <= mine) & (at < s["lens"][:, None, None])
    if c["window"]:
        seen &= at > mine - c["window"]
    seen = seen[:, None, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(seqs, hk, group * n, length), spread(v, vs)).view(seqs, hk, group, n, d)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    lse = torch.where(total > 0, top + total.log(), torch.full_like(top, -math.inf))
    seq, place = _token_places(s, tokens)
    j = (place - (s["lens"] - news)[seq]).long()
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, n, heads, d)[seq, j]
    lse = lse.permute(0, 3, 1, 2, 4).reshape(seqs, n, heads)[seq, j]
    return {"out": out.to(s["q"].dtype), "lse": lse}


_PLAIN = {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}

_decode = None


def _framework():
    global _decode
    if _decode is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "contract-stablehlo-mlx_b200"))
        from shlo import decode
        _decode = decode
    return _decode


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_rope(s):
    fw = _framework()
    c = s["case"]
    out = torch.empty(s["x"].shape, dtype=s["x"].dtype, device="cuda")
    fw.rope_noalloc(s["x"], s["pos"], s["phases"], out, interleaved=c["pairs"] == "interleaved", inverse=c["back"],
                    factor=s["factor"], stream=_stream())
    return out


def _own_append(s):
    fw = _framework()
    pool = fw.Pool(*s["pool"])
    fw.append_noalloc(pool, s["k"], s["v"], s["starts"], s["lens"], s["tables"], stream=_stream())
    n, dt = s["seq"].shape[0], s["k"].dtype
    shape = (n, s["case"]["heads"], s["case"]["dim"])
    k, v = torch.empty(shape, dtype=dt, device="cuda"), torch.empty(shape, dtype=dt, device="cuda")
    fw.gather_noalloc(pool, s["tables"], s["seq"], s["at"], k, v, stream=_stream())
    return {"k": k, "v": v, "k_scale": s["pool"][2], "v_scale": s["pool"][3]}


def _minetend(s):
    fw = _framework()
    q = s["q"]
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
    fw.attend_noalloc(fw.Pool(*s["pool"]), q, s["starts"], s["lens"], s["tables"], out, lse=lse, scale=s["scale"],
                      causal=True, window=s["case"]["window"], workspace=s["work"], stream=_stream())
    return {"out": out, "lse": lse}


_OWN = {"rope": _own_rope, "append": _own_append, "attend": _minetend}


# ------------------------------------------------------------ work, exact ----

def work(case):
    size = 2 if case["type"] == "f16" else 4
    if case["op"] == "rope":
        t, h, d, r = case["tokens"], case["heads"], case["dim"], case["rot"]
        return {"bytes": 2 * t * h * d * size + 4 * t + 8 * (r // 2), "flops": t * h * (r // 2) * 6}
    if case["op"] == "append":
        sizes = _append_sizes(case)
        h, d, p = case["heads"], case["dim"], case["page"]
        new = sum(n for _, n in sizes)
        tail = sum(c % p for c, n in sizes if n)  # older tokens of the pages that are written into
        pages = sum(_pages(c + n, p) - c // p for c, n in sizes)
        back = new + tail
        return {"bytes": 2 * h * d * (new * (size + 1) + tail) + 8 * h * pages + 2 * h * d * back * (1 + size),
                "flops": 2 * h * d * (3 * new + tail + back)}
    h, hk, d, w = case["heads"], case["kv_heads"], case["dim"], case["window"]
    keys = pairs = rows = 0
    for length, n in _attend_sizes(case):
        rows += n
        if length == 0:
            continue
        first = length - n
        low = max(0, first - w + 1) if w else 0
        keys += length - low
        for j in range(n):
            pairs += min(w, first + j + 1) if w else first + j + 1
    return {"bytes": 2 * keys * hk * d + 8 * hk * _pages(keys, case["page"]) + 2 * rows * h * d * size + 4 * rows * h,
            "flops": 4 * pairs * h * d}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, s)


def _exact_rope(case, s):
    f, factor = _frequencies(case)
    angle = s["pos"].double()[:, None] * torch.from_numpy(f).cuda()[None, :]
    turn = torch.polar(torch.full_like(angle, factor), -angle if case["back"] else angle)[:, None, :]
    x = s["x"].double()
    r, shape = case["rot"], x.shape
    if case["pairs"] == "half":
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
        y = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(x[..., :r].contiguous().view(shape[0], shape[1], r // 2, 2)) * turn
        y = torch.view_as_real(z).reshape(shape[0], shape[1], r)
    return torch.cat([y, x[..., r:]], -1)


def _exact_append(case, s):
    p = case["page"]
    k, v, ks, vs = s["pool"]
    starts, tables = s["starts"].tolist(), s["tables"].tolist()
    got = {}
    for name, x, pool, scales in (("k", s["k"], k, ks), ("v", s["v"], v, vs)):
        scales, x, parts = scales.double(), x.double(), []
        for b, length in enumerate(s["lens"].tolist()):
            n = starts[b + 1] - starts[b]
            at = length - n - (length - n) % p
            while n and at < length:
                page, old = tables[b][at // p], max(0, length - n - at)
                end = min(length, at + p)
                base = starts[b] + at + old - (length - n)
                new = x[base:base + end - at - old].transpose(0, 1)  # [head, token, dim]
                scale = new.abs().amax((1, 2)) / 127.0
                kept = torch.zeros(new.shape[0], 0, new.shape[2], dtype=torch.float64, device="cuda")
                if old:
                    scale = torch.maximum(scale, scales[page])
                    kept = torch.round(pool[page, :, :old].double() * (scales[page] / scale)[:, None, None])
                scales[page] = scale
                q = torch.cat([kept, torch.round(new / scale[:, None, None])], 1)
                parts.append((q * scale[:, None, None]).transpose(0, 1))
                at += p
        got[name], got[name + "_scale"] = torch.cat(parts), scales
    return got


def _exact_attend(case, s):
    if work(case)["flops"] > 2e12:
        return None
    p, w = case["page"], case["window"]
    k, v, ks, vs = s["pool"]
    q = s["q"].double()
    group = case["heads"] // case["kv_heads"]
    starts, out = s["starts"].tolist(), torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lens"].tolist()):
        n = starts[b + 1] - starts[b]
        if not n or not length:
            continue
        ids = s["tables"][b, :_pages(length, p)].long()
        place = torch.arange(length, device="cuda")
        mine = torch.arange(length - n, length, device="cuda")[:, None]
        hidden = place[None, :] > mine
        if w:
            hidden |= place[None, :] <= mine - w
        for h in range(case["kv_heads"]):
            keys = (k[ids, h].double() * ks[ids, h].double()[:, None, None]).reshape(-1, case["dim"])[:length]
            vals = (v[ids, h].double() * vs[ids, h].double()[:, None, None]).reshape(-1, case["dim"])[:length]
            for i in range(h * group, (h + 1) * group):
                z = (q[starts[b]:starts[b + 1], i] @ keys.T * s["scale"]).masked_fill(hidden, -math.inf)
                lse[starts[b]:starts[b + 1], i] = torch.logsumexp(z, 1)
                out[starts[b]:starts[b + 1], i] = torch.softmax(z, 1) @ vals
    return {"out": out, "lse": lse}
