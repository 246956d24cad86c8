"""Cases of the operators of a decoder in 8 bits and of its beam search: the norm of queries and keys for each head with
the position rotation in the same pass, the product of activations and weights in 8-bit integers, the selection over
beams and vocabulary, and the reordering of the paged cache that follows it.

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
        dict(name="norm_rope_step", op="norm_rope", type="f16", tokens=16, q_heads=32, k_heads=8, more=8, dim=128,
             rot=128, pairs="half", base=10000.0, positions=4096, back=False),
        # prompts packed into one call
        dict(name="norm_rope_prompt", op="norm_rope", type="f16", tokens=16384, q_heads=32, k_heads=8, more=8, dim=128,
             rot=128, pairs="half", base=500000.0, positions=131072, back=False),
        # a training step's gradients, 32 bits, interleaved pairs in part of an 80-wide head, an odd token count
        dict(name="norm_rope_gradient", op="norm_rope", type="f32", tokens=24001, q_heads=9, k_heads=3, more=3, dim=80,
             rot=32, pairs="interleaved", base=10000.0, positions=8000, back=True),
        # one token through the framework's own decoder's first projection (512 to 12 heads of 64): pure latency
        dict(name="linear8_token", op="linear8", type="f32", rows=1, n=512, m=768, bias=True),
        # one step of 24 sequences through a feed-forward's first projection: the weights' bytes
        dict(name="linear8_step", op="linear8", type="f16", rows=24, n=4096, m=12288, bias=False),
        # odd sizes, 32 bits: a short prompt
        dict(name="linear8_odd", op="linear8", type="f32", rows=333, n=1999, m=1001, bias=True),
        # packed prompts, the largest product
        dict(name="linear8_prompt", op="linear8", type="f16", rows=8192, n=4096, m=8192, bias=False),
        # one request, four beams, a small vocabulary: latency
        dict(name="beam_step", op="beam", type="f32", seqs=1, beams=4, keep=4, vocab=32001, masked=0.0, ended=0.0),
        # a full serving batch over a large vocabulary
        dict(name="beam_batch", op="beam", type="f16", seqs=64, beams=8, keep=8, vocab=128256, masked=0.0, ended=0.05),
        # wide beams, twice as many kept as there are beams, a grammar that masks most tokens
        dict(name="beam_wide", op="beam", type="f32", seqs=5, beams=32, keep=64, vocab=50257, masked=0.9, ended=0.1),
        # the same request's four beams go on: a page or two to copy
        dict(name="fork_step", op="fork", type="f32", seqs=1, beams=4, len_lo=200, len_hi=256, heads=8, dim=64, page=64,
             layout="heads", dead=0.0, sizes=1),
        # 64 requests of eight beams with long contexts, wide tables
        dict(name="fork_batch", op="fork", type="f16", seqs=64, beams=8, len_lo=100, len_hi=30000, heads=8, dim=128,
             page=128, layout="tokens", dead=0.02, sizes=2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope", "linear8", "linear8", "beam", "fork"])
    kind = rng.choice(["f16", "f16", "f32"])
    if op == "norm_rope":
        dim = rng.choice([64, 72, 80, 96, 128, 192, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        q_heads, k_heads = _log(rng, 1, 48), rng.choice([0, 1, 2, 4, 8, 16])
        back = rng.random() < 0.5
        most = 80_000_000 // ((q_heads + k_heads) * dim * (2 if kind == "f32" else 1) * (2 if back else 1))
        return dict(op=op, type=kind, tokens=_log(rng, 1, max(1, min(60000, most))), q_heads=q_heads, k_heads=k_heads,
                    more=rng.choice([0, 0, 1, 8]), dim=dim, rot=rot - rot % 2,
                    pairs=rng.choice(["half", "interleaved"]), base=rng.choice([10000.0, 500000.0, 1000000.0]),
                    positions=_log(rng, 16, 1000000), back=back)
    if op == "linear8":
        n, m = _log(rng, 16, 16384), _log(rng, 16, 65536)
        while n * m > 300_000_000:
            m //= 2
        most = min(8192, 250_000_000_000 // (n * m), 60_000_000 // max(n, m))
        return dict(op=op, type=kind, rows=_log(rng, 1, max(1, most)), n=n, m=m, bias=rng.random() < 0.5)
    if op == "beam":
        vocab, beams = _log(rng, 100, 200000), _log(rng, 1, 32)
        seqs = _log(rng, 1, max(1, min(64, 60_000_000 // (vocab * beams * (2 if kind == "f32" else 1)))))
        return dict(op=op, type=kind, seqs=seqs, beams=beams, keep=rng.choice([beams, beams, 2 * beams]), vocab=vocab,
                    masked=rng.choice([0.0, 0.0, 0.5, 0.99]), ended=rng.choice([0.0, 0.1]))
    heads, dim = _log(rng, 1, 16), 16 * rng.randint(2, 16)
    seqs, beams, page = _log(rng, 1, 64), _log(rng, 1, 16), rng.choice([16, 32, 64, 128, 256])
    while seqs * beams * page * heads * dim > 67_000_000:
        seqs, page = max(1, seqs // 2), max(16, page // 2)
    most = max(16, min(30000, 1_000_000_000 // (seqs * beams * heads * dim)))
    return dict(op=op, type=kind, seqs=seqs, beams=beams, len_lo=1, len_hi=_log(rng, 1, most), heads=heads, dim=dim,
                page=page, layout=rng.choice(["heads", "tokens"]), dead=rng.choice([0.0, 0.1]),
                sizes=rng.randint(1, 1 << 30))


def _fork_sizes(case):
    """Of each sequence its length, the same for all of its beams; of each new row the row that it continues, or -1."""
    r = random.Random(case["sizes"])
    lens = [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["seqs"])]
    parents = []
    for s in range(case["seqs"]):
        for _ in range(case["beams"]):  # the better beams have more children
            b = min(r.randrange(case["beams"]), r.randrange(case["beams"]))
            parents.append(-1 if r.random() < case["dead"] else s * case["beams"] + b)
    return lens, parents


# ---------------------------------------------------------------- prepare ----

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _int8(shape, g):
    """8-bit values near a bell, up to the ends of the range."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 26):
        n = min(1 << 26, flat.numel() - at)
        flat[at:at + n] = (torch.randn(n, device="cuda", generator=g) * 36.0).clamp_(-127, 127).to(torch.int8)
    return out


def prepare(case, seed):
    g = _generator(seed)
    s = {"op": case["op"], "case": case}
    {"norm_rope": _prepare_norm_rope, "linear8": _prepare_linear8, "beam": _prepare_beam, "fork": _prepare_fork}[
        case["op"]](s, case, g, _TYPES[case["type"]])
    return s


def _prepare_norm_rope(s, case, g, dt):
    t, h, d = case["tokens"], case["q_heads"] + case["k_heads"], case["dim"]
    # a projection's rows: queries, keys, and the values that the call leaves alone
    rows = torch.randn(t, h + case["more"], d, device="cuda", generator=g)
    rows *= torch.rand(t, 1, 1, device="cuda", generator=g) * 3.0 + 0.1
    s["x"] = rows.to(dt)[:, :h]
    # runs of successive positions from random beginnings, as packed prompts have them
    run = max(1, t // 8)
    first = torch.randint(0, max(1, case["positions"] - run), (t // run + 1,), device="cuda", generator=g)
    at = torch.arange(t, device="cuda")
    s["pos"] = (first[at // run] + at % run).to(torch.int32)
    f = case["base"] ** (-2.0 * np.arange(case["rot"] // 2, dtype=np.float64) / case["rot"])
    s["phases"] = torch.from_numpy(np.rint(f / (2 * math.pi) * 2.0 ** 64).astype(np.int64)).cuda()
    s["wq"] = (1.0 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(dt)
    s["wk"] = (1.0 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(dt)
    s["eps"], s["factor"] = 1e-6, 1.0
    if case["back"]:
        s["dy"] = (torch.randn(t, h, d, device="cuda", generator=g) * 0.1).to(dt)
        s["work"] = torch.zeros(32 << 20, dtype=torch.uint8, device="cuda")


def _prepare_linear8(s, case, g, dt):
    r, n, m = case["rows"], case["n"], case["m"]
    x = torch.randn(r, n, device="cuda", generator=g)
    # some channels of a decoder's activations are tens of times larger than the rest
    x *= 1.0 + 20.0 * (torch.rand(n, device="cuda", generator=g) < 0.003)
    x *= torch.rand(r, 1, device="cuda", generator=g) * 2.0 + 0.2
    s["x"] = x.to(dt)
    pad = -(-n // 16) * 16  # rows of weights begin on 16-byte boundaries
    s["w"] = _int8((m, pad), g)[:, :n]
    s["w_scale"] = (torch.rand(m, device="cuda", generator=g) + 0.5) * (1.0 / (36.0 * math.sqrt(n)))
    s["bias"] = torch.randn(m, device="cuda", generator=g) if case["bias"] else None
    s["work"] = torch.zeros(max(1 << 20, r * (pad + 256)), dtype=torch.uint8, device="cuda")


def _prepare_beam(s, case, g, dt):
    n, b, v = case["seqs"], case["beams"], case["vocab"]
    z = torch.randn(n * b, v, device="cuda", generator=g)
    z *= torch.rand(n * b, 1, device="cuda", generator=g) * 2.0 + 1.0  # from nearly flat to peaked
    if case["masked"]:
        z.masked_fill_(torch.rand(n * b, v, device="cuda", generator=g) < case["masked"], -math.inf)
    s["z"] = z.to(dt)
    # the beams' scores so far, a few units apart
    s["scores"] = -20.0 - torch.rand(n, b, device="cuda", generator=g) * 4.0 - torch.rand(n, 1, device="cuda", generator=g) * 40.0
    s["ended"] = (torch.rand(n, b, device="cuda", generator=g) < case["ended"]).to(torch.int32)
    s["end"] = 2
    s["work"] = torch.zeros(32 << 20, dtype=torch.uint8, device="cuda")


def _prepare_fork(s, case, g, dt):
    lens, parents = _fork_sizes(case)
    p, h, d, b = case["page"], case["heads"], case["dim"], case["beams"]
    rows = len(lens) * b
    # beams of a sequence share the pages that are full; each has its own last one
    full = [n // p for n in lens]
    part = [1 if n % p else 0 for n in lens]
    width = max(f + q for f, q in zip(full, part)) + 1
    pages = sum(full) + b * sum(part) + rows
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).cpu().numpy()
    tables = np.full((rows, width), -1, np.int32)
    at = 0
    for i in range(len(lens)):
        tables[i * b:(i + 1) * b, :full[i]] = order[at:at + full[i]]
        at += full[i]
        if part[i]:
            tables[i * b:(i + 1) * b, full[i]] = order[at:at + b]
            at += b
    s["tables"] = torch.from_numpy(tables).cuda()
    s["fresh"] = torch.from_numpy(order[at:at + rows].copy()).cuda()
    s["lens"] = _i32(np.repeat(lens, b).tolist())
    s["parents"] = _i32(parents)
    shape = (pages, h, p, d) if case["layout"] == "heads" else (pages, p, h, d)
    kv = [_int8(shape, g) for _ in range(2)]
    if case["layout"] == "tokens":
        kv = [x.transpose(1, 2) for x in kv]
    s["pool"] = kv + [torch.rand(pages, h, device="cuda", generator=g) * 0.03 + 0.015 for _ in range(2)]
    # what the call may copy: each new row's tokens in a page that is not full
    seq = [(r, lens[r // b]) for r in range(rows) if parents[r] >= 0]
    s["seq"] = _i32(np.repeat([r for r, _ in seq], [n % p for _, n in seq]).astype(np.int32).tolist())
    s["at"] = _i32(np.concatenate([np.arange(n - n % p, n) for _, n in seq] + [[]]).astype(np.int32).tolist())
    s["dt"] = dt


# -------------------------------------------------------------------- run ----

def run(state):
    if own:
        return _OWN[state["op"]](state)
    return _PLAIN[state["op"]](state)


def _plain_norm_rope(s):
    c = s["case"]
    r, hq = c["rot"], c["q_heads"]
    # the product of position and phase wraps at whole turns; its upper half is the turn's fraction, signed
    turns = (s["pos"].to(torch.int64)[:, None] * s["phases"][None, :]) >> 32
    angle = turns.to(torch.float32) * (2.0 * math.pi / 2.0 ** 32)
    cos, sin = (angle.cos() * s["factor"])[:, None, :], (angle.sin() * s["factor"])[:, None, :]
    if c["pairs"] == "half":
        ia, ib = slice(0, r // 2), slice(r // 2, r)
    else:
        ia, ib = slice(0, r, 2), slice(1, r, 2)
    x = s["x"].to(torch.float32)
    w = torch.cat([s["wq"].to(torch.float32).expand(hq, -1), s["wk"].to(torch.float32).expand(c["k_heads"], -1)])
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"])
    if not c["back"]:
        z = x * inv * w
        y = z.clone()
        a, b = z[..., ia], z[..., ib]
        y[..., ia] = a * cos - b * sin
        y[..., ib] = b * cos + a * sin
        return y.to(s["x"].dtype)
    dy = s["dy"].to(torch.float32)
    dz = dy.clone()
    a, b = dy[..., ia], dy[..., ib]
    dz[..., ia] = a * cos + b * sin
    dz[..., ib] = b * cos - a * sin
    n = x * inv
    dw = (dz * n).sum(0, dtype=torch.float64)
    dn = dz * w
    dx = (dn - n * (dn * n).mean(-1, keepdim=True)) * inv
    return {"dx": dx.to(s["x"].dtype), "dwq": dw[:hq].sum(0).to(torch.float32), "dwk": dw[hq:].sum(0).to(torch.float32)}


def _plain_linear8(s):
    n = s["x"].shape[1]
    # (64 bits: a value next to a border between two steps goes to the right one)
    x = s["x"].to(torch.float64)
    top = x.abs().amax(1, keepdim=True)
    q = torch.round(x * 127.0 / torch.where(top > 0, top, torch.ones_like(top))).to(torch.float32)
    w = s["w"].to(torch.float32)
    # 1024 products of 7 by 7 bits: sums that 24 bits hold
    acc = torch.zeros(q.shape[0], w.shape[0], dtype=torch.int32, device="cuda")
    for at in range(0, n, 1024):
        acc += torch.matmul(q[:, at:at + 1024], w[:, at:at + 1024].T).to(torch.int32)
    y = acc.to(torch.float32) * (top / 127.0).to(torch.float32) * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _ordered(z):
    """Whole numbers in the order of 32-bit floats, -0 and 0 alike."""
    bits = (z.to(torch.float32) + 0.0).view(torch.int32)
    return torch.where(bits < 0, bits ^ 0x7fffffff, bits).to(torch.int64)


def _plain_beam(s):
    c = s["case"]
    n, b, v = c["seqs"], c["beams"], c["vocab"]
    k = min(c["keep"], v)
    # (64 bits: candidates of two beams may lie closer together than a 32-bit sum keeps)
    z = s["z"].to(torch.float64)
    top = z.amax(1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    lse = top + (z - top).exp_().sum(1, keepdim=True).log()
    del z
    keys = (_ordered(s["z"]) << 32) + (2 ** 32 - 1 - torch.arange(v, device="cuda"))
    token = 2 ** 32 - 1 - (keys.topk(k, 1).values & (2 ** 32 - 1))
    del keys
    gain = s["z"].gather(1, token).to(torch.float64) - lse
    ended = (s["ended"] != 0).view(n * b, 1)
    gain = torch.where(ended, torch.where(torch.arange(k, device="cuda") == 0, 0.0, -math.inf).to(torch.float64), gain)
    token = torch.where(ended, torch.full_like(token, s["end"]), token)
    total = s["scores"].to(torch.float64).view(n * b, 1) + gain
    total = torch.where(total.isnan(), torch.full_like(total, -math.inf), total).view(n, b * k)
    if total.shape[1] < c["keep"]:
        total = torch.cat([total, torch.full((n, c["keep"] - b * k), -math.inf, dtype=torch.float64, device="cuda")], 1)
    total, at = total.sort(dim=1, descending=True, stable=True)
    total, at = total[:, :c["keep"]], at[:, :c["keep"]].clamp(max=b * k - 1)
    none = total == -math.inf
    parent = torch.arange(n, device="cuda")[:, None] * b + at // k
    token = token.view(n, b * k).gather(1, at)
    return {"scores": total.to(torch.float32), "parents": parent.masked_fill(none, -1).to(torch.int32),
            "tokens": token.masked_fill(none, -1).to(torch.int32)}


def _plain_fork(s):
    p = s["case"]["page"]
    k, v, ks, vs = s["pool"]
    parents = s["parents"].long()
    live, parent = parents >= 0, parents.clamp(min=0)
    lens = torch.where(live, s["lens"][parent], torch.zeros_like(s["lens"]))
    last = (lens // p).long()
    tables = s["tables"][parent]
    width = torch.arange(tables.shape[1], device="cuda")
    tables = torch.where(width[None, :] < ((lens + p - 1) // p)[:, None], tables, torch.full_like(tables, -1))
    # all but the first of a row's continuations need a copy of its last page, where that is not full
    again = torch.ones(len(parents), len(parents), device="cuda").tril(-1).bool() & (parents[:, None] == parents[None, :])
    copied = (again.any(1) & live & (lens % p > 0)).nonzero()[:, 0]
    old, new = tables[copied, last[copied]].long(), s["fresh"][copied].long()
    filled = torch.arange(p, device="cuda")[None, :] < (lens[copied] % p)[:, None]
    for x, scale in ((k, ks), (v, vs)):
        x[new] = torch.where(filled[:, None, :, None], x[old], x[new])
        scale[new] = scale[old]
    tables[copied, last[copied]] = new.to(torch.int32)
    seq, at = s["seq"].long(), s["at"].long()
    page = tables[seq, at // p].long()
    got = [(x[page, :, at % p].to(torch.float32) * scale[page][:, :, None]).to(s["dt"]) for x, scale in ((k, ks), (v, vs))]
    return {"tables": tables, "lens": lens, "k": got[0], "v": got[1]}


_PLAIN = {"norm_rope": _plain_norm_rope, "linear8": _plain_linear8, "beam": _plain_beam, "fork": _plain_fork}

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


def _own_norm_rope(s):
    fw, c, x = _framework(), s["case"], s["x"]
    dx = torch.empty(x.shape, dtype=x.dtype, device="cuda")
    inter = c["pairs"] == "interleaved"
    if not c["back"]:
        fw.norm_rope_noalloc(x, s["pos"], s["phases"], dx, q_heads=c["q_heads"], q_weight=s["wq"], k_weight=s["wk"],
                             eps=s["eps"], interleaved=inter, factor=s["factor"], stream=_stream())
        return dx
    dw = torch.empty(2, c["dim"], dtype=torch.float32, device="cuda")
    fw.norm_rope_grad_noalloc(x, s["dy"], s["pos"], s["phases"], dx, dw[0], dw[1], q_heads=c["q_heads"],
                              q_weight=s["wq"], k_weight=s["wk"], workspace=s["work"], eps=s["eps"], interleaved=inter,
                              factor=s["factor"], stream=_stream())
    return {"dx": dx, "dwq": dw[0], "dwk": dw[1]}


def _own_linear8(s):
    fw, x = _framework(), s["x"]
    y = torch.empty(x.shape[0], s["w"].shape[0], dtype=x.dtype, device="cuda")
    fw.linear8_noalloc(x, s["w"], s["w_scale"], y, bias=s["bias"], workspace=s["work"], stream=_stream())
    return y


def _own_beam(s):
    fw, c = _framework(), s["case"]
    shape = (c["seqs"], c["keep"])
    scores = torch.empty(shape, dtype=torch.float32, device="cuda")
    parents = torch.empty(shape, dtype=torch.int32, device="cuda")
    tokens = torch.empty(shape, dtype=torch.int32, device="cuda")
    fw.beam_select_noalloc(s["z"], s["scores"], scores, parents, tokens, ended=s["ended"], end_token=s["end"],
                           workspace=s["work"], stream=_stream())
    return {"scores": scores, "parents": parents, "tokens": tokens}


def _own_fork(s):
    fw, c = _framework(), s["case"]
    pool = fw.Pool(*s["pool"])
    tables, lens = torch.empty_like(s["tables"]), torch.empty_like(s["lens"])
    fw.fork_noalloc(pool, s["tables"], s["lens"], s["parents"], s["fresh"], tables, lens, stream=_stream())
    shape = (s["seq"].shape[0], c["heads"], c["dim"])
    k, v = torch.empty(shape, dtype=s["dt"], device="cuda"), torch.empty(shape, dtype=s["dt"], device="cuda")
    fw.gather_noalloc(pool, tables, s["seq"], s["at"], k, v, stream=_stream())
    return {"tables": tables, "lens": lens, "k": k, "v": v}


_OWN = {"norm_rope": _own_norm_rope, "linear8": _own_linear8, "beam": _own_beam, "fork": _own_fork}


# ------------------------------------------------------------ work, exact ----

def work(case):
    size = 2 if case["type"] == "f16" else 4
    if case["op"] == "norm_rope":
        t, h, d, r = case["tokens"], case["q_heads"] + case["k_heads"], case["dim"], case["rot"]
        if case["back"]:
            return {"bytes": 3 * t * h * d * size + 4 * t + 8 * (r // 2) + 2 * d * (size + 4), "flops": t * h * (12 * d + 3 * r)}
        return {"bytes": 2 * t * h * d * size + 4 * t + 8 * (r // 2) + 2 * d * size, "flops": t * h * (4 * d + 3 * r)}
    if case["op"] == "linear8":
        r, n, m = case["rows"], case["n"], case["m"]
        return {"bytes": r * n * size + m * n + 4 * m * (2 if case["bias"] else 1) + r * m * size, "flops": 2 * r * n * m}
    if case["op"] == "beam":
        rows = case["seqs"] * case["beams"]
        live = rows * (1.0 - case["ended"])
        return {"bytes": int(live * case["vocab"] * size) + 8 * rows + 12 * case["seqs"] * case["keep"],
                "flops": int(live * case["vocab"] * 4)}
    lens, parents = _fork_sizes(case)
    p, token = case["page"], case["heads"] * case["dim"]
    rows, seen, copied, read = len(parents), set(), 0, 0
    for r in parents:
        if r < 0:
            continue
        tail = lens[r // case["beams"]] % p
        read += tail
        if r in seen:
            copied += tail
        seen.add(r)
    pages = sum(-(-lens[r // case["beams"]] // p) for r in parents if r >= 0)
    return {"bytes": 4 * token * copied + 2 * token * read * (1 + size) + 4 * (2 * pages + 4 * rows) + 8 * read,
            "flops": 2 * token * read}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "linear8": _exact_linear8, "beam": _exact_beam, "fork": _exact_fork}[
        case["op"]](case, s)


def _exact_norm_rope(case, s):
    r, hq = case["rot"], case["q_heads"]
    f = case["base"] ** (-2.0 * np.arange(r // 2, dtype=np.float64) / r)
    angle = s["pos"].double()[:, None] * torch.from_numpy(f).cuda()[None, :]
    dx, dws = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda"), []

    def turned(x, turn):
        shape = x.shape
        if case["pairs"] == "half":
            z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
            y = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(x[..., :r].contiguous().view(shape[0], shape[1], r // 2, 2)) * turn
            y = torch.view_as_real(z).reshape(shape[0], shape[1], r)
        return torch.cat([y, x[..., r:]], -1)

    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)[:, None, :]
    for lo, hi, w in ((0, hq, s["wq"].double()), (hq, hq + case["k_heads"], s["wk"].double())):
        x = s["x"][:, lo:hi].double()
        rms = ((x ** 2).sum(-1, keepdim=True) / case["dim"] + s["eps"]).sqrt()
        if not case["back"]:
            dx[:, lo:hi] = turned(x / rms * w, turn)
            continue
        dz = turned(s["dy"][:, lo:hi].double(), turn.conj())
        dws.append((dz * x / rms).sum((0, 1)))
        # d(x_i / rms) / d x_j = (delta_ij - x_i x_j / (dim rms^2)) / rms
        g = dz * w
        dx[:, lo:hi] = g / rms - x * (g * x).sum(-1, keepdim=True) / (case["dim"] * rms ** 3)
    return {"dx": dx, "dwq": dws[0], "dwk": dws[1]} if case["back"] else dx


def _exact_linear8(case, s):
    x = s["x"].double()
    top = x.abs().amax(1, keepdim=True)
    # the nearest whole number to 127 |x| / top, of two equally near ones the even one, by exact comparisons
    safe = torch.where(top > 0, top, torch.ones_like(top))
    q = (127.0 * x.abs() / safe).floor()
    more, half = 254.0 * x.abs() - (2.0 * q + 1.0) * safe, q % 2 == 1
    q = torch.where((more > 0) | ((more == 0) & half), q + 1.0, q) * x.sign()
    y = torch.empty(x.shape[0], s["w"].shape[0], dtype=torch.float64, device="cuda")
    for at in range(0, y.shape[1], 8192):
        y[:, at:at + 8192] = q @ s["w"][at:at + 8192].double().T
    y *= top / 127.0
    y *= s["w_scale"].double()
    return y + s["bias"].double() if case["bias"] else y


def _exact_beam(case, s):
    n, b, k = case["seqs"], case["beams"], case["keep"]
    out = {"scores": torch.full((n, k), -math.inf, dtype=torch.float64, device="cuda"),
           "parents": torch.full((n, k), -1, dtype=torch.int32, device="cuda"),
           "tokens": torch.full((n, k), -1, dtype=torch.int32, device="cuda")}
    for i in range(n):
        z = s["z"][i * b:(i + 1) * b].double()
        total = torch.log_softmax(z, 1) + s["scores"][i].double()[:, None]
        ended = (s["ended"][i] != 0)[:, None]
        only = torch.arange(case["vocab"], device="cuda")[None, :] == s["end"]
        total = torch.where(ended, torch.where(only, s["scores"][i].double()[:, None], -math.inf), total).view(-1)
        total = torch.where(total.isnan(), -math.inf, total)
        # everything at least as good as the k-th, in order of index, then by value
        at = (total >= total.topk(min(k, total.numel())).values[-1]).nonzero()[:, 0]
        best, order = total[at].sort(descending=True, stable=True)
        best, at = best[:k], at[order][:k]
        keep = int((best > -math.inf).sum())
        out["scores"][i, :keep] = best[:keep]
        out["parents"][i, :keep] = (at[:keep] // case["vocab"] + i * b).to(torch.int32)
        out["tokens"][i, :keep] = (at[:keep] % case["vocab"]).to(torch.int32)
    return out


def _exact_fork(case, s):
    k, v, ks, vs = s["pool"]
    p, width = case["page"], s["tables"].shape[1]
    old, lens, fresh = s["tables"].cpu().numpy(), s["lens"].tolist(), s["fresh"].tolist()
    tables, news, source, seen = np.full((len(fresh), width), -1, np.int32), [], [], set()
    for r, parent in enumerate(s["parents"].tolist()):
        n = lens[parent] if parent >= 0 else 0
        news.append(n)
        pages = -(-n // p)
        if n:
            tables[r, :pages] = old[parent, :pages]
        source.append(int(old[parent, n // p]) if n % p else -1)
        if n % p and parent in seen:
            tables[r, n // p] = fresh[r]
        seen.add(parent)
    page = torch.tensor(source, device="cuda")[s["seq"].long()]
    at = s["at"].long() % p
    return {"tables": torch.from_numpy(tables).cuda(), "lens": _i32(news),
            "k": k[page, :, at].double() * ks[page][:, :, None].double(),
            "v": v[page, :, at].double() * vs[page][:, :, None].double()}
