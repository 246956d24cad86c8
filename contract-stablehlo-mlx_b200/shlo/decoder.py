"""A causal transformer that generates step by step: the denoiser's encoder layer (the
framework's norm, mul_mat and gelu_erf kernels) with rotary positions and an attention
over a paged cache in 8 bits in place of the attention over whole sequences.

    m = Decoder(Config(), pages=256)
    a = m.start(prompt)            # a sequence; its prompt, embedded [n, d]
    y = m.step([(a, x), (b, x2)])  # new tokens of several sequences at once -> their outputs, in order
    m.stop(a)                      # its pages may be used again

    m = Decoder(Config(norm_heads=True, bits8=True, vocab=1000), pages=256)
    best = m.search([5, 17, 3], beams=4, steps=20, end=2)  # [(score, tokens)], the best first

norm_heads: queries and keys are normed for each head, with the rotation. bits8: weights
in 8 bits, and activations rounded to 8 bits for each product. vocab: an embedding and an
output over a vocabulary, for search().

Everything a step computes stays on the device; the host keeps which pages a sequence
has. Weights are random (N(0, 0.02), norm gains 1 + N(0, 0.02)), from a seed.
"""
from __future__ import annotations

from dataclasses import dataclass
from types import MappingProxyType

import numpy as np

from . import decode as D
from . import mlx as M
from . import run as Run
from ._lib import ShloError
from .denoiser import EPS_BITS


@dataclass(frozen=True)
class Config:
    layers: int = 2
    d: int = 512
    heads: int = 8
    kv_heads: int = 2
    ffn: int = 2048
    page_tokens: int = 64
    base: float = 10000.0
    window: int = 0
    norm_heads: bool = False
    bits8: bool = False
    vocab: int = 0

    @property
    def dh(self) -> int:
        return self.d // self.heads


def init_weights(cfg: Config, seed: int = 1) -> dict:
    rng = np.random.default_rng(seed)
    out = {}
    qkv = (cfg.heads + 2 * cfg.kv_heads) * cfg.dh
    for li in range(cfg.layers):
        for name, shape in (("g1", (cfg.d,)), ("b1", (cfg.d,)), ("wqkv", (qkv, cfg.d)), ("cqkv", (qkv,)),
                            ("wo", (cfg.d, cfg.d)), ("co", (cfg.d,)), ("g2", (cfg.d,)), ("b2", (cfg.d,)),
                            ("w1", (cfg.ffn, cfg.d)), ("c1", (cfg.ffn,)), ("w2", (cfg.d, cfg.ffn)), ("c2", (cfg.d,))):
            v = rng.standard_normal(shape) * 0.02
            out["l%d_%s" % (li, name)] = (v + 1.0 if name in ("g1", "g2") else v).astype(np.float32)
    if cfg.norm_heads:
        for li in range(cfg.layers):
            for name in ("gq", "gk"):
                out["l%d_%s" % (li, name)] = (rng.standard_normal(cfg.dh) * 0.02 + 1.0).astype(np.float32)
    if cfg.vocab:
        out["embed"] = rng.standard_normal((cfg.vocab, cfg.d)).astype(np.float32)
        out["head"] = (rng.standard_normal((cfg.vocab, cfg.d)) * 0.1).astype(np.float32)
        out["chead"] = np.zeros(cfg.vocab, np.float32)
    return out


class Sequence:
    """A running sequence: its length and its pages."""

    __slots__ = ("tokens", "pages")

    def __init__(self):
        self.tokens, self.pages = 0, []


class Decoder:
    shared = MappingProxyType({})  # page -> sequences that hold it beside the first

    def __init__(self, cfg: Config, pages: int, weights: dict | None = None):
        self.cfg = cfg
        weights = weights or init_weights(cfg)
        self.embed = weights.get("embed")  # (rows of it go to the device as they are needed)
        self.w = {k: M.of_numpy(v) for k, v in weights.items() if k != "embed"}
        if cfg.bits8:
            for k in [k for k, v in weights.items() if k != "embed" and v.ndim == 2]:
                self.w[k] = D.quantise_rows(self.w[k])
        phases, self.factor = D.rope_phases(cfg.dh, cfg.base)
        self.phases = M.of_numpy(phases)
        self.caches = [D.Cache(pages, cfg.kv_heads, cfg.dh, cfg.page_tokens) for _ in range(cfg.layers)]
        self.free = list(range(pages))[::-1]
        self.shared = {}

    def start(self, prompt: np.ndarray):
        """(a new sequence, the outputs of its prompt [n, d])."""
        s = Sequence()
        return s, self.step([(s, prompt)])

    def stop(self, s: Sequence) -> None:
        for p in s.pages[::-1]:
            if self.shared.get(p):
                self.shared[p] -= 1
            else:
                self.free.append(p)
        s.tokens, s.pages = 0, []

    def fork(self, rows, parents):
        """New sequences, number i going on from rows[parents[i]] as it is now; the rows themselves stop. Full pages are
        shared; a last page that is not full is copied for all but the first that go on from its owner."""
        if len({id(s) for s in rows}) != len(rows):
            raise ShloError("decoder: a sequence named twice in one fork")
        for p in parents:
            if not 0 <= p < len(rows):
                raise ShloError("decoder: a parent %d of %d rows" % (p, len(rows)))
        page = self.cfg.page_tokens
        seen, copied = set(), []
        for i, p in enumerate(parents):
            copied.append(p in seen and rows[p].tokens % page > 0)
            seen.add(p)
        if sum(copied) > len(self.free):
            raise ShloError("decoder: %d pages needed, %d free" % (sum(copied), len(self.free)))
        take = iter(self.free[::-1])
        fresh = [next(take) if c else -1 for c in copied]
        width = max([len(s.pages) for s in rows] + [1])
        tables = np.array([s.pages + [-1] * (width - len(s.pages)) for s in rows], np.int32)
        batch = [M.of_numpy(np.asarray(a, np.int32)) for a in (tables, [s.tokens for s in rows], parents, fresh)]
        for cache in self.caches:
            cache.fork(*batch)
        del self.free[len(self.free) - sum(copied):]
        out = []
        for p, f, c in zip(parents, fresh, copied):
            s = Sequence()
            s.tokens, s.pages = rows[p].tokens, rows[p].pages[:-1] + [f] if c else list(rows[p].pages)
            for q in s.pages[:-1] if c else s.pages:
                self.shared[q] = self.shared.get(q, 0) + 1
            out.append(s)
        for s in rows:
            self.stop(s)
        return out

    def search(self, prompt, beams: int, steps: int, end: int = -1):
        """The `beams` best continuations of a prompt (token numbers) by `steps` tokens, or up to the token `end`: a list
        of (logarithm of their probability, tokens), the best first."""
        cfg = self.cfg
        if not cfg.vocab:
            raise ShloError("decoder: search needs a vocabulary")
        if len(prompt) == 0 or not all(0 <= t < cfg.vocab for t in prompt):
            raise ShloError("decoder: a prompt is one token or more of a vocabulary of %d" % cfg.vocab)
        s, y = self.start(self.embed[np.asarray(prompt)])
        rows, texts, scores, y = [s], [[]], np.zeros((1, 1), np.float32), y[-1:]
        ended = np.zeros((1, 1), np.int32)
        try:
            for left in range(steps, 0, -1):
                z = self._dense(M.of_numpy(np.ascontiguousarray(y)), "head", "chead", cfg.vocab, cfg.d, len(rows))
                got = D.beam_select(M.reshape(z, [len(rows), cfg.vocab]), M.of_numpy(scores), beams, ended=M.of_numpy(ended),
                                    end_token=end)
                scores, parents, tokens = (M.to_numpy(a) for a in got)
                live = [(int(p), int(t)) for p, t in zip(parents[0], tokens[0]) if p >= 0]  # (a vocabulary may be smaller)
                over = [bool(ended[0, p]) for p, _ in live]
                texts = [texts[p] if o else texts[p] + [t] for (p, t), o in zip(live, over)]
                scores = np.ascontiguousarray(scores[:, :len(live)])
                ended = np.array([[o or t == end for (_, t), o in zip(live, over)]], np.int32)
                if ended.all() or left == 1:  # (no page is taken for what nobody reads)
                    break
                rows = self.fork(rows, [p for p, _ in live])
                # (a beam that has ended takes its token again: nothing reads what follows)
                y = self.step([(r, self.embed[[max(t, 0)]]) for r, (_, t) in zip(rows, live)])
        finally:
            for r in rows:
                self.stop(r)
        return [(float(a), t) for a, t in zip(scores[0], texts)]

    def step(self, news) -> np.ndarray:
        """New tokens [n, d] of each (sequence, tokens) in turn -> their outputs [all, d]. A sequence is named once
        a step: its tokens of one step are one run of positions. A step that fails leaves every sequence's length
        and pages as they were (rounded again, at most, in the page that its last tokens share with the new ones)."""
        cfg = self.cfg
        news = [(s, np.asarray(x, np.float32)) for s, x in news]
        if len({id(s) for s, _ in news}) != len(news):
            raise ShloError("decoder: a sequence named twice in one step")
        t = sum(len(x) for _, x in news)
        if t == 0:
            return np.zeros((0, cfg.d), np.float32)
        lens = [s.tokens + len(x) for s, x in news]
        need = [-(-n // cfg.page_tokens) - len(s.pages) for (s, _), n in zip(news, lens)]
        if sum(need) > len(self.free):
            raise ShloError("decoder: %d pages needed, %d free" % (sum(need), len(self.free)))
        # The pages that the step adds stay on the free list until its outputs are there.
        take = iter(self.free[::-1])
        pages = [s.pages + [next(take) for _ in range(n)] for (s, _), n in zip(news, need)]
        width = max(len(p) for p in pages)
        tables = np.array([p + [-1] * (width - len(p)) for p in pages], np.int32)
        starts = np.concatenate([[0], np.cumsum([len(x) for _, x in news])]).astype(np.int32)
        batch = [M.of_numpy(a) for a in (starts, np.array(lens, np.int32), tables)]
        at = M.of_numpy(np.concatenate([np.arange(s.tokens, n, dtype=np.int32) for (s, _), n in zip(news, lens)]))
        h = M.of_numpy(np.concatenate([x for _, x in news]))
        for li in range(cfg.layers):
            h = self._layer(h, li, t, at, batch)
        out = M.to_numpy(M.reshape(h, [t, cfg.d]))
        for (s, _), n, p in zip(news, lens, pages):
            s.tokens, s.pages = n, p
        del self.free[len(self.free) - sum(need):]
        return out

    def _dense(self, x, name, bias, m, k, t, res=None, flags=Run.EP_BIAS):
        if self.cfg.bits8:
            y = D.linear8(M.reshape(x, [t, k]), *self.w[name], bias=self.w[bias])
            if flags & Run.EP_RES:
                y = M.binary(0, y, M.reshape(res, [t, m]))
            return Run.gelu_erf(M.reshape(y, [t * m]), t * m) if flags & Run.EP_GELU else y
        return Run.mul_mat_bias(self.w[name], x, k, m, t, t, 0, self.w[bias], res, flags)

    def _layer(self, h, li, t, at, batch):
        cfg, p = self.cfg, "l%d_" % li
        hq, hk, dh = cfg.heads, cfg.kv_heads, cfg.dh
        a = Run.norm_affine(h, cfg.d, t, EPS_BITS, self.w[p + "g1"], self.w[p + "b1"])
        qkv = M.reshape(self._dense(a, p + "wqkv", p + "cqkv", (hq + 2 * hk) * dh, cfg.d, t), [t, hq + 2 * hk, dh])

        def heads(lo, hi):
            return M.slice_(qkv, [0, lo, 0], [t, hi, dh], [1, 1, 1])
        if cfg.norm_heads:
            qk = D.norm_rope(heads(0, hq + hk), at, self.phases, self.w[p + "gq"], self.w[p + "gk"], q_heads=hq, eps=1e-6,
                             factor=self.factor)
        else:
            qk = D.rope(heads(0, hq + hk), at, self.phases, factor=self.factor)
        cache = self.caches[li]
        cache.append(M.slice_(qk, [0, hq, 0], [t, hq + hk, dh], [1, 1, 1]), heads(hq + hk, hq + 2 * hk), *batch)
        o = cache.attend(M.slice_(qk, [0, 0, 0], [t, hq, dh], [1, 1, 1]), *batch, scale=dh ** -0.5, window=cfg.window)
        h = self._dense(M.reshape(o, [t, cfg.d]), p + "wo", p + "co", cfg.d, cfg.d, t, h, Run.EP_BIAS | Run.EP_RES)
        a = Run.norm_affine(h, cfg.d, t, EPS_BITS, self.w[p + "g2"], self.w[p + "b2"])
        f = self._dense(a, p + "w1", p + "c1", cfg.ffn, cfg.d, t, None, Run.EP_BIAS | Run.EP_GELU)
        return self._dense(f, p + "w2", p + "c2", cfg.d, cfg.ffn, t, h, Run.EP_BIAS | Run.EP_RES)
