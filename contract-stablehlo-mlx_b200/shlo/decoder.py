"""A causal transformer that generates step by step: the denoiser's encoder layer (the
framework's norm, mul_mat and gelu_erf kernels) with rotary positions and an attention
over a paged cache in 8 bits in place of the attention over whole sequences.

    m = Decoder(Config(), pages=256)
    a = m.start(prompt)            # a sequence; its prompt, embedded [n, d]
    y = m.step([(a, x), (b, x2)])  # new tokens of several sequences at once -> their outputs, in order
    m.stop(a)                      # its pages may be used again

Everything a step computes stays on the device; the host keeps which pages a sequence
has. Weights are random (N(0, 0.02), norm gains 1 + N(0, 0.02)), from a seed.
"""
from __future__ import annotations

from dataclasses import dataclass

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
    return out


class Sequence:
    """A running sequence: its length and its pages."""

    __slots__ = ("tokens", "pages")

    def __init__(self):
        self.tokens, self.pages = 0, []


class Decoder:
    def __init__(self, cfg: Config, pages: int, weights: dict | None = None):
        self.cfg = cfg
        self.w = {k: M.of_numpy(v) for k, v in (weights or init_weights(cfg)).items()}
        phases, self.factor = D.rope_phases(cfg.dh, cfg.base)
        self.phases = M.of_numpy(phases)
        self.caches = [D.Cache(pages, cfg.kv_heads, cfg.dh, cfg.page_tokens) for _ in range(cfg.layers)]
        self.free = list(range(pages))[::-1]

    def start(self, prompt: np.ndarray):
        """(a new sequence, the outputs of its prompt [n, d])."""
        s = Sequence()
        return s, self.step([(s, prompt)])

    def stop(self, s: Sequence) -> None:
        self.free += s.pages[::-1]
        s.tokens, s.pages = 0, []

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
        return Run.mul_mat_bias(self.w[name], x, k, m, t, t, 0, self.w[bias], res, flags)

    def _layer(self, h, li, t, at, batch):
        cfg, p = self.cfg, "l%d_" % li
        hq, hk, dh = cfg.heads, cfg.kv_heads, cfg.dh
        a = Run.norm_affine(h, cfg.d, t, EPS_BITS, self.w[p + "g1"], self.w[p + "b1"])
        qkv = M.reshape(self._dense(a, p + "wqkv", p + "cqkv", (hq + 2 * hk) * dh, cfg.d, t), [t, hq + 2 * hk, dh])

        def heads(lo, hi):
            return M.slice_(qkv, [0, lo, 0], [t, hi, dh], [1, 1, 1])
        qk = D.rope(heads(0, hq + hk), at, self.phases, factor=self.factor)
        cache = self.caches[li]
        cache.append(M.slice_(qk, [0, hq, 0], [t, hq + hk, dh], [1, 1, 1]), heads(hq + hk, hq + 2 * hk), *batch)
        o = cache.attend(M.slice_(qk, [0, 0, 0], [t, hq, dh], [1, 1, 1]), *batch, scale=dh ** -0.5, window=cfg.window)
        h = self._dense(M.reshape(o, [t, cfg.d]), p + "wo", p + "co", cfg.d, cfg.d, t, h, Run.EP_BIAS | Run.EP_RES)
        a = Run.norm_affine(h, cfg.d, t, EPS_BITS, self.w[p + "g2"], self.w[p + "b2"])
        f = self._dense(a, p + "w1", p + "c1", cfg.ffn, cfg.d, t, None, Run.EP_BIAS | Run.EP_GELU)
        return self._dense(f, p + "w2", p + "c2", cfg.d, cfg.ffn, t, h, Run.EP_BIAS | Run.EP_RES)
