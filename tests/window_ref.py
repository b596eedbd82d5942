"""Plain implementation in 64 bits of the sliding-window operators, and ragged
paged batches for their tests. numpy on the host; nothing of the package."""
from __future__ import annotations

import math

import numpy as np
import torch

PAGE = 16
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative


def visible(p: int, window: int, sinks: int) -> np.ndarray:
    j = np.arange(max(p + 1, 0))
    return j if window == 0 else j[(j > p - window) | (j < sinks)]


def kv_head(h: int, Hq: int, Hkv: int, grouped: bool) -> int:
    return h // (Hq // Hkv) if grouped else h % Hkv


def e4m3(x: torch.Tensor) -> torch.Tensor:
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def encode(x: torch.Tensor, fmt: str, scale=None):
    """f32 [..., D] -> (codes uint8, exponent bytes or None) from the formats' definitions."""
    if fmt == "e4m3":
        return e4m3(x / scale).view(torch.uint8), None
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 9, torch.tensor(-127)).clamp(min=-127)
    c = e4m3(torch.ldexp(b, -e.unsqueeze(-1))).flatten(-2)
    return c.view(torch.uint8), (e + 127).to(torch.uint8)


class Batch:
    """A ragged batch: sequence s has tokens[s] tokens, the last new[s] of them
    new. `dead` is what the table entries that no window reaches hold; slots
    that hold no token, and pages that nobody owns, are filled with `junk`."""

    def __init__(self, seed, tokens, new, Hq, Hkv, D, fmt="bf16", grouped=True, window=0, sinks=0, dead=-1,
                 junk=float("nan"), spare=2, magnitude=1.0):
        g = torch.Generator().manual_seed(seed)
        self.tokens, self.new, self.Hq, self.Hkv, self.D = list(tokens), list(new), Hq, Hkv, D
        self.fmt, self.grouped, self.window, self.sinks = fmt, grouped, window, sinks
        self.g = g
        need = []
        for n, m in zip(tokens, new):
            seen = set()
            for p in range(n - m, n):
                seen |= set((visible(p, window, sinks) // PAGE).tolist())
            if m == 0:
                seen = set(range(-(-n // PAGE)))
            need.append(sorted(seen | set(range(max(n - m, 0) // PAGE, -(-n // PAGE)))))
        self.P = sum(len(x) for x in need) + spare
        order = torch.randperm(self.P, generator=g).tolist()
        self.indptr, self.ids, k = [0], [], 0
        live = torch.zeros(self.P, PAGE, dtype=torch.bool)
        for n, x in zip(tokens, need):
            t = [dead] * (-(-n // PAGE))
            for j in x:
                t[j] = order[k]
                live[order[k], :max(0, min(PAGE, n - PAGE * j))] = True
                k += 1
            self.ids += t
            self.indptr.append(len(self.ids))
        self.rows = sum(new)
        self.q_indptr = np.concatenate([[0], np.cumsum(new)]).tolist()
        shape = (self.P, 2, Hkv, PAGE, D)
        x = torch.randn(shape, generator=g) * magnitude
        x[:, 0, :, :, ::17] *= 3.0
        self.scales = None
        hole = ~live[:, None, None, :, None]
        if fmt == "f32":
            self.pool = x
        elif fmt == "bf16":
            self.pool = x.to(torch.bfloat16)
        elif fmt == "e4m3":
            self.scales = torch.rand(2, Hkv, generator=g) * 0.02 * magnitude + 0.01 * magnitude
            self.pool = encode(x, "e4m3", self.scales[None, :, :, None, None])[0]
        else:
            self.pool, self.scales = encode(x, "mxfp8")
        if junk is not None:
            if fmt in ("f32", "bf16"):
                self.pool = torch.where(hole, torch.tensor(junk, dtype=self.pool.dtype), self.pool)
            else:  # 0x7f: the NaN code; 0xff: the NaN exponent
                self.pool = torch.where(hole, torch.tensor(0x7F, dtype=torch.uint8), self.pool)
                if fmt == "mxfp8":
                    self.scales = torch.where(hole, torch.tensor(0xFF, dtype=torch.uint8), self.scales)
        self.q = torch.randn(self.rows, Hq, D, generator=g)

    def values(self) -> np.ndarray:
        """The pool's values in 64 bits."""
        if self.fmt in ("f32", "bf16"):
            return self.pool.double().numpy()
        x = self.pool.view(torch.float8_e4m3fn).double()
        if self.fmt == "e4m3":
            return (x * self.scales.double()[None, :, :, None, None]).numpy()
        e = torch.exp2(self.scales.double() - 127)
        e = torch.where(self.scales == 255, torch.tensor(float("nan"), dtype=torch.float64), e)
        return (x * e.repeat_interleave(32, -1)).numpy()

    def place(self, s: int, j):
        """Page and slot of token(s) j of sequence s."""
        j = np.asarray(j)
        return np.asarray(self.ids, dtype=np.int64)[self.indptr[s] + j // PAGE], j % PAGE

    def attention(self, q=None, skip=lambda page: False):
        """(out, lse, size) of every row: size = sum_j w_j |v_j|, what a rounding
        of the weights is relative to; reach = max_j scale |q|.|k_j|; and mass =
        sum_j |v_j| (MXFP8: with the largest of the tokens' exponents in place
        of each one's own), what weights that are tiny but not zero add up to."""
        vals = self.values()
        q = (self.q if q is None else q).double().numpy()
        out = np.zeros((self.rows, self.Hq, self.D))
        size = np.zeros_like(out)
        lse = np.full((self.rows, self.Hq), -np.inf)
        reach = np.zeros((self.rows, self.Hq))
        mass = np.zeros_like(out)
        for s, (n, m) in enumerate(zip(self.tokens, self.new)):
            pos = np.arange(n - m, n)
            j = np.unique(np.concatenate([visible(p, self.window, self.sinks) for p in pos] or [[]])).astype(int)
            if not len(j):
                continue
            page, slot = self.place(s, j)
            keep = np.array([not skip(p) and 0 <= p < self.P for p in page])
            j, page, slot = j[keep], page[keep], slot[keep]
            see = j <= pos[:, None]
            if self.window:
                see &= (j > pos[:, None] - self.window) | (j < self.sinks)
            some = see.any(1)
            r = np.arange(self.q_indptr[s], self.q_indptr[s] + m)[some]
            see = see[some]
            for h in range(self.Hq if len(r) else 0):
                c = kv_head(h, self.Hq, self.Hkv, self.grouped)
                k, v = vals[page, 0, c, slot], vals[page, 1, c, slot]
                x = np.where(see, q[r, h] @ k.T / math.sqrt(self.D), -np.inf)
                far = np.where(see, np.abs(q[r, h]) @ np.abs(k).T / math.sqrt(self.D), 0)
                reach[r, h] = far.max(1)
                mx = x.max(1, keepdims=True)
                w = np.exp(x - mx)
                lse[r, h] = (mx + np.log(w.sum(1, keepdims=True)))[:, 0]
                w /= w.sum(1, keepdims=True)
                dark = ~see.any(0)  # tokens that no row sees may hold anything
                v = np.where(dark[:, None], 0, v)
                out[r, h], size[r, h] = w @ v, w @ np.abs(v)
                av = np.abs(v)
                if self.fmt == "mxfp8":
                    e = self.scales.numpy()[page, 1, c, slot].astype(int)
                    e = np.where(dark[:, None], 0, e)
                    av *= np.repeat(2.0 ** (e.max(0) - e), 32, -1)
                mass[r, h] = see @ np.where(dark[:, None], 0, av)
        return out, lse, size, reach, mass


def check_attention(got, got_lse, want, what="", weights=2.0 ** -8):
    """Error bound, elementwise. The scores are f32 sums of D products: each is
    off by at most D 2^-24 reach, and so is the LSE (plus its own logarithm and
    sum: 2^-18 covers them). A weight then is off by twice that, relatively, and
    by its rounding `weights` (half a step of the type that the products take);
    the sum adds D-independent f32 roundings (2^-16 covers sums of up to 2^8
    terms per partial sum). FP8 pages take f16 weights, held as 2^7 w relative
    to a reference that is at most the largest weight: below f16's normal range
    a weight is off by up to half of f16's smallest step, 2^-25 / 2^7 = 2^-32 of
    the largest weight (which is at most 1), and times |v| these add up to
    2^-32 mass. The output is rounded once more."""
    out, lse, size, reach, mass = want
    got_t = got.dtype
    g, gl = got.detach().cpu().double().numpy(), got_lse.detach().cpu().double().numpy()
    dead = np.isinf(lse)
    assert np.array_equal(np.isneginf(gl), dead), f"{what}: rows that see nothing"
    assert np.all(g[dead] == 0), f"{what}: rows that see nothing are zero"
    assert np.isfinite(g).all(), f"{what}: not finite"
    score = out.shape[-1] * 2.0 ** -24 * reach
    f = ~dead
    assert np.all(np.abs(gl - np.where(f, lse, 0))[f] <= (score + 2.0 ** -18 * (1 + np.abs(np.where(f, lse, 0))))[f]), f"{what}: lse"
    w = 2.0 ** -18 if got_t == torch.float32 else weights
    tol = HALF[got_t] * np.abs(out) + (2 * score[..., None] + w + 2.0 ** -16) * size * (1 + HALF[got_t]) + 2.0 ** -32 * mass + 1e-30
    err = np.abs(g - out)
    assert np.all(err <= tol), f"{what}: worst error / bound {np.max(err / tol):.2f}"
