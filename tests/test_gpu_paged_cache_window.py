"""PagedKVCache with sliding-window layers: chunks of several sequences, a
decode loop in which the engine gives pages back, and read-back, all together
as a model's program uses them, against tests/window_ref.py in 64 bits."""
import numpy as np
import pytest
import torch

import dendrite_b200 as dd
from tests.window_ref import PAGE, Batch, check_attention, encode

pytestmark = pytest.mark.gpu

HQ, HKV, D, P = 8, 2, 128, 96


class Mirror:
    """What the cache holds, on the host: the K/V that each sequence was given,
    as the pool's type stores them."""

    def __init__(self, fmt, scales, windows):
        self.fmt, self.scales, self.windows = fmt, scales, windows
        self.kv = [[] for _ in windows]     # per layer, per sequence: [tokens, 2, HKV, D] float64

    def stored(self, layer, k, v):
        out = []
        for which, x in ((0, k), (1, v)):
            x = x.float()
            if self.fmt == "bf16":
                out.append(x.to(torch.bfloat16).double())
            elif self.fmt == "e4m3":
                c, _ = encode(x, "e4m3", self.scales[layer][which][:, None])
                out.append(c.view(torch.float8_e4m3fn).double() * self.scales[layer][which].double()[:, None])
            else:
                c, e = encode(x, "mxfp8")
                out.append(c.view(torch.float8_e4m3fn).double() * torch.exp2(e.double() - 127).repeat_interleave(32, -1))
        return torch.stack(out, 1)

    def reference(self, layer, seqs, counts, q):
        """attention() of a Batch whose pool is this mirror's."""
        window, sinks = self.windows[layer] or (0, 0)
        b = Batch.__new__(Batch)
        b.tokens = [len(self.kv[layer][s]) for s in seqs]
        b.new, b.Hq, b.Hkv, b.D, b.fmt, b.grouped = list(counts), HQ, HKV, D, "f64", True
        b.window, b.sinks, b.rows = window, sinks, sum(counts)
        b.q_indptr = np.concatenate([[0], np.cumsum(counts)]).tolist()
        pages = [-(-n // PAGE) for n in b.tokens]
        b.indptr = np.concatenate([[0], np.cumsum(pages)]).tolist()
        b.P = b.indptr[-1]
        b.ids = list(range(b.P))
        pool = np.zeros((b.P, 2, HKV, PAGE, D))
        for i, s in enumerate(seqs):
            for j, x in enumerate(self.kv[layer][s]):
                pool[b.indptr[i] + j // PAGE, :, :, j % PAGE] = x
        b.values = lambda: pool
        return b.attention(q)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8"])
def test_chunks_decode_and_read_back(cuda, fmt):
    g = torch.Generator().manual_seed(5)
    windows = [None, (24, 3), (40, 0)]
    scales = [torch.rand(2, HKV, generator=g) * 0.02 + 0.01 for _ in windows] if fmt == "e4m3" else None
    cache = dd.PagedKVCache(len(windows), P, HQ, HKV, D, kv_dtype=fmt, e4m3_scales=scales, device=cuda, windows=windows)
    host = Mirror(fmt, scales, windows)
    free = iter(torch.randperm(P, generator=g).tolist())
    tables, lens = [], []

    def qkv(rows):
        x = torch.randn(rows, HQ + 2 * HKV, D, generator=g).to(torch.bfloat16)
        dx = x.to(cuda)
        return x, (dx[:, :HQ], dx[:, HQ:HQ + HKV], dx[:, HQ + HKV:])

    def check(out, want, layer, what, weights):
        if fmt == "e4m3" and not windows[layer]:
            # The full-attention layer runs the cascade plan, which rounds code * scale
            # to bf16: V is off by 2^-8, and so, times reach, are the scores (D 2^-24
            # 2^9 = 2^-8 at D = 128).
            weights, want = weights + 2.0 ** -8, (*want[:3], want[3] * 2.0 ** 9, want[4])
        check_attention(out, torch.tensor(want[1]), want, what, weights)

    def csr():
        return np.cumsum([0] + [len(t) for t in tables]).astype(np.int32), np.array([i for t in tables for i in t], np.uint32)

    def chunk(counts):
        for s, m in enumerate(counts):
            lens[s] += m
            while len(tables[s]) * PAGE < lens[s]:
                tables[s].append(next(free))
        cache.begin_chunks(*csr(), lens, counts)
        for layer in range(len(windows)):
            x, parts = qkv(sum(counts))
            out = cache.layer_chunk(layer, *parts)
            r = 0
            for s, m in enumerate(counts):
                kv = host.stored(layer, x[r:r + m, HQ:HQ + HKV], x[r:r + m, HQ + HKV:])
                host.kv[layer][s] += list(kv.numpy())
                r += m
            want = host.reference(layer, range(len(counts)), counts, x[:, :HQ])
            lse = torch.tensor(want[1])
            check_attention(out, lse, want, f"chunk {counts} layer {layer}", 2.0 ** -8)

    for _ in range(3):
        tables.append([])
        lens.append(0)
        for layer in host.kv:
            layer.append([])
    chunk([37, 1, 90])            # prompts, ragged
    chunk([5, 60, 0])             # more of two of them
    # one prompt by itself, through the single-sequence call
    tables.append([next(free) for _ in range(2)])
    lens.append(21)
    for layer in range(len(windows)):
        host.kv[layer].append([])
        x, parts = qkv(21)
        out = cache.layer_prefill(layer, *parts, tables[3], 0)
        host.kv[layer][3] = list(host.stored(layer, x[:, HQ:HQ + HKV], x[:, HQ + HKV:]).numpy())
        want = host.reference(layer, [3], [21], x[:, :HQ])
        check(out, want, layer, f"prompt layer {layer}", 2.0 ** -8)
    for step in range(20):
        for s in range(4):
            if lens[s] % PAGE == 0:
                tables[s].append(next(free))
        cache.begin_step(*csr(), np.array(lens))
        for s in range(4):
            lens[s] += 1
        for layer in range(len(windows)):
            x, parts = qkv(4)
            out = cache.layer_step(layer, *parts)
            kv = host.stored(layer, x[:, HQ:HQ + HKV], x[:, HQ + HKV:]).numpy()
            for s in range(4):
                host.kv[layer][s].append(kv[s])
            want = host.reference(layer, range(4), [1] * 4, x[:, :HQ])
            check(out, want, layer, f"step {step} layer {layer}", 2.0 ** -11)
    first, count = [3, 0, 17, 40], [30, 61, 0, 1]
    for layer in range(len(windows)):
        for dt in (torch.float32, torch.bfloat16):
            k, v = cache.read_tokens(layer, *csr(), first, count, dt)
            want = np.concatenate([np.array(host.kv[layer][s][first[s]:first[s] + count[s]]).reshape(-1, 2, HKV, D)
                                   for s in range(4)])
            assert torch.equal(k.cpu(), torch.tensor(want[:, 0]).float().to(dt))
            assert torch.equal(v.cpu(), torch.tensor(want[:, 1]).float().to(dt))


def test_windowed_cache_gives_pages_back(cuda):
    """All layers windowed: pages behind the window go back to the engine, who
    gives them to another sequence; the first one's outputs do not notice."""
    g = torch.Generator().manual_seed(6)
    cache = dd.PagedKVCache(1, 6, HQ, HKV, D, device=cuda, windows=[(20, 2)])
    host = Mirror("bf16", None, [(20, 2)])
    host.kv[0].append([])
    free, table, n = list(range(6)), [], 0
    for step in range(150):
        if n % PAGE == 0:
            table.append(free.pop(0))
        x = torch.randn(1, HQ + 2 * HKV, D, generator=g).to(torch.bfloat16)
        dx = x.to(cuda)
        ids = np.array([i if i is not None else 2 ** 32 - 1 for i in table], np.uint32)
        assert cache.begin_step(np.array([0, len(table)]), ids, [n]) is False
        out = cache.layer_step(0, dx[:, :HQ], dx[:, HQ:HQ + HKV], dx[:, HQ + HKV:])
        host.kv[0][0].append(host.stored(0, x[:, HQ:HQ + HKV], x[:, HQ + HKV:]).numpy()[0])
        n += 1
        want = host.reference(0, [0], [1], x[:, :HQ])
        check_attention(out, torch.tensor(want[1]), want, f"step {step}", 2.0 ** -11)
        # Behind the next token's window, and not the first tokens' page: back, and written over.
        for j in range(1, max(0, n - 20) // PAGE):
            if table[j] is not None:
                cache.pools[0][table[j]] = float("nan")
                free.append(table[j])
                table[j] = None
