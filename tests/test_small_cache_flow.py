"""The smaller cache as a serving loop uses it: prompts written in 4 bits, their
weights, decode steps that add to them, eviction, and decode from what is left;
eager and captured into graphs."""
import numpy as np
import pytest
import torch

import attnkernels as ak
from oracle import small_cache as oracle

pytestmark = pytest.mark.gpu


class Loop:
    """Two sequences of a layer; every tensor of the loop, and its oracle in float64."""

    def __init__(self, fmt, dtype, seed=0):
        self.fmt, self.dtype = fmt, dtype
        self.hq, self.hkv, self.d, self.bs, self.length = 8, 2, 64, 16, 256
        self.g = torch.Generator().manual_seed(seed)
        self.tables = torch.randperm(40, generator=self.g)[:32].view(2, 16).to(torch.int32).cuda()
        if fmt == "mxfp4":
            self.caches = [torch.zeros(40, self.hkv, self.bs, w, dtype=torch.uint8, device="cuda") for w in (32, 2, 32, 2)]
        else:
            self.caches = [torch.zeros(40, self.hkv, self.bs, self.d, dtype=dtype, device="cuda") for _ in range(2)]
        self.lens = torch.zeros(2, dtype=torch.int32, device="cuda")
        self.weights = torch.zeros(2, self.hkv, self.length, device="cuda")

    def rows(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.dtype).cuda()

    def slots(self, b, positions):
        return self.tables[b, positions // self.bs].long() * self.bs + positions % self.bs

    def write(self, k, v, slots):
        if self.fmt == "mxfp4":
            ak.reshape_and_cache_mxfp4(k, v, *self.caches, slots)
        else:
            ak.reshape_and_cache(k, v, *self.caches, slots)

    def decode(self, q):
        if self.fmt == "mxfp4":
            return ak.paged_decode_mxfp4(q, *self.caches, self.tables, self.lens, self.length, weights=self.weights)
        return ak.paged_decode_weights(q, *self.caches, self.tables, self.lens, self.length, self.weights)

    def evict(self, budget, recent):
        k, v = (self.caches[0], self.caches[2]) if self.fmt == "mxfp4" else self.caches
        scales = (self.caches[1], self.caches[3]) if self.fmt == "mxfp4" else (None, None)
        self.lens, self.weights, kept = ak.evict_cache(k, v, self.tables, self.lens, self.weights, budget, recent, *scales)
        return kept

    def prompt(self, lens):
        total = sum(lens)
        q, k, v = self.rows(total, self.hq, self.d), self.rows(total, self.hkv, self.d), self.rows(total, self.hkv, self.d)
        cu = torch.tensor([0, lens[0], total], dtype=torch.int32, device="cuda")
        self.write(k, v, torch.cat([self.slots(b, torch.arange(n, device="cuda")) for b, n in enumerate(lens)]))
        ak.prompt_weights(q, k, cu, max(lens), self.weights)
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return q, k, v

    def step(self):
        k, v, q = self.rows(2, self.hkv, self.d), self.rows(2, self.hkv, self.d), self.rows(2, self.hq, self.d)
        at = self.lens.long()
        self.write(k, v, torch.cat([self.slots(b, at[b:b + 1]) for b in range(2)]))
        self.lens = self.lens + 1
        return q, k, v, self.decode(q)


@pytest.mark.parametrize("fmt,dtype", [("mxfp4", torch.float16), ("mxfp4", torch.bfloat16), ("full", torch.float16),
                                       ("full", torch.bfloat16)])
def test_prompt_steps_eviction_steps(fmt, dtype):
    loop, half = Loop(fmt, dtype), torch.finfo(dtype).eps / 2
    lens = [100, 61]
    q, k, v = loop.prompt(lens)
    held = oracle.mxfp4_decode if fmt == "mxfp4" else None

    def value(x):  # what the cache holds of rows
        x = x.double().cpu().numpy()
        return held(*oracle.mxfp4_encode(x)) if held else x

    # the oracle's cache: rows [n, Hkv, D] of each sequence, and the weights
    cut = np.cumsum([0] + lens)
    keys = [value(k[cut[b]:cut[b + 1]]) for b in range(2)]
    vals = [value(v[cut[b]:cut[b + 1]]) for b in range(2)]
    w, _ = oracle.prompt(q.double().cpu().numpy(), k.double().cpu().numpy(), cut.tolist(), loop.length)
    for round_ in range(2):
        for _ in range(3):
            q1, k1, v1, out = loop.step()
            for b in range(2):
                keys[b] = np.concatenate((keys[b], value(k1[b:b + 1])))
                vals[b] = np.concatenate((vals[b], value(v1[b:b + 1])))
                for h in range(loop.hq):
                    s = keys[b][:, h // 4] @ q1[b, h].double().cpu().numpy() * loop.d ** -0.5
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    w[b, h // 4, :len(p)] += p
                    spread = p @ np.abs(vals[b][:, h // 4])
                    err = np.abs(out[b, h].double().cpu().numpy() - p @ vals[b][:, h // 4])
                    assert (err <= spread * (2.1 * half + 2.0 ** -14)).all()
        # weights: each is off by at most 2^-14 of itself (scores of some tens of rounding steps), as is every sum of them
        assert (np.abs(loop.weights.double().cpu().numpy() - w) <= w * 2.0 ** -14).all()
        before = loop.weights.cpu().numpy()
        kept = loop.evict(48, 8).cpu().numpy()
        assert loop.lens.tolist() == [48, 48]
        for b in range(2):
            for h in range(2):
                assert kept[b, h].tolist() == oracle.keep(before[b, h, :len(keys[b])], 48, 8).tolist()
            keys[b] = np.stack([keys[b][kept[b, h], h] for h in range(2)], 1)
            vals[b] = np.stack([vals[b][kept[b, h], h] for h in range(2)], 1)
            w[b] = np.stack([np.pad(w[b, h, kept[b, h]], (0, loop.length - 48)) for h in range(2)])


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
def test_captured_steps_replay(fmt):
    """A step's write and decode, and the other calls, captured; replays with eager work between equal the eager calls
    bit for bit, also where two graphs share a memory pool."""
    loop = Loop(fmt, torch.float16, seed=3)
    lens = [200, 77]
    q, k, v = loop.prompt(lens)
    k1, v1, q1 = loop.rows(2, 2, 64), loop.rows(2, 2, 64), loop.rows(2, 8, 64)
    slots = torch.cat([loop.slots(b, torch.tensor([n], device="cuda")) for b, n in enumerate(lens)])
    loop.lens = loop.lens + 1
    cu = torch.tensor([0, 200, 277], dtype=torch.int32, device="cuda")
    start = loop.weights.clone()
    caches = [c.clone() for c in loop.caches]

    def restore():
        loop.weights.copy_(start)
        for c, x in zip(loop.caches, caches):
            c.copy_(x)

    def step():
        loop.write(k1, v1, slots)
        return [loop.decode(q1), ak.paged_decode_mxfp4(q1, *loop.caches, loop.tables, loop.lens, 256, partition_size=256)
                if fmt == "mxfp4" else loop.decode(q1)]

    def upkeep():
        fresh = torch.empty_like(start)
        ak.prompt_weights(q, k, cu, 200, fresh)
        args = (loop.caches[0], loop.caches[2], loop.tables, loop.lens, fresh, 50, 10, loop.caches[1], loop.caches[3]) if \
            fmt == "mxfp4" else (*loop.caches, loop.tables, loop.lens, fresh, 50, 10)
        return [*ak.evict_cache(*args), fresh]

    pool, graphs = None, []
    for work in (step, upkeep):
        restore()
        want = [x.clone() for x in work()] + [loop.weights.clone()] + [c.clone() for c in loop.caches]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        graphs.append(graph)  # a memory pool lives as long as a graph of it
        with torch.cuda.graph(graph, pool=pool):
            got = work()
        pool = graph.pool()
        for i in range(4):
            restore()
            for x in got:
                x.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(got + [loop.weights] + loop.caches, want):
                assert torch.equal(x, y), (work.__name__, i)
            junk = torch.randn(1 << 20, device="cuda").sum()  # eager work between replays
            torch.cuda.synchronize()
            del junk


def test_gathered_rows_go_to_a_full_cache():
    """A 4-bit sequence moved to an fp16 cache decodes as it did, but for the roundings of P and the output."""
    loop = Loop("mxfp4", torch.float16, seed=5)
    loop.prompt([90, 33])
    q = loop.rows(2, 8, 64)
    full = [torch.zeros(40, 2, 16, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    for b, n in enumerate([90, 33]):
        slots = loop.slots(b, torch.arange(n, device="cuda"))
        ak.reshape_and_cache(*ak.gather_cache_mxfp4(*loop.caches, slots), *full, slots)
    a = ak.paged_decode_mxfp4(q, *loop.caches, loop.tables, loop.lens, 90)
    b = ak.paged_decode(q, *full, loop.tables, loop.lens, 90)
    top = full[1].abs().max()
    assert (a - b).abs().max() <= 4.1 * 2.0 ** -11 * top
