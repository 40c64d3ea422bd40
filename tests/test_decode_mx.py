"""Decode over 4-bit caches, and with attention weights over 4-bit, fp16 and bf16
ones, against the float64 oracle."""
import numpy as np
import pytest
import torch

import attnkernels as ak
from oracle import small_cache as oracle

pytestmark = pytest.mark.gpu


class Case:
    """A batch over a scattered pool, whose unused rows hold NaN (4-bit: the NaN scale)."""

    def __init__(self, lens, hkv, group, d, bs=16, fmt="mxfp4", dtype=torch.float16, seed=0, spare=3):
        r = np.random.default_rng(seed)
        self.fmt, self.dtype, self.d, self.lens = fmt, dtype, d, lens
        blocks = [-(-n // bs) for n in lens]
        pool = sum(blocks) + spare
        order = r.permutation(pool)
        self.tables = np.full((len(lens), max(blocks + [1])), pool + 7, dtype=np.int32)
        at = 0
        used = np.zeros((pool, bs), dtype=bool)
        for b, (nb, n) in enumerate(zip(blocks, lens)):
            self.tables[b, :nb] = order[at:at + nb]
            for i in range(n):
                used[self.tables[b, i // bs], i % bs] = True
            at += nb
        to = lambda x: torch.from_numpy(x).to(dtype).double().numpy()  # noqa: E731
        self.q = to(r.standard_normal((len(lens), hkv * group, d)))
        self.values, self.caches = [], []
        for _ in range(2):
            x = to(r.standard_normal((pool, hkv, bs, d)))
            if fmt == "mxfp4":
                codes, scales = oracle.mxfp4_encode(x)
                scales = np.where(used[:, None, :, None], scales, 255).astype(np.uint8)
                self.caches += [torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()]
                self.values.append(oracle.mxfp4_decode(codes, scales))
            else:
                x = np.where(used[:, None, :, None], x, np.nan)
                self.values.append(x)
                self.caches.append(torch.from_numpy(x).to(dtype).cuda())
        self.weights = r.random((len(lens), hkv, max(lens + [1]) + 5)).astype(np.float32)

    def gpu(self, x, kind=None):
        return torch.from_numpy(np.ascontiguousarray(x)).cuda() if kind is None else torch.from_numpy(x).to(kind).cuda()

    def run(self, weights=None, longest=None, scale=None, partition=None, lens=None):
        q, tables = self.gpu(self.q, self.dtype), self.gpu(self.tables)
        lens = self.gpu(np.array(self.lens if lens is None else lens, dtype=np.int32))
        longest = max(max(self.lens), 1) if longest is None else longest
        if self.fmt == "mxfp4":
            return ak.paged_decode_mxfp4(q, *self.caches, tables, lens, longest, scale=scale, partition_size=partition,
                                         weights=weights)
        return ak.paged_decode_weights(q, *self.caches, tables, lens, longest, weights, scale=scale,
                                       partition_size=partition)

    def check(self, out, weights=None, before=None, scale=None, lens=None):
        scale = self.d ** -0.5 if scale is None else scale
        lens = self.lens if lens is None else lens
        want, added, spread, reach = oracle.decode(self.q, *self.values, self.tables, lens, scale)
        half = torch.finfo(self.dtype).eps / 2
        # A score sums D exact products in fp32 and is rounded a few times more: off by at most ds; a weight's
        # relative error is then about 2 ds (its own, and the sum's), and the exponentials' 2^-22.
        ds = (self.d + 8) * 2.0 ** -24 * (reach + 8)
        rel = 2 * ds + 2.0 ** -20
        # P is rounded to the type, the output too; fp16 holds a P below 2^-21 of the largest to 2^-32 of it.
        tol = spread * (half * 1.01 + rel[..., None]) + np.abs(want) * half * 1.01 + \
            2.0 ** -32 * max(lens + [1]) * np.nanmax([np.nanmax(np.abs(np.nan_to_num(v))) for v in self.values]) + 2.0 ** -25
        got = out.double().cpu().numpy()
        assert got.shape == want.shape and (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
        if weights is not None:
            w = weights.double().cpu().numpy()
            group = self.q.shape[1] // w.shape[1]
            for b, add in enumerate(added):
                n = add.shape[1]
                full = before[b].astype(np.float64)
                full[:, :n] += add
                rel_b = rel[b].reshape(-1, group).max(1, keepdims=True) if n else 0.0
                allowed = np.zeros_like(full)
                allowed[:, :n] = add * (rel_b + group * 2.0 ** -24) + np.abs(full[:, :n]) * 2.0 ** -24 + 2.0 ** -40
                assert (np.abs(w[b] - full) <= allowed).all()

    def tracked(self, **how):
        w = self.gpu(self.weights)
        out = self.run(weights=w, **how)
        how.pop("partition", None), how.pop("longest", None)
        self.check(out, w, self.weights, **how)
        return out, w


FORMATS = [("mxfp4", torch.float16), ("mxfp4", torch.bfloat16), ("full", torch.float16), ("full", torch.bfloat16)]


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hkv,group", [(2, 1), (1, 2), (2, 4), (1, 5), (2, 8), (1, 16)])
def test_ragged_batches(fmt, dtype, d, hkv, group):
    c = Case([1, 31, 0, 32, 33, 300, 777], hkv, group, d, fmt=fmt, dtype=dtype, seed=group)
    c.tracked()
    if fmt == "mxfp4":
        c.check(c.run())


@pytest.mark.parametrize("fmt,dtype", FORMATS)
@pytest.mark.parametrize("bs", [1, 5, 8, 12, 16, 32, 48, 64, 1024])
def test_page_sizes(fmt, dtype, bs):
    c = Case([517, 3, 96], 2, 4, 128, bs=bs, fmt=fmt, dtype=dtype, seed=bs)
    c.tracked()
    c.tracked(partition=256)
    if fmt == "mxfp4":
        c.check(c.run())
        c.check(c.run(partition=256))


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("partition", [256, 300, 1024, 1 << 20])
def test_splits(fmt, d, partition):
    """Few splits, many, one."""
    c = Case([9000, 1, 256, 257, 0], 1, 3, d, fmt=fmt, seed=partition)
    c.tracked(partition=partition)
    if fmt == "mxfp4":
        for _ in range(2):  # the counters are left at zero
            c.check(c.run(partition=partition))


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(fmt, scale):
    Case([200, 77], 2, 4, 128, fmt=fmt, seed=3).tracked(scale=scale)


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
@pytest.mark.parametrize("partition", [None, 256])
def test_bad_pages_are_left_out(fmt, partition):
    """Pages outside the pool: some tokens, a whole split, a whole sequence."""
    c = Case([600, 600, 40], 2, 4, 128, fmt=fmt, seed=5)
    c.tables[0, 3] = -1
    c.tables[0, 20] = 1 << 30
    c.tables[1, :16] = c.values[0].shape[0]
    c.tables[2, :] = -5
    out, w = c.tracked(partition=partition)
    assert not out[2].any() and torch.equal(w[2], c.gpu(c.weights)[2])
    if fmt == "mxfp4":
        c.check(c.run(partition=partition))


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
def test_lengths_past_the_table_and_max_context_len(fmt):
    """Contexts longer than the table's row or max_context_len are cut there, negative ones are empty."""
    c = Case([64, 64, 64], 2, 2, 64, fmt=fmt, seed=6)
    c.tracked(lens=[64, 40, 0], longest=64)
    w = c.gpu(c.weights)
    out = c.run(weights=w, lens=[1000, 40, -3], longest=64)
    c.check(out, w, c.weights, lens=[64, 40, 0])
    w = c.gpu(c.weights)
    out = c.run(weights=w, lens=[64, 40, 7], longest=33)
    c.check(out, w, c.weights, lens=[33, 33, 7])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_keys_of_minus_infinity_weigh_nothing(dtype):
    """Scores of -inf in some tokens, in whole tiles at the start, in every token."""
    c = Case([300, 300, 50], 1, 2, 64, fmt="full", dtype=dtype, seed=7)
    c.q = np.abs(c.q)
    for b, gone in ((0, [1, 5, 299]), (1, range(0, 200)), (2, range(50))):
        for t in gone:
            c.values[0][c.tables[b, t // 16], 0, t % 16] = -np.inf
    c.caches[0] = torch.from_numpy(c.values[0]).to(dtype).cuda()
    out, w = c.tracked()
    assert not out[2].any() and torch.equal(w[2], c.gpu(c.weights)[2])


def test_nan_stays_in_its_sequence_and_head():
    for fmt in ("mxfp4", "full"):
        c = Case([100, 100], 2, 2, 128, fmt=fmt, seed=8)
        page = int(c.tables[0, 2])
        if fmt == "mxfp4":
            c.caches[1][page, 1, 3, 0] = 255
        else:
            c.caches[0][page, 1, 3, 0] = float("nan")
        w = c.gpu(c.weights)
        out = c.run(weights=w)
        assert out[0, 2:].isnan().all() and not out[0, :2].isnan().any() and not out[1].isnan().any()
        assert w[0, 1, :100].isnan().all() and not w[0, 0].isnan().any() and not w[1].isnan().any()
        assert not w[0, 1, 100:].isnan().any()


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
def test_late_maxima(fmt):
    """Scores that grow along the context: the subtracted maximum moves, by little and by much."""
    c = Case([512, 512], 1, 2, 64, fmt=fmt, seed=9)
    c.q = np.abs(c.q)
    for b, step in ((0, 0.01), (1, 0.2)):
        for t in range(512):
            c.values[0][c.tables[b, t // 16], 0, t % 16] = np.abs(c.values[0][c.tables[b, t // 16], 0, t % 16]) * step * t / 64
    x = torch.from_numpy(np.nan_to_num(c.values[0])).half().double().numpy()
    if fmt == "mxfp4":
        codes, scales = oracle.mxfp4_encode(x)
        c.caches[0], c.caches[1] = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
        x = oracle.mxfp4_decode(codes, scales)
    else:
        c.caches[0] = torch.from_numpy(x).half().cuda()
    c.values[0] = x
    c.tracked()


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
def test_views_of_weights_and_other_strides(fmt):
    """weights as a view of a larger buffer, heads before sequences; q and the integer arrays in other layouts."""
    c = Case([70, 200, 9], 2, 4, 64, fmt=fmt, seed=10)
    L = c.weights.shape[2]
    big = torch.full((2, 5, L + 3), 9.0, device="cuda")
    view = big[:, 1:4, :L].transpose(0, 1)
    view.copy_(c.gpu(c.weights))
    q = c.gpu(c.q, torch.float16).transpose(0, 1).contiguous().transpose(0, 1)
    tables = c.gpu(c.tables).t().contiguous().t().long()
    lens = torch.tensor(c.lens, device="cuda")
    if fmt == "mxfp4":
        out = ak.paged_decode_mxfp4(q, *c.caches, tables, lens, 200, weights=view)
    else:
        out = ak.paged_decode_weights(q, *c.caches, tables, lens, 200, view)
    c.check(out, view, c.weights)
    assert (big[:, 0] == 9).all() and (big[:, 4] == 9).all() and (big[:, :, L:] == 9).all()


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
def test_shared_pages_are_counted_apart(fmt):
    c = Case([96, 96], 2, 2, 64, fmt=fmt, seed=11)
    c.tables[1] = c.tables[0]
    c.tracked()


def test_agrees_with_paged_decode():
    """The same fp16 caches through paged_decode: two roundings of P and of the output apart."""
    c = Case([500, 64, 3], 2, 4, 128, fmt="full", seed=12)
    out, _ = c.tracked()
    other = ak.paged_decode(c.gpu(c.q, torch.float16), *[torch.nan_to_num(x) for x in c.caches], c.gpu(c.tables),
                            c.gpu(np.array(c.lens, dtype=np.int32)), 500)
    _, _, spread, _ = oracle.decode(c.q, *c.values, c.tables, c.lens, 128 ** -0.5)
    assert ((out - other).double().cpu().numpy() <= 2 ** -11 * 4.1 * spread + 2 ** -20).all()


def test_rows_past_4_gib():
    """A pool whose last rows lie past 2^32 bytes (and past 2^31 elements) of each cache."""
    hkv, d, bs = 8, 128, 16
    blocks = (5 << 30) // (hkv * d * bs * 2)
    k = torch.empty(blocks, hkv, bs, d, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    small = Case([100, 37], hkv, 2, d, fmt="full", seed=13)
    pool = small.values[0].shape[0]
    for big, x in ((k, small.caches[0]), (v, small.caches[1])):
        big[-pool:] = x
    tables = small.gpu(small.tables) + (blocks - pool)
    w = small.gpu(small.weights)
    out = ak.paged_decode_weights(small.gpu(small.q, torch.float16), k, v, tables,
                                  small.gpu(np.array(small.lens, dtype=np.int32)), 100, w)
    small.check(out, w, small.weights)


def test_no_sequences():
    c = Case([5], 2, 2, 64, seed=14)
    out = ak.paged_decode_mxfp4(torch.empty(0, 4, 64, device="cuda").half(), *c.caches,
                                torch.empty(0, 1, dtype=torch.int32, device="cuda"),
                                torch.empty(0, dtype=torch.int32, device="cuda"), 5)
    assert out.shape == (0, 4, 64)


def test_refuses_what_the_kernels_do_not_serve():
    c = Case([5], 1, 17, 64, seed=15)
    with pytest.raises(RuntimeError, match="at most 16"):
        c.run()
    c = Case([5], 1, 2, 64, seed=15)
    with pytest.raises(RuntimeError, match="max_context_len"):
        c.run(longest=0)
    w = c.gpu(c.weights)
    with pytest.raises(RuntimeError, match="overlap"):
        Case([5, 5], 2, 2, 64, seed=15).run(weights=w.expand(2, 2, w.shape[2]))


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
def test_other_streams_and_repeats(fmt):
    """Results do not depend on the stream or the call; weights add up over calls."""
    c = Case([800, 41, 2000], 2, 4, 128, fmt=fmt, seed=16)
    first, w = c.tracked()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w2 = c.gpu(c.weights)
        again = c.run(weights=w2)
        split = c.run(weights=w2, partition=256)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)
    c.check(split)
    twice = 2 * (w - c.gpu(c.weights)) + c.gpu(c.weights)
    assert torch.allclose(w2, twice, rtol=2 ** -18, atol=2 ** -20)


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
@pytest.mark.parametrize("partition", [None, 256])
def test_more_sequences_than_lanes(fmt, partition):
    """Splits are counted 64 sequences at a time; the longest contexts are not among the first."""
    r = np.random.default_rng(17)
    lens = [int(n) for n in r.integers(0, 150, 150)]
    lens[70], lens[149], lens[64], lens[63] = 1900, 1201, 0, 600
    c = Case(lens, 2, 2, 64, fmt=fmt, seed=17)
    c.tracked(partition=partition)
    if fmt == "mxfp4":
        for _ in range(2):
            c.check(c.run(partition=partition))


@pytest.mark.parametrize("fmt,group", [("mxfp4", 2), ("full", 1), ("full", 9)])
def test_weights_of_large_batches(fmt, group):
    """Enough tokens that a thread has four of them, and more than eight heads."""
    r = np.random.default_rng(18)
    lens = [int(n) for n in r.integers(0, 40, 260)]
    lens[100] = 1021
    Case(lens, 8, group, 64, fmt=fmt, seed=18).tracked()


def test_contexts_past_2_24():
    """Tokens past 2^24 of one sequence, whose cut is counted in integers: 2^24 + 300 tokens on one shared page, and
    the last 300 on their own."""
    n, bs = (1 << 24) + 300, 1024
    c = Case([bs, 300], 1, 2, 64, bs=bs, fmt="mxfp4", seed=19, spare=0)
    page, last = int(c.tables[0, 0]), int(c.tables[1, 0])
    tables = torch.full((1, -(-n // bs)), page, dtype=torch.int32, device="cuda")
    tables[0, -1] = last
    w = torch.zeros(1, 1, n, device="cuda")
    q = c.gpu(c.q, torch.float16)[:1]
    out = ak.paged_decode_mxfp4(q, *c.caches, tables, torch.tensor([n], dtype=torch.int32, device="cuda"), n, weights=w)
    k, v = (torch.from_numpy(np.concatenate([x[page, 0], x[last, 0, :300]])) for x in c.values)
    s = k @ torch.from_numpy(c.q[0]).T / 8
    times = torch.ones(bs + 300).double()
    times[:bs] = (1 << 24) // bs
    p = torch.exp(s - s.max()) * times[:, None]
    p = p / p.sum(0)
    # P and the output are rounded once each (2^-11).  A wave has 2^11 tiles, so its sums take 2^11 additions one after
    # the other, each off by a step at most (2^-12 in all).
    assert torch.allclose(out[0].double().cpu(), p.T @ v, rtol=0,
                          atol=(2.0 ** -10 + 2.0 ** -11) * float((p.T @ v.abs()).max()))
    want = (p / times[:, None]).sum(1)
    got = w[0, 0].double().cpu()
    assert torch.allclose(got[:1 << 24].view(-1, bs), want[None, :bs].expand((1 << 24) // bs, bs), rtol=2.0 ** -11, atol=0)
    assert torch.allclose(got[1 << 24:], want[bs:], rtol=2.0 ** -11, atol=0)
