"""Eviction from paged caches by accumulated weight against the oracle: positions,
weights and every byte of the caches are compared exactly."""
import numpy as np
import pytest
import torch

import attnkernels as ak
from oracle import small_cache as oracle

pytestmark = pytest.mark.gpu

KINDS = ["float16", "bfloat16", "mxfp4"]


def _pool(blocks, hkv, bs, d, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "mxfp4":
        return [torch.randint(0, 256, (blocks, hkv, bs, w), generator=g, dtype=torch.uint8) for w in
                (d // 2, d // 2, d // 32, d // 32)]
    return [torch.randn(blocks, hkv, bs, d, generator=g).to(getattr(torch, kind)) for _ in range(2)]


def _tables(lens, bs, extra, seed, width=0):
    r = np.random.default_rng(seed)
    blocks = [-(-max(n, 0) // bs) for n in lens]
    pool = sum(blocks) + extra
    order = r.permutation(pool).astype(np.int32)
    tables = np.full((len(lens), max(blocks + [width, 1])), -1, dtype=np.int32)
    at = 0
    for b, nb in enumerate(blocks):
        tables[b, :nb] = order[at:at + nb]
        at += nb
    return tables, order[at:], pool


def _bytes(x):
    return x.cpu().contiguous().view(torch.uint8).reshape(*x.shape[:3], -1).numpy()


def _run(caches, tables, lens, weights, budget, recent, new=None):
    gpu = [c.cuda() for c in caches]
    scales = gpu[2:] or [None, None]
    w = weights.cuda() if not weights.is_cuda else weights
    got = ak.evict_cache(gpu[0], gpu[1], torch.from_numpy(tables).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), w,
                         budget, recent, *scales, new_block_tables=None if new is None else torch.from_numpy(new).cuda())
    want = oracle.evict([_bytes(c) for c in caches], tables, lens, weights.cpu().numpy(), budget, recent, new)
    assert np.array_equal(got[0].cpu().numpy(), want[0])
    assert np.array_equal(got[2].cpu().numpy(), want[2])
    assert np.array_equal(got[1].cpu().numpy(), want[1], equal_nan=True)
    for a, b in zip(gpu, want[3]):
        assert np.array_equal(_bytes(a), b)
    return got


def _weights(lens, hkv, length, seed, levels=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(torch.randn(len(lens), hkv, length, generator=g))
    return torch.round(w * levels) / levels if levels else w


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (40, 0), (40, 13), (40, 40), (200, 64), (2000, 3)])
def test_ragged_batches(kind, d, budget, recent):
    lens = [0, 1, 39, 40, 41, 300, 777]
    tables, _, pool = _tables(lens, 16, 2, seed=budget)
    _run(_pool(pool, 2, 16, d, kind, budget), tables, lens, _weights(lens, 2, 780, budget), budget, recent)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bs", [1, 5, 8, 12, 64, 1024])
def test_page_sizes(kind, bs):
    lens = [500, 77]
    tables, _, pool = _tables(lens, bs, 1, seed=bs)
    _run(_pool(pool, 3, bs, 64, kind, bs), tables, lens, _weights(lens, 3, 500, bs), 60, 20)


@pytest.mark.parametrize("d,kind", [(32, "mxfp4"), (96, "mxfp4"), (96, "float16"), (512, "mxfp4"), (512, "bfloat16"),
                                    (8, "float16"), (200, "float16")])
def test_row_sizes(d, kind):
    """Rows that are not whole 128-byte columns, scale rows of 1, 3 and 16 bytes."""
    lens = [150, 90]
    tables, _, pool = _tables(lens, 16, 1, seed=d)
    _run(_pool(pool, 2, 16, d, kind, d), tables, lens, _weights(lens, 2, 150, d), 50, 10)


@pytest.mark.parametrize("levels", [1, 3, 20])
def test_ties_go_to_the_first(levels):
    """Weights of few values, the sum of a bin's more than one sweep of the kernel among them."""
    lens = [9000, 500]
    tables, _, pool = _tables(lens, 16, 0, seed=levels)
    _run(_pool(pool, 1, 16, 64, "mxfp4", levels), tables, lens, _weights(lens, 1, 9000, levels, levels), 3000, 100)


def test_weights_of_every_kind():
    """Zeros of both signs, negative weights, infinities, NaN of both signs, subnormals, the largest and smallest."""
    values = torch.tensor([0.0, -0.0, -1.0, 1.0, float("inf"), -float("inf"), float("nan"), 1e-45, -1e-45, 3.4e38, -3.4e38,
                           1.0000001, 1e-38])
    values = torch.cat((values, torch.tensor([-0x400000], dtype=torch.int32).view(torch.float32)))  # a negative NaN
    g = torch.Generator().manual_seed(1)
    lens = [100, 64]
    tables, _, pool = _tables(lens, 16, 0, seed=1)
    w = values[torch.randint(0, len(values), (2, 2, 100), generator=g)]
    for budget in (5, 17, 40, 63):
        _run(_pool(pool, 2, 16, 64, "float16", 1), tables, lens, w, budget, 4)
        _run(_pool(pool, 2, 16, 64, "float16", 1), tables, lens, torch.zeros_like(w), budget, 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,budget", [(5000, 4200), (20000, 300), (20000, 19990)])
def test_long_contexts(kind, n, budget):
    lens = [n]
    tables, _, pool = _tables(lens, 16, 0, seed=n)
    _run(_pool(pool, 2, 16, 128, kind, n), tables, lens, _weights(lens, 2, n, n), budget, 64)


@pytest.mark.parametrize("kind", KINDS)
def test_into_new_pages(kind):
    """Every kept row goes to new pages, of sequences that keep everything too; the old pages stay, shared ones among
    them."""
    lens = [300, 20, 0, 300]
    tables, spare, pool = _tables(lens, 16, 40, seed=2)
    tables[3] = tables[0]
    new = spare[:28].reshape(4, 7).copy()
    caches = _pool(pool, 2, 16, 64, kind, 2)
    _run(caches, tables, lens, _weights(lens, 2, 300, 2), 100, 30, new)


def test_bad_pages_and_long_lengths():
    """Rows on pages outside the pool are neither read nor written; lengths past the table or the weights are cut."""
    lens = [200, 200, 5000, -4]
    tables, _, pool = _tables([200, 200, 100, 0], 16, 0, seed=3)
    caches = _pool(pool, 2, 16, 64, "float16", 3)
    tables[0, [2, 9]] = pool
    tables[1, [0, 12]] = -7
    _run(caches, tables, lens, _weights(lens, 2, 300, 3), 60, 16)
    _run(caches, tables[:2], lens[:2], _weights(lens[:2], 2, 150, 3), 60, 16)


def test_views_of_weights_and_one_call_after_another():
    lens, hkv = [400, 90, 250], 2
    tables, _, pool = _tables(lens, 16, 0, seed=4)
    caches = _pool(pool, hkv, 16, 64, "bfloat16", 4)
    big = torch.randn(hkv, 5, 410, device="cuda")
    view = big[:, 1:4, :400].transpose(0, 1)
    before = big.clone()
    _run(caches, tables, lens, view, 100, 7)
    assert torch.equal(big, before)
    # evicting twice: the second call goes on from the first one's caches, weights and lengths
    gpu = [c.cuda() for c in caches]
    t = torch.from_numpy(tables).cuda()
    n1, w1, _ = ak.evict_cache(*gpu, t, torch.tensor(lens).cuda(), view, 200, 7)
    middle = [c.cpu() for c in gpu]
    n2, w2, k2 = ak.evict_cache(*gpu, t, n1, w1, 50, 5)
    want = oracle.evict([_bytes(c) for c in middle], tables, n1.tolist(), w1.cpu().numpy(), 50, 5)
    assert np.array_equal(n2.cpu(), want[0]) and np.array_equal(w2.cpu(), want[1]) and np.array_equal(k2.cpu(), want[2])
    for a, b in zip(gpu, want[3]):
        assert np.array_equal(_bytes(a), b)


def test_no_sequences():
    caches = [c.cuda() for c in _pool(2, 2, 16, 64, "float16", 5)]
    n, w, kept = ak.evict_cache(*caches, torch.empty(0, 3, dtype=torch.int32).cuda(), torch.empty(0, dtype=torch.int32).cuda(),
                                torch.empty(0, 2, 10).cuda(), 5)
    assert n.shape == (0,) and w.shape == (0, 2, 10) and kept.shape == (0, 2, 5)
