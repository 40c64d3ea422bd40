"""Attention weights of packed prompts, summed per token, against the float64 oracle."""
import numpy as np
import pytest
import torch

import attnkernels as ak
from oracle import small_cache as oracle

pytestmark = pytest.mark.gpu


def _case(lens, hq, hkv, d, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    total = sum(lens)
    q = (spread * torch.randn(total, hq, d, generator=g)).to(dtype)
    k = torch.randn(total, hkv, d, generator=g).to(dtype)
    return q, k, torch.tensor([0] + lens).cumsum(0).to(torch.int32)


def _check(q, k, cu, got, last=None, scale=None):
    want, reach = oracle.prompt(q.double().numpy(), k.double().numpy(), cu.tolist(), got.shape[2], last, scale)
    d = q.shape[2]
    # A score: D products in fp32 and a few roundings; a weight: its own score's and its row sum's error.  The sums over
    # queries and heads are of positive terms: a row's sum takes up to 2500 / 32 additions one after the other, a
    # column's 512 / 4 within a range and one for each of the ranges and heads, together under 2^8 halves of a step.
    rel = 2 * (d + 8) * 2.0 ** -24 * (reach + 8) + 2.0 ** -16
    got = got.double().cpu().numpy()
    assert (np.abs(got - want) <= want * rel + 2.0 ** -60).all(), np.nanmax(np.abs(got - want) / (want * rel + 2.0 ** -60))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 1), (5, 1), (8, 2)])
@pytest.mark.parametrize("last", [None, 1, 64, 77])
def test_ragged_prompts(dtype, d, hq, hkv, last):
    lens = [1, 0, 63, 64, 65, 300, 0, 129]
    q, k, cu = _case(lens, hq, hkv, d, dtype, seed=hq)
    w = torch.full((len(lens), hkv, 310), float("nan"), device="cuda")
    ak.prompt_weights(q.cuda(), k.cuda(), cu.cuda(), 300, w, last=last)
    _check(q, k, cu, w, last)


@pytest.mark.parametrize("lens", [[1], [2], [31], [32], [33], [255], [256], [257], [1111], [2500, 7]])
def test_lengths(lens):
    q, k, cu = _case(lens, 4, 2, 128, torch.float16, seed=lens[0])
    for last in (None, 16, max(1, lens[0] // 2), 10 * lens[0]):
        w = torch.full((len(lens), 2, max(lens)), float("nan"), device="cuda")
        ak.prompt_weights(q.cuda(), k.cuda(), cu.cuda(), max(lens), w, last=last)
        _check(q, k, cu, w, last)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_scales_and_large_scores(scale):
    q, k, cu = _case([400], 2, 1, 64, torch.float16, seed=1, spread=2.0)
    w = torch.empty(1, 1, 400, device="cuda")
    ak.prompt_weights(q.cuda(), k.cuda(), cu.cuda(), 400, w, scale=scale)
    _check(q, k, cu, w, scale=scale)


def test_growing_scores():
    """Later keys score far above earlier ones (past 2^80 of the first tile's), and far below."""
    for sign in (1.0, -1.0):
        q, k, cu = _case([500], 1, 1, 64, torch.float16, seed=2)
        q = q.abs()
        k = (k.abs() * (torch.arange(500)[:, None, None] / 250 * sign)).half()
        w = torch.empty(1, 1, 500, device="cuda")
        ak.prompt_weights(q.cuda(), k.cuda(), cu.cuda(), 500, w, scale=1.0)
        want, reach = oracle.prompt(q.double().numpy(), k.double().numpy(), cu.tolist(), 500, scale=1.0)
        rel = 2 * 72 * 2.0 ** -24 * (reach + 8) + 2.0 ** -18
        assert (np.abs(w.double().cpu().numpy() - want) <= want * rel + 2.0 ** -60).all()


def test_keys_of_minus_infinity_weigh_nothing():
    q, k, cu = _case([200], 2, 1, 64, torch.bfloat16, seed=3)
    q = q.abs()
    k[[3, 50, 199]] = -float("inf")
    k[100:170] = -float("inf")
    w = torch.empty(1, 1, 200, device="cuda")
    ak.prompt_weights(q.cuda(), k.cuda(), cu.cuda(), 200, w)
    _check(q, k, cu, w)
    assert not w[0, 0, 100:170].any()


def test_first_keys_of_minus_infinity_leave_rows_empty():
    """Queries that see only keys of -inf give nothing; the others go on."""
    q, k, cu = _case([150], 1, 1, 64, torch.float16, seed=4)
    q = q.abs()
    k[:70] = -float("inf")
    w = torch.empty(1, 1, 150, device="cuda")
    ak.prompt_weights(q.cuda(), k.cuda(), cu.cuda(), 150, w)
    assert not w.isnan().any() and not w[0, 0, :70].any()
    assert abs(float(w.sum()) - 80) < 80 * 2.0 ** -16


def test_slices_of_a_fused_projection_and_views_of_weights():
    lens, hq, hkv, d = [130, 64], 4, 2, 128
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(194, (hq + 2 * hkv) * d, generator=g).half()
    q, k = qkv[:, :hq * d].view(194, hq, d), qkv[:, hq * d:(hq + hkv) * d].view(194, hkv, d)
    gpu = qkv.cuda()
    gq, gk = gpu[:, :hq * d].view(194, hq, d), gpu[:, hq * d:(hq + hkv) * d].view(194, hkv, d)
    cu = torch.tensor([0, 130, 194], dtype=torch.int32)
    big = torch.full((hkv, 4, 150), 9.0, device="cuda")
    view = big[:, 1:3, :140].transpose(0, 1)
    ak.prompt_weights(gq, gk, cu, 130, view)  # a host cu_seqlens is checked and copied
    _check(q, k, cu, view)
    assert (big[:, 0] == 9).all() and (big[:, 3] == 9).all() and (big[:, :, 140:] == 9).all()
    apart = gq.transpose(0, 1).contiguous().transpose(0, 1)
    again = torch.empty_like(view)
    ak.prompt_weights(apart, gk, cu.cuda().long(), 130, again)
    assert torch.equal(again, view)


def test_inconsistent_offsets_stay_in_bounds():
    """A device cu_seqlens is used as given: starts past the rows, falling offsets, lengths past max_seqlen."""
    q, k, _ = _case([100], 2, 1, 64, torch.float16, seed=6)
    w = torch.full((4, 1, 80), float("nan"), device="cuda")
    ak.prompt_weights(q.cuda(), k.cuda(), torch.tensor([-5, 300, 20, 90, 95], dtype=torch.int32, device="cuda"), 64, w)
    torch.cuda.synchronize()
    assert not w.isnan().any() and not w[1].any()
    want, _ = oracle.prompt(q[90:95].double().numpy(), k[90:95].double().numpy(), [0, 5], 80)
    assert np.allclose(w[3].double().cpu().numpy(), want[0], rtol=2 ** -14)


def test_nothing_to_do():
    w = torch.full((3, 2, 8), 5.0, device="cuda")
    none = torch.empty(0, 4, 64, device="cuda").half()
    ak.prompt_weights(none, none[:, :2], torch.zeros(4, dtype=torch.int32, device="cuda"), 0, w)
    assert not w.any()
    ak.prompt_weights(none, none[:, :2], torch.zeros(1, dtype=torch.int32, device="cuda"), 0, w[:0])


def test_many_ranges_and_splits_agree_with_one():
    """Prompts long enough for several query ranges and key splits; a prompt's weights do not depend on its batch but
    for rounding."""
    q, k, cu = _case([2300], 4, 2, 64, torch.float16, seed=7)
    w = torch.empty(1, 2, 2300, device="cuda")
    ak.prompt_weights(q.cuda(), k.cuda(), cu.cuda(), 2300, w)
    _check(q, k, cu, w)
    cu2 = torch.tensor([0, 2300] + [2300] * 40, dtype=torch.int32)
    w2 = torch.empty(41, 2, 2300, device="cuda")
    ak.prompt_weights(q.cuda(), k.cuda(), cu2.cuda(), 2300, w2)
    _check(q, k, cu, w2[:1])
    assert not w2[1:].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
def test_long_prompts(dtype, d):
    """Enough work for 64 columns a wave."""
    lens = [2000, 1]
    q, k, cu = _case(lens, 32, 2, d, dtype, seed=d)
    w = torch.full((2, 2, 2005), float("nan"), device="cuda")
    ak.prompt_weights(q.cuda(), k.cuda(), cu.cuda(), 2000, w)
    _check(q, k, cu, w)


@pytest.mark.parametrize("hq,hkv,last", [(64, 8, 77), (64, 64, 100), (64, 16, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_prompts(hq, hkv, last, dtype):
    """64 columns a wave for a few queries of each of 41 prompts: several heads' queries in one stream, and a stream of
    all of them, which writes the weights itself.  max_seqlen is a bound far above the lengths."""
    lens = [300, 0, 1, 65, 64, 63, 256, 257] + [123 + 6 * i for i in range(31)] + [0, 281]
    q, k, cu = _case(lens, hq, hkv, 64, dtype, seed=hkv)
    w = torch.full((41, hkv, 2500), float("nan"), device="cuda")
    ak.prompt_weights(q.cuda(), k.cuda(), cu.cuda(), 1000, w, last=last)
    _check(q, k, cu, w, last)


@pytest.mark.parametrize("last", [1, 64, 512])
def test_one_stream_writes_all_of_the_weights(last):
    """One query head per kv head and few queries: no sums to add, and zeros behind the prompts all the same."""
    lens = [300, 0, 129, 1]
    q, k, cu = _case(lens, 3, 3, 128, torch.float16, seed=last)
    big = torch.full((4, 3, 1010), float("nan"), device="cuda")
    ak.prompt_weights(q.cuda(), k.cuda(), cu.cuda(), 300, big[:, :, :1001], last=last)
    _check(q, k, cu, big[:, :, :1001], last)
    assert big[:, :, 1001:].isnan().all()
