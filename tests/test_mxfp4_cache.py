"""The 4-bit paged cache's writer and reader against the float64 oracle.  The
format leaves no freedom, so codes, scales and values are compared exactly."""
import numpy as np
import pytest
import torch

import attnkernels as ak
from oracle import small_cache as oracle

pytestmark = pytest.mark.gpu


def _caches(blocks, hkv, bs, d, fill=0xA5):
    return [torch.full((blocks, hkv, bs, w), fill, dtype=torch.uint8, device="cuda") for w in (d // 2, d // 32) * 2]


def _check(key, value, slots, caches, before):
    """caches hold the oracle's rows at the slots, and what they held before elsewhere."""
    blocks, hkv, bs = caches[0].shape[:3]
    want = [c.cpu().numpy() for c in before]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * bs:
            for i, x in ((0, key), (2, value)):
                want[i][s // bs, :, s % bs], want[i + 1][s // bs, :, s % bs] = oracle.mxfp4_encode(
                    x[t].double().cpu().numpy())
    for got, w in zip(caches, want):
        assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,hkv,d,blocks,bs", [(1, 8, 128, 4, 16), (37, 8, 128, 64, 16), (300, 32, 128, 40, 16),
                                               (129, 4, 64, 50, 16), (64, 2, 32, 30, 12), (17, 3, 96, 9, 5), (5, 1, 512, 3, 2)])
def test_writes_what_the_oracle_says(dtype, T, hkv, d, blocks, bs):
    g = torch.Generator(device="cuda").manual_seed(T)
    key, value = (torch.randn(T, hkv, d, generator=g, device="cuda") *
                  torch.exp2(torch.randint(-12, 9, (T, hkv, 1), generator=g, device="cuda")) for _ in range(2))
    key, value = key.to(dtype), value.to(dtype)
    caches = _caches(blocks, hkv, bs, d)
    before = [c.clone() for c in caches]
    slots = torch.randperm(blocks * bs, generator=torch.Generator().manual_seed(T))[:T].cuda()
    ak.reshape_and_cache_mxfp4(key, value, *caches, slots)
    _check(key, value, slots, caches, before)
    back = ak.gather_cache_mxfp4(*caches, slots, dtype)
    for x, got in ((key, back[0]), (value, back[1])):
        want = oracle.mxfp4_decode(*oracle.mxfp4_encode(x.double().cpu().numpy()))
        assert got.dtype == dtype and np.array_equal(got.double().cpu().numpy(), torch.from_numpy(want).to(dtype).double())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_value_of_the_type(dtype):
    """All 65536 bit patterns, each beside a group top that gives it a scale: itself, and tops of 2^k and 1.75 2^k
    around it (ties, the step at 7, subnormals, infinities and NaN)."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    tops = torch.tensor([0.0, 1.0, 1.75, 8.0, 2.0 ** -10, 1.75 * 2.0 ** -6, 2.0 ** -14, 2.0 ** 12])
    rows = torch.zeros(65536, 8, 32, dtype=dtype)
    rows[:, :, 3] = bits[:, None]
    rows[:, :, 17] = tops.to(dtype)
    key = rows.cuda().contiguous()
    value = -key
    caches = _caches(4096, 8, 16, 32)
    before = [c.clone() for c in caches]
    slots = torch.arange(65536).cuda()
    ak.reshape_and_cache_mxfp4(key, value, *caches, slots)
    for i, x in ((0, key), (2, value)):
        codes, scales = oracle.mxfp4_encode(x.double().cpu().numpy())
        got_c, got_s = (caches[j].cpu().transpose(1, 2).reshape(65536, 8, -1).numpy() for j in (i, i + 1))
        assert np.array_equal(got_s, scales)
        # zeros may keep either sign; every other code is the oracle's
        wrong = got_c != codes
        low, high = ((got_c ^ codes) & 15), ((got_c ^ codes) >> 4)
        assert not wrong.any() or (((low == 0) | ((low == 8) & (codes & 7 == 0))) &
                                   ((high == 0) | ((high == 8) & (codes >> 4 & 7 == 0)))).all()
    assert before[0].shape == caches[0].shape


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_reads_every_code_and_scale(dtype):
    """Every code with every scale byte, read as the values rounded to the type."""
    codes = torch.arange(16, dtype=torch.uint8).repeat(2)  # 32 channels: each code twice
    packed = (codes[0::2] | codes[1::2] << 4).expand(256, 16).reshape(16, 1, 16, 16).contiguous().cuda()
    scales = torch.arange(256, dtype=torch.uint8).reshape(16, 1, 16, 1).contiguous().cuda()
    slots = torch.arange(256).cuda()
    key, value = ak.gather_cache_mxfp4(packed, scales, packed, scales, slots, dtype)
    want = oracle.mxfp4_decode(packed.cpu().numpy().reshape(256, 16), scales.cpu().numpy().reshape(256, 1))
    want = torch.from_numpy(want).to(dtype)
    assert torch.equal(torch.nan_to_num(key.cpu().float()[:, 0], nan=7.5), torch.nan_to_num(want.float(), nan=7.5))
    assert torch.equal(key.view(torch.int16), value.view(torch.int16))


def test_strided_rows_padding_and_int32_slots():
    T, hkv, d = 50, 8, 128
    qkv = torch.randn(T, 5, hkv, d, device="cuda").half()
    key, value = qkv[:, 1], qkv[:, 3]
    for slots in (torch.arange(3, 3 + T, device="cuda"), torch.arange(3, 3 + T, dtype=torch.int32)):
        slots = slots.clone()
        slots[[0, 7]] = -1
        slots[9] = 8 * 16
        caches = _caches(8, hkv, 16, d)
        before = [c.clone() for c in caches]
        ak.reshape_and_cache_mxfp4(key, value, *caches, slots)
        _check(key, value, slots, caches, before)
        k, v = ak.gather_cache_mxfp4(*caches, slots)
        assert not k[[0, 7, 9]].any() and not v[[0, 7, 9]].any() and k[1].any()
    # rows that are not on 16 bytes, and heads apart
    odd = torch.randn(T * hkv * d + 1, device="cuda").half()[1:].view(T, hkv, d)
    apart = torch.randn(hkv, T, d, device="cuda").half().transpose(0, 1)
    caches = _caches(8, hkv, 16, d)
    before = [c.clone() for c in caches]
    slots = torch.arange(T, device="cuda")
    ak.reshape_and_cache_mxfp4(odd, apart, *caches, slots)
    _check(odd, apart, slots, caches, before)


def test_no_tokens():
    caches = _caches(2, 2, 16, 64)
    none = torch.empty(0, 2, 64, device="cuda", dtype=torch.float16)
    ak.reshape_and_cache_mxfp4(none, none, *caches, torch.empty(0, dtype=torch.int64, device="cuda"))
    key, value = ak.gather_cache_mxfp4(*caches, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert key.shape == value.shape == (0, 2, 64) and (caches[0] == 0xA5).all()
