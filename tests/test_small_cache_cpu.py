"""The smaller cache without a GPU: the float64 oracle against brute force, the
entry points' refusals (they check shapes before devices), the C-ABI's."""
import ctypes

import numpy as np
import pytest
import torch

import attnkernels as ak
from conftest import PKG_DIR
from oracle import small_cache as oracle


# --- the oracle -------------------------------------------------------------------------------------------------------


def test_codes_are_the_nearest_values():
    r = np.random.default_rng(0)
    x = r.standard_normal((200, 64)) * np.exp2(r.integers(-20, 20, (200, 1)))
    codes, scales = oracle.mxfp4_encode(x)
    got = oracle.mxfp4_decode(codes, scales)
    grid = np.concatenate((oracle.FP4, -oracle.FP4))
    factor = np.repeat(np.exp2(scales.astype(float) - 127), 32, axis=-1)
    best = np.abs(x[..., None] - grid * factor[..., None]).min(-1)
    assert np.array_equal(np.abs(x - got), best)
    # a group's largest magnitude is below 7 steps, and at least 3.5: no smaller scale would hold it
    top = (np.abs(x) / factor).reshape(200, 2, 32).max(-1)
    assert top.max() < 7 and top.min() >= 3.5


def test_ties_go_to_the_even_code_and_the_scale_rounds_up_at_seven():
    x = np.zeros((1, 32))
    x[0, :8] = [4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -5]
    codes, scales = oracle.mxfp4_encode(x)
    assert oracle.mxfp4_decode(codes, scales)[0, :8].tolist() == [4, 0, 1, 1, 2, 2, 4, -4] and scales[0, 0] == 127
    for top, want in ((6.9, 127), (7.0, 128), (0.0, 1), (np.inf, 255), (np.nan, 255)):
        x[0] = 0
        x[0, 5] = top
        assert oracle.mxfp4_encode(x)[1][0, 0] == want


def test_rows_survive_a_second_rounding():
    """A stored value is its own rounding, unless its group's top came down (7 and below to 6: the scale stays)."""
    r = np.random.default_rng(1)
    once = oracle.mxfp4_decode(*oracle.mxfp4_encode(r.standard_normal((50, 128))))
    assert np.array_equal(oracle.mxfp4_decode(*oracle.mxfp4_encode(once)), once)


def test_keep_by_brute_force():
    r = np.random.default_rng(2)
    for _ in range(200):
        n, budget = int(r.integers(1, 12)), int(r.integers(1, 12))
        recent = int(r.integers(0, budget + 1))
        w = r.integers(0, 4, n).astype(float)
        got = oracle.keep(w, budget, recent).tolist()
        if n <= budget:
            assert got == list(range(n))
            continue
        assert len(got) == budget and got == sorted(set(got)) and got[budget - recent:] == list(range(n - recent, n))
        for i in range(n - recent):  # no token left out is heavier, or as heavy and before one kept
            if i not in got:
                assert all(w[j] > w[i] or (w[j] == w[i] and j < i) for j in got[:budget - recent])


def test_prompt_weights_sum_to_the_queries():
    r = np.random.default_rng(3)
    q, k = r.standard_normal((20, 4, 64)), r.standard_normal((20, 2, 64))
    w, _ = oracle.prompt(q, k, [0, 13, 13, 20], 16)
    assert np.allclose(w.sum(-1), [[26, 26], [0, 0], [14, 14]])
    w, _ = oracle.prompt(q, k, [0, 13, 13, 20], 16, last=5)
    assert np.allclose(w.sum(-1), [[10, 10], [0, 0], [10, 10]]) and (w[0, :, 13:] == 0).all()


# --- refusals ---------------------------------------------------------------------------------------------------------


def _mx(blocks=4, hkv=2, bs=16, d=64):
    u8 = dict(dtype=torch.uint8)
    return [torch.zeros(blocks, hkv, bs, w, **u8) for w in (d // 2, d // 32, d // 2, d // 32)]


def _rows(t=3, hkv=2, d=64, dtype=torch.float16):
    return torch.zeros(t, hkv, d, dtype=dtype)


SLOTS = torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize("message,key,value,caches,slots", [
    ("same shape", _rows(), _rows(4), _mx(), SLOTS),
    ("same shape", _rows()[0], _rows()[0], _mx(), SLOTS),
    ("both be fp16", _rows(dtype=torch.float32), _rows(dtype=torch.float32), _mx(), SLOTS),
    ("both be fp16", _rows(), _rows(dtype=torch.bfloat16), _mx(), SLOTS),
    ("multiple of 32", _rows(d=48), _rows(d=48), _mx(), SLOTS),
    ("uint8", _rows(), _rows(), [c.to(torch.int8) for c in _mx()], SLOTS),
    ("same shape", _rows(), _rows(), _mx(d=128), SLOTS),
    ("scales must be", _rows(), _rows(), _mx()[:1] + _mx(d=128)[1:2] + _mx()[2:], SLOTS),
    ("contiguous", _rows(), _rows(), [_mx(hkv=4)[0][:, ::2]] + _mx()[1:], SLOTS),
    ("kv heads of key", _rows(hkv=1), _rows(hkv=1), _mx(), SLOTS),
    ("num_tokens", _rows(), _rows(), _mx(), SLOTS[:2]),
    ("GPU tensors", _rows(), _rows(), _mx(), SLOTS),
])
def test_write_refusals(message, key, value, caches, slots):
    with pytest.raises(ValueError, match=message):
        ak.reshape_and_cache_mxfp4(key, value, *caches, slots)


def test_gather_refusals():
    with pytest.raises(ValueError, match="float16 or torch.bfloat16"):
        ak.gather_cache_mxfp4(*_mx(), SLOTS, torch.float32)
    with pytest.raises(ValueError, match="num_tokens"):
        ak.gather_cache_mxfp4(*_mx(), SLOTS[None])
    with pytest.raises(ValueError, match="GPU tensors"):
        ak.gather_cache_mxfp4(*_mx(), SLOTS)


def _decode_args(**over):
    a = dict(q=_rows(2, 4), k=torch.zeros(4, 2, 16, 64, dtype=torch.float16), tables=torch.zeros(2, 3, dtype=torch.int32),
             lens=torch.ones(2, dtype=torch.int32), longest=40, weights=torch.zeros(2, 2, 48))
    a["v"] = a["k"]
    a.update(over)
    return a


DECODE_REFUSALS = [
    ("fp16 or bf16", dict(q=_rows(2, 4, dtype=torch.float32))),
    ("head_dim must be 64 or 128", dict(q=_rows(2, 4, 96))),
    ("block_tables", dict(tables=torch.zeros(3, 3, dtype=torch.int32))),
    ("integers", dict(tables=torch.zeros(2, 3))),
    ("context_lens", dict(lens=torch.ones(2, 1, dtype=torch.int32))),
    (r"weights must be float32 \[B, H_kv", dict(weights=torch.zeros(2, 4, 48))),
    (r"weights must be float32 \[B, H_kv", dict(weights=torch.zeros(2, 2, 48, dtype=torch.float64))),
    ("at least as long", dict(weights=torch.zeros(2, 2, 39))),
    ("last dimension", dict(weights=torch.zeros(2, 2, 96)[:, :, ::2])),
    ("GPU tensors", dict()),
]


@pytest.mark.parametrize("message,over", DECODE_REFUSALS)
def test_decode_refusals(message, over):
    a = _decode_args(**over)
    with pytest.raises(ValueError, match=message):
        ak.paged_decode_weights(a["q"], a["k"], a["v"], a["tables"], a["lens"], a["longest"], a["weights"])
    with pytest.raises(ValueError, match=message):
        d = a["q"].shape[2] if a["q"].shape[2] != 96 else 64
        ak.paged_decode_mxfp4(a["q"], *_mx(d=d), a["tables"], a["lens"], a["longest"], weights=a["weights"])


def test_decode_cache_refusals():
    a = _decode_args()
    for k, v, message in ((a["k"].bfloat16(), a["k"], "all be fp16"), (a["k"][..., :32], a["v"][..., :32], "matching q"),
                          (a["k"], a["v"][:3], "matching q"), (a["k"].transpose(0, 1), a["v"].transpose(0, 1), "contiguous")):
        with pytest.raises(ValueError, match=message):
            ak.paged_decode_weights(a["q"], k, v, a["tables"], a["lens"], 40, a["weights"])


@pytest.mark.parametrize("message,over", [
    ("both fp16 or both bf16", dict(q=_rows(10, 4, dtype=torch.float32))),
    ("total and D of q", dict(k=_rows(9))),
    ("multiple of the kv heads", dict(k=_rows(10, 3))),
    ("head_dim must be 64 or 128", dict(q=_rows(10, 4, 96), k=_rows(10, 2, 96))),
    ("integers", dict(cu=torch.tensor([0.0, 10.0]))),
    ("non-decreasing", dict(cu=torch.tensor([0, 12]))),
    ("non-decreasing", dict(cu=torch.tensor([4, 2]))),
    ("shorter than a sequence", dict(longest=9)),
    ("at least 1", dict(last=0)),
    (r"weights must be float32 \[B, H_kv", dict(weights=torch.zeros(2, 2, 16))),
    ("at least as long", dict(weights=torch.zeros(1, 2, 9))),
    ("GPU tensors", dict()),
])
def test_prompt_refusals(message, over):
    a = dict(q=_rows(10, 4), k=_rows(10), cu=torch.tensor([0, 10]), longest=10, weights=torch.zeros(1, 2, 16), last=None)
    a.update(over)
    with pytest.raises(ValueError, match=message):
        ak.prompt_weights(a["q"], a["k"], a["cu"], a["longest"], a["weights"], last=a["last"])


@pytest.mark.parametrize("message,over", [
    ("budget", dict(budget=0)),
    ("budget", dict(recent=-1)),
    ("budget", dict(budget=4, recent=5)),
    ("both be fp16", dict(k=torch.zeros(4, 2, 16, 32, dtype=torch.uint8), v=torch.zeros(4, 2, 16, 32, dtype=torch.uint8))),
    ("come together", dict(ks=torch.zeros(4, 2, 16, 2, dtype=torch.uint8))),
    ("contiguous", dict(k=torch.zeros(4, 4, 16, 64).half()[:, ::2], v=torch.zeros(4, 4, 16, 64).half()[:, ::2])),
    ("multiple of 16 bytes", dict(k=torch.zeros(4, 2, 16, 12).half(), v=torch.zeros(4, 2, 16, 12).half())),
    ("weights must be float32", dict(weights=torch.zeros(3, 2, 48))),
    ("integers", dict(lens=torch.ones(2))),
    ("pages for budget", dict(new=torch.zeros(2, 1, dtype=torch.int32))),
    ("GPU tensors", dict()),
])
def test_evict_refusals(message, over):
    a = _decode_args(budget=20, recent=4, ks=None, vs=None, new=None)
    a.update(over)
    with pytest.raises(ValueError, match=message):
        ak.evict_cache(a["k"], a["v"], a["tables"], a["lens"], a["weights"], a["budget"], a["recent"], a["ks"], a["vs"],
                       a["new"])


# --- the C-ABI: every call below is refused before it touches a GPU ------------------------------------------------------

FAKE = 4096
vp, i64, f64, sz, ci = ctypes.c_void_p, ctypes.c_int64, ctypes.c_double, ctypes.c_size_t, ctypes.c_int


@pytest.fixture(scope="module")
def lib():
    ak.load_extension()
    L = ctypes.CDLL(str(PKG_DIR / "attnkernels" / "libattnkernels.so"))
    L.ak_last_error.restype = ctypes.c_char_p
    L.ak_reshape_and_cache_mxfp4.argtypes = [vp] * 7 + [i64] * 7 + [ci, vp]
    L.ak_gather_cache_mxfp4.argtypes = [vp] * 7 + [i64] * 5 + [ci, vp]
    L.ak_paged_decode_mx_workspace_size.argtypes = [i64] * 6 + [ci]
    L.ak_paged_decode_mx_workspace_size.restype = sz
    L.ak_paged_decode_mxfp4.argtypes = [vp] * 9 + [i64] * 11 + [f64, i64, ci, vp, sz, vp, i64, vp]
    L.ak_paged_decode_weights.argtypes = [vp] * 7 + [i64] * 11 + [f64, i64, ci, vp, sz, vp]
    L.ak_prompt_weights_workspace_size.argtypes = [i64] * 7
    L.ak_prompt_weights_workspace_size.restype = sz
    L.ak_prompt_weights.argtypes = [vp] * 4 + [i64] * 12 + [f64, ci, vp, sz, vp]
    L.ak_evict_cache.argtypes = [vp] * 2 + [i64] + [vp] * 2 + [i64] + [vp] * 4 + [i64] * 3 + [vp] * 3 + [i64] * 8 + [vp]
    return L


def _refused(lib, rc, code, word):
    assert rc == code and word in lib.ak_last_error().decode(), (rc, lib.ak_last_error())


def _write(lib, name="ak_reshape_and_cache_mxfp4", **over):
    a = dict(key=FAKE, slots=FAKE, kc=FAKE, tokens=4, hkv=2, d=64, blocks=4, bs=16, stride=128)
    a.update(over)
    return lib.ak_reshape_and_cache_mxfp4(a["key"], FAKE, a["kc"], FAKE, FAKE, FAKE, a["slots"], a["tokens"], a["hkv"],
                                          a["d"], a["blocks"], a["bs"], a["stride"], 128, 0, None)


def test_capi_write_refusals(lib):
    for code, word, over in ((2, "multiple of 32", dict(d=40)), (2, "multiple of 32", dict(d=544)),
                             (1, "invalid size", dict(tokens=-1)), (1, "invalid size", dict(bs=0)),
                             (1, "null", dict(key=None)), (1, "null", dict(kc=None)), (1, "aligned", dict(key=FAKE + 8)),
                             (1, "aligned", dict(slots=FAKE + 4)), (1, "strides", dict(stride=120)),
                             (1, "strides", dict(stride=132)), (1, "out of range", dict(blocks=1 << 60))):
        _refused(lib, _write(lib, **over), code, word)
    assert _write(lib, tokens=0) == 0 and _write(lib, blocks=0) == 0


def _decode(lib, weights=FAKE, full=False, **over):
    a = dict(q=FAKE, ks=FAKE, wb=96, wh=48, wl=48, batch=2, hq=4, hkv=2, d=64, blocks=4, bs=16, mb=3, ctx=40, part=256,
             ws=FAKE, bytes=1 << 30, counters=None, ncount=0)
    a.update(over)
    head = [a["wb"], a["wh"], a["wl"], a["batch"], a["hq"], a["hkv"], a["d"], a["blocks"], a["bs"], a["mb"], a["ctx"], 1.0,
            a["part"], 0, a["ws"], a["bytes"]]
    if full:
        return lib.ak_paged_decode_weights(a["q"], FAKE, FAKE, FAKE, FAKE, FAKE, weights, *head, None)
    return lib.ak_paged_decode_mxfp4(a["q"], FAKE, a["ks"], FAKE, FAKE, FAKE, FAKE, FAKE, weights, *head, a["counters"],
                                     a["ncount"], None)


def test_capi_decode_refuses_misaligned_scales(lib):
    _refused(lib, _decode(lib, ks=FAKE + 2), 1, "scales must be 16-byte aligned")


@pytest.mark.parametrize("code,word,over", [
    (1, "multiple of num_kv_heads", dict(hq=5)), (1, "positive multiple of 256", dict(part=100)), (1, "positive multiple of 256", dict(part=-256)),
    (2, "at most 16", dict(hq=34)), (2, "head_dim", dict(d=32)), (1, "invalid size", dict(bs=0)),
    (1, "max_context_len", dict(ctx=0)), (1, "empty block table", dict(mb=0)), (1, "null", dict(q=None)),
    (1, "aligned", dict(q=FAKE + 2)), (1, "out of range", dict(ctx=1 << 31, wl=1 << 31, wh=1 << 31, wb=1 << 32)),
    (1, "out of range", dict(batch=65536)), (1, "shorter", dict(wl=39)), (1, "overlap", dict(wh=40)),
    (1, "overlap", dict(wb=0)), (1, "overlap", dict(wb=48)), (3, "bytes required", dict(bytes=64)),
    (1, "workspace must be", dict(ws=FAKE + 4)),
])
def test_capi_decode_refusals(lib, code, word, over):
    _refused(lib, _decode(lib, **over), code, word)
    _refused(lib, _decode(lib, full=True, **over), code, word)


def test_capi_decode_more_refusals(lib):
    _refused(lib, _decode(lib, ks=None), 1, "null")
    _refused(lib, _decode(lib, weights=None, full=True), 1, "null")
    _refused(lib, _decode(lib, weights=None, counters=FAKE, ncount=3), 1, "counters")
    _refused(lib, _decode(lib, weights=None, ctx=1000, bytes=64), 3, "bytes required")
    _refused(lib, _decode(lib, weights=None, ctx=1 << 29, part=256, bytes=1 << 62, batch=2000), 1, "splits")
    assert _decode(lib, batch=0) == 0
    for part in (0, 256):
        assert lib.ak_paged_decode_mx_workspace_size(2, 4, 2, 64, 40, part, 0) == 0
        assert lib.ak_paged_decode_mx_workspace_size(2, 4, 2, 64, 40, part, 1) >= 2 * 4 * (66 + 64) * 4
    assert lib.ak_paged_decode_mx_workspace_size(2, 4, 2, 64, 1000, 0, 0) > 0


def _prompt(lib, **over):
    a = dict(q=FAKE, cu=FAKE, w=FAKE, wb=32, wh=16, wl=16, batch=2, total=20, hq=4, hkv=2, d=64, qs=256, ks=128, longest=16,
             last=16, ws=FAKE, bytes=1 << 30)
    a.update(over)
    return lib.ak_prompt_weights(a["q"], FAKE, a["cu"], a["w"], a["wb"], a["wh"], a["wl"], a["batch"], a["total"], a["hq"],
                                 a["hkv"], a["d"], a["qs"], a["ks"], a["longest"], a["last"], 1.0, 0, a["ws"], a["bytes"],
                                 None)


@pytest.mark.parametrize("code,word,over", [
    (1, "multiple of num_kv_heads", dict(hq=3)), (2, "head_dim", dict(d=96)), (1, "invalid size", dict(last=0)),
    (1, "invalid size", dict(batch=-1)), (1, "shorter", dict(wl=15)), (1, "null", dict(q=None)), (1, "null", dict(w=None)),
    (1, "aligned", dict(q=FAKE + 8)), (1, "aligned", dict(cu=FAKE + 2)), (1, "strides", dict(qs=248)),
    (1, "strides", dict(ks=132)), (1, "out of range", dict(batch=65536)), (1, "overlap", dict(wh=8)),
    (3, "bytes required", dict(bytes=16)), (1, "workspace must be", dict(ws=FAKE + 4)),
])
def test_capi_prompt_refusals(lib, code, word, over):
    _refused(lib, _prompt(lib, **over), code, word)


def _evict(lib, **over):
    a = dict(k=FAKE, row=128, ks=None, vs=None, scale=0, new=None, w=FAKE, wb=96, wh=48, wl=48, kept=FAKE, batch=2, hkv=2,
             blocks=4, bs=16, mb=3, nmb=0, budget=20, recent=4)
    a.update(over)
    return lib.ak_evict_cache(a["k"], FAKE, a["row"], a["ks"], a["vs"], a["scale"], FAKE, a["new"], FAKE, a["w"], a["wb"],
                              a["wh"], a["wl"], FAKE, FAKE, a["kept"], a["batch"], a["hkv"], a["blocks"], a["bs"], a["mb"],
                              a["nmb"], a["budget"], a["recent"], None)


@pytest.mark.parametrize("code,word,over", [
    (1, "invalid size", dict(bs=0)), (1, "budget", dict(budget=0)), (1, "recent", dict(recent=21)),
    (2, "multiple of 16", dict(row=24)), (2, "multiple of 16", dict(row=2048)), (2, "scales", dict(ks=FAKE, vs=FAKE)),
    (1, "null", dict(k=None)), (1, "null", dict(ks=FAKE, scale=2)), (1, "aligned", dict(k=FAKE + 8)),
    (1, "aligned", dict(kept=FAKE + 2)), (1, "out of range", dict(budget=1 << 31)), (1, "overlap", dict(wh=1)),
    (1, "pages for budget", dict(new=FAKE, nmb=1)),
])
def test_capi_evict_refusals(lib, code, word, over):
    _refused(lib, _evict(lib, **over), code, word)
    assert _evict(lib, batch=0) == 0
