"""The C entry points of the 4-bit cache, attention weights and eviction on device
memory, against the same operators of the Python interface."""
import ctypes
import pathlib

import numpy as np
import pytest
import torch

import attnkernels as ak
from test_decode_mx import Case

pytestmark = pytest.mark.gpu

LIB = pathlib.Path(ak.__file__).parent / "libattnkernels.so"
vp, i64, f64, c_int, size = ctypes.c_void_p, ctypes.c_int64, ctypes.c_double, ctypes.c_int, ctypes.c_size_t


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(str(LIB))
    L.ak_last_error.restype = ctypes.c_char_p
    L.ak_reshape_and_cache_mxfp4.argtypes = [vp] * 7 + [i64] * 7 + [c_int, vp]
    L.ak_gather_cache_mxfp4.argtypes = [vp] * 7 + [i64] * 5 + [c_int, vp]
    L.ak_paged_decode_mx_workspace_size.argtypes = [i64] * 6 + [c_int]
    L.ak_paged_decode_mx_workspace_size.restype = size
    L.ak_paged_decode_mxfp4.argtypes = [vp] * 9 + [i64] * 11 + [f64, i64, c_int, vp, size, vp, i64, vp]
    L.ak_paged_decode_weights.argtypes = [vp] * 7 + [i64] * 11 + [f64, i64, c_int, vp, size, vp]
    L.ak_prompt_weights_workspace_size.argtypes = [i64] * 7
    L.ak_prompt_weights_workspace_size.restype = size
    L.ak_prompt_weights.argtypes = [vp] * 4 + [i64] * 12 + [f64, c_int, vp, size, vp]
    L.ak_evict_cache.argtypes = [vp] * 2 + [i64] + [vp] * 2 + [i64] + [vp] * 4 + [i64] * 3 + [vp] * 3 + [i64] * 8 + [vp]
    return L


def ptr(t):
    return vp(t.data_ptr()) if t is not None else None


def stream():
    return vp(torch.cuda.current_stream().cuda_stream)


def check(lib, rc):
    assert rc == 0, lib.ak_last_error()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_writer_and_reader(lib, dtype):
    g = torch.Generator().manual_seed(0)
    key, value = (torch.randn(40, 3, 64, generator=g).to(dtype).cuda() for _ in range(2))
    slots = torch.randperm(96, generator=g)[:40].cuda()
    slots[7] = -1
    caches = [torch.zeros(6, 3, 16, n, dtype=torch.uint8, device="cuda") for n in (32, 2, 32, 2)]
    other = [x.clone() for x in caches]
    ak.reshape_and_cache_mxfp4(key, value, *other, slots)
    bf = int(dtype == torch.bfloat16)
    check(lib, lib.ak_reshape_and_cache_mxfp4(ptr(key), ptr(value), *map(ptr, caches), ptr(slots), 40, 3, 64, 6, 16, 192,
                                              192, bf, stream()))
    assert all(torch.equal(x, y) for x, y in zip(caches, other))
    k, v = torch.empty_like(key), torch.empty_like(value)
    check(lib, lib.ak_gather_cache_mxfp4(*map(ptr, caches), ptr(slots), ptr(k), ptr(v), 40, 3, 64, 6, 16, bf, stream()))
    k2, v2 = ak.gather_cache_mxfp4(*other, slots, dtype)
    assert torch.equal(k, k2) and torch.equal(v, v2)


@pytest.mark.parametrize("partition", [0, 256])
@pytest.mark.parametrize("fmt,counters,tracked", [("mxfp4", False, False), ("mxfp4", True, False), ("mxfp4", False, True),
                                                  ("mxfp4", True, True), ("full", False, True)])
def test_decode(lib, fmt, counters, tracked, partition):
    """Without counters a second kernel merges the splits, of sequences with several of them, one, or no token."""
    c = Case([2000, 0, 100, 256, 700], 2, 4, 64, fmt=fmt, seed=partition)
    q, tables = c.gpu(c.q, torch.float16), c.gpu(c.tables)
    lens = c.gpu(np.array(c.lens, dtype=np.int32))
    out = torch.full_like(q, float("nan"))
    w = c.gpu(c.weights) if tracked else None
    need = lib.ak_paged_decode_mx_workspace_size(5, 8, 2, 64, 2000, partition, int(tracked))
    assert need > 0
    workspace = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    count = torch.zeros(10, dtype=torch.int32, device="cuda") if counters else None
    sizes = [*(w.stride()[:2] if tracked else (0, 0)), w.shape[2] if tracked else 0, 5, 8, 2, 64,
             c.caches[0].shape[0], 16, tables.shape[1], 2000]
    for _ in range(2):  # the counters are left at zero
        if tracked:
            w.copy_(c.gpu(c.weights))
        if fmt == "mxfp4":
            rc = lib.ak_paged_decode_mxfp4(ptr(q), *map(ptr, c.caches), ptr(tables), ptr(lens), ptr(out), ptr(w), *sizes,
                                           64 ** -0.5, partition, 0, ptr(workspace), need, ptr(count),
                                           10 if counters else 0, stream())
        else:
            rc = lib.ak_paged_decode_weights(ptr(q), *map(ptr, c.caches), ptr(tables), ptr(lens), ptr(out), ptr(w),
                                             *sizes, 64 ** -0.5, partition, 0, ptr(workspace), need, stream())
        check(lib, rc)
        c.check(out, w, c.weights)
    assert (workspace[need:] == 0xFF).all()


@pytest.mark.parametrize("last", [64, 1000])
def test_prompt(lib, last):
    g = torch.Generator().manual_seed(last)
    q, k = (torch.randn(700, h, 128, generator=g).half().cuda() for h in (4, 2))
    cu = torch.tensor([0, 600, 600, 700], dtype=torch.int32, device="cuda")
    want = torch.empty(3, 2, 640, device="cuda")
    ak.prompt_weights(q, k, cu, 600, want, last=last)
    got = torch.full_like(want, float("nan"))
    need = lib.ak_prompt_weights_workspace_size(3, 700, 4, 2, 128, 600, last)
    workspace = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    check(lib, lib.ak_prompt_weights(ptr(q), ptr(k), ptr(cu), ptr(got), *got.stride()[:2], 640, 3, 700, 4, 2, 128, 512,
                                     256, 600, last, 128 ** -0.5, 0, ptr(workspace), need, stream()))
    assert torch.equal(got, want) and (workspace[need:] == 0xFF).all()


@pytest.mark.parametrize("fmt", ["mxfp4", "full"])
def test_eviction(lib, fmt):
    c = Case([300, 20, 0, 129], 2, 1, 64, fmt=fmt, seed=3)
    tables, lens = c.gpu(c.tables), c.gpu(np.array(c.lens, dtype=np.int32))
    w = c.gpu(c.weights)
    mine = [x.clone() for x in c.caches]
    how = dict(k_scales=c.caches[1], v_scales=c.caches[3]) if fmt == "mxfp4" else {}
    values = c.caches[::2] if fmt == "mxfp4" else c.caches
    want = ak.evict_cache(*values, tables, lens, w, 100, 30, **how)
    new_lens, kept = torch.full_like(lens, -7), torch.full((4, 2, 100), -7, dtype=torch.int32, device="cuda")
    new_w = torch.full_like(w, float("nan"))
    if fmt == "mxfp4":
        rows = [ptr(mine[0]), ptr(mine[2]), 32, ptr(mine[1]), ptr(mine[3]), 2]
    else:
        rows = [ptr(mine[0]), ptr(mine[1]), 128, None, None, 0]
    check(lib, lib.ak_evict_cache(*rows, ptr(tables), None, ptr(lens), ptr(w), *w.stride()[:2], w.shape[2], ptr(new_lens), ptr(new_w),
                                  ptr(kept), 4, 2, mine[0].shape[0], 16, tables.shape[1], 0, 100, 30, stream()))
    assert torch.equal(new_lens, want[0]) and torch.equal(new_w, want[1]) and torch.equal(kept, want[2])
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(mine, c.caches))
