"""The calls of the smaller-cache operators whose speed is measured: the 4-bit
(MXFP4) paged cache and the decode over it, attention weights summed per cached
token by decode and prompt, and the eviction that goes by them.

``run`` makes the calls through the library's public entry points where ``own``
is true; otherwise it computes the same in elementary torch operations, in 32
bits.  Sizes are those of the library's own benchmark and tests, or generic:
32 or 64 query heads over 8 kv heads (or 32 over 32), pages of 16 tokens
scattered over a pool by a random permutation, as a paged allocator leaves them.

The 4-bit format: 32 channels of a token and head share a scale 2^e; a value is
a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6, the nearest to x / 2^e (ties to the
even code).  e is the exponent of the largest magnitude, rounded to two
significant bits, less 2.  Two channels share a byte, the even one in the low half.
"""
import math
import os
import random
import sys

import torch

own = False


def _ak():
    path = os.path.join(os.getcwd(), "flash-attention-from-scratch_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import attnkernels
    return attnkernels


def listed():
    return [
        # One decode step's new tokens of a full batch into the 4-bit cache, and their values back: latency.
        {"name": "write4_step", "kind": "write4", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "append": True, "dtype": "bfloat16"},
        # A batch of prompts' tokens, sliced from a fused projection.
        {"name": "write4_prompts", "kind": "write4", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "append": False, "dtype": "float16"},
        # One sequence's next token over the 4-bit cache: an interactive step's latency.
        {"name": "decode4_one", "kind": "decode", "format": "mxfp4", "tracked": False, "batch": 1, "heads": 32,
         "kv_heads": 8, "low": 1000, "high": 1000, "lens_seed": 0, "dim": 128, "page": 16, "dtype": "float16"},
        # The benchmark's grouped-query layer with a 4-bit cache, a full serving batch.
        {"name": "decode4_layer", "kind": "decode", "format": "mxfp4", "tracked": False, "batch": 16, "heads": 32,
         "kv_heads": 8, "low": 8192, "high": 8192, "lens_seed": 0, "dim": 128, "page": 16, "dtype": "float16"},
        # Very long contexts, one query head per kv head, head size 64, and the weights that eviction needs.
        {"name": "decode4_long_tracked", "kind": "decode", "format": "mxfp4", "tracked": True, "batch": 8,
         "heads": 32, "kv_heads": 32, "low": 32768, "high": 32768, "lens_seed": 0, "dim": 64, "page": 16,
         "dtype": "float16"},
        # A step of two short chats that keeps track of attention weights.
        {"name": "decode_weights_short", "kind": "decode", "format": "full", "tracked": True, "batch": 2, "heads": 32,
         "kv_heads": 8, "low": 700, "high": 1000, "lens_seed": 1, "dim": 128, "page": 16, "dtype": "bfloat16"},
        # Continuous batching over ragged long contexts, eight query heads per kv head.
        {"name": "decode_weights_group8", "kind": "decode", "format": "full", "tracked": True, "batch": 16,
         "heads": 64, "kv_heads": 8, "low": 512, "high": 8192, "lens_seed": 3, "dim": 128, "page": 16,
         "dtype": "float16"},
        # One chat prompt of odd length: every query counts.
        {"name": "prompt_weights_one", "kind": "prompt", "batch": 1, "heads": 32, "kv_heads": 8, "low": 1111,
         "high": 1111, "lens_seed": 0, "last": 0, "dim": 128, "dtype": "float16"},
        # Packed prompts of mixed lengths, of which the last 64 queries count.
        {"name": "prompt_weights_window", "kind": "prompt", "batch": 12, "heads": 32, "kv_heads": 8, "low": 64,
         "high": 4096, "lens_seed": 5, "last": 64, "dim": 128, "dtype": "bfloat16"},
        # One long prompt, every query counts: two passes of the scores' product.
        {"name": "prompt_weights_long", "kind": "prompt", "batch": 1, "heads": 32, "kv_heads": 8, "low": 8192,
         "high": 8192, "lens_seed": 0, "last": 0, "dim": 128, "dtype": "float16"},
        # One chat's 4-bit cache cut back to 1024 tokens.
        {"name": "evict_one", "kind": "evict", "format": "mxfp4", "batch": 1, "kv_heads": 8, "low": 1200,
         "high": 1200, "lens_seed": 0, "budget": 1024, "recent": 256, "dim": 128, "page": 16, "dtype": "float16"},
        # A serving batch's full-precision caches, contexts of all lengths cut back to 2048 tokens.
        {"name": "evict_batch", "kind": "evict", "format": "full", "batch": 16, "kv_heads": 8, "low": 1024,
         "high": 8192, "lens_seed": 2, "budget": 2048, "recent": 512, "dim": 128, "page": 16, "dtype": "float16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


# No drawn case costs more than the largest listed ones of its kind.
_MOST = {"write4": 1.5e8, "decode": 6.0e8, "prompt": 2.7e11, "evict": 2.5e8}


def draw(rng):
    kind = rng.choice(["write4", "decode", "decode", "decode", "prompt", "prompt", "evict"])
    while True:
        case = {"kind": kind, "dim": rng.choice([64, 128, 128]), "dtype": rng.choice(["float16", "bfloat16"]),
                "kv_heads": rng.choice([2, 4, 8, 8, 32])}
        case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
        if case["heads"] > 64:
            continue
        if kind == "write4":
            append = rng.random() < 0.4  # a decode step: one token per sequence
            case.update(tokens=_log_int(rng, 1, 256 if append else 16384), page=rng.choice([16, 16, 8, 12, 64]),
                        append=append)
        elif kind == "decode":
            high = _log_int(rng, 1, 32768)
            tracked = rng.random() < 0.6
            case.update(batch=_log_int(rng, 1, 64), high=high, low=rng.choice([high, high, 1 + high // 8, 0]),
                        lens_seed=rng.randrange(1 << 20), page=rng.choice([16, 16, 16, 8, 12, 32, 64]),
                        tracked=tracked, format=rng.choice(["mxfp4", "full"]) if tracked else "mxfp4")
            if case["batch"] * high * case["kv_heads"] * case["dim"] > 1 << 30:  # the plain form's padded rows
                continue
        elif kind == "prompt":
            high = _log_int(rng, 1, 8192)
            batch = _log_int(rng, 1, 16)
            last = rng.choice([0, 0, 16, 64, 77])
            case.update(batch=batch, high=high, low=rng.choice([high, 1 + high // 8, 0]),
                        lens_seed=rng.randrange(1 << 20), last=last)
            if batch * case["heads"] * high * min(last or high, high) > 1 << 31:  # the plain form's padded scores
                continue
        else:
            high = _log_int(rng, 16, 16384)
            budget = max(1, int(high * rng.uniform(0.2, 0.9)))
            case.update(batch=_log_int(rng, 1, 32), high=high, low=rng.choice([high, 1 + high // 8, 0]),
                        lens_seed=rng.randrange(1 << 20), page=rng.choice([16, 16, 8, 12, 64]), budget=budget,
                        recent=int(budget * rng.choice([0, 0.1, 0.25, 0.5, 1])), format=rng.choice(["mxfp4", "full"]))
            del case["heads"]
        cost = work(case)
        if cost["flops" if kind == "prompt" else "bytes"] <= _MOST[kind]:
            return case


def _lens(case):
    """Sequence lengths: uniform in [low, high], the last one the longest."""
    r = random.Random(case["lens_seed"])
    return [r.randint(case["low"], case["high"]) for _ in range(case["batch"] - 1)] + [case["high"]]


def work(case):
    """Bytes: each input element read once, each output element written once.  FLOP: 2 D for each score and each
    weighted value; a prompt's scores once."""
    kind, hkv, dim = case["kind"], case["kv_heads"], case["dim"]
    row4 = dim / 2 + dim / 32  # bytes of a row in 4 bits, with its scales
    if kind == "write4":  # rows read, cache rows written, values written
        return {"bytes": 2.0 * case["tokens"] * hkv * (2 * dim + row4 + 2 * dim), "flops": 0.0}
    lens = _lens(case)
    total = sum(lens)
    if kind == "decode":
        row = row4 if case["format"] == "mxfp4" else 2 * dim
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": total * hkv * (2.0 * row + (8 if case["tracked"] else 0)) + 4.0 * len(lens) * case["heads"] *
                dim + 4.0 * (pages + len(lens)), "flops": 4.0 * total * case["heads"] * dim}
    if kind == "prompt":
        pairs = sum(m * n - m * (m - 1) / 2 for n in lens for m in (min(case["last"] or n, n),))
        rows = sum(min(case["last"] or n, n) for n in lens)
        return {"bytes": 2.0 * dim * (total * hkv + rows * case["heads"]) + 4.0 * len(lens) * case["high"] * hkv,
                "flops": 2.0 * pairs * case["heads"] * dim}
    row = row4 if case["format"] == "mxfp4" else 2 * dim
    cut = sum(case["budget"] for n in lens if n > case["budget"])  # rows that move: their sequence is cut
    return {"bytes": hkv * (4.0 * total + 4.0 * len(lens) * (case["high"] + case["budget"]) + 4.0 * row * cut),
            "flops": 0.0}


# --- inputs ---------------------------------------------------------------------------------------------------------


def _rows(g, *shape, dtype):
    """Keys or values: normal, with channels of different spread, as projections have them."""
    spread = torch.exp(0.4 * torch.randn(shape[-1], generator=g, device="cuda"))
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16) * spread.half()).to(dtype)


def _pages(g, case, lens):
    """Block tables of a pool a tenth larger than needed."""
    page = case["page"]
    blocks = [-(-n // page) for n in lens]
    pool = -(-sum(blocks) * 11 // 10) + 1
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    counts = torch.tensor(blocks, device="cuda")
    at = torch.arange(max(blocks + [1]), device="cuda")[None, :]
    tables = order[((counts.cumsum(0) - counts)[:, None] + at).clamp_(max=pool - 1)]
    return pool, torch.where(at < counts[:, None], tables, 0).to(torch.int32)


def _weights(g, lens, longest, hkv, mean):
    """Weights summed so far: a few heavy tokens, many light ones; 0 past the context.  Kept to 8 bits of mantissa,
    so that some are equal."""
    w = mean * torch.exp(1.5 * torch.randn(len(lens), hkv, max(longest, 1), generator=g, device="cuda") - 1.125)
    n = torch.tensor(lens, device="cuda")[:, None, None]
    return torch.where(torch.arange(w.shape[2], device="cuda") < n, w.bfloat16().float(), 0.0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, hkv, dim, dtype = case["kind"], case["kv_heads"], case["dim"], getattr(torch, case["dtype"])
    s = {"case": dict(case)}
    if kind == "write4":
        tokens, page = case["tokens"], case["page"]
        qkv = _rows(g, tokens, (case["heads"] + 2 * hkv) * dim, dtype=dtype)
        key, value = qkv[:, case["heads"] * dim:].view(tokens, 2, hkv, dim).unbind(1)
        index = torch.arange(tokens, device="cuda")
        pool = -(-(tokens if case["append"] else -(-tokens // page)) * 11 // 10)
        order = torch.randperm(pool, generator=g, device="cuda")
        rows = torch.randint(page, (tokens,), generator=g, device="cuda") if case["append"] else index % page
        s.update(key=key, value=value,
                 slots=order[index if case["append"] else index // page] * page + rows)
        for x in "kv":
            s[x] = torch.zeros(pool, hkv, page, dim // 2, dtype=torch.uint8, device="cuda")
            s[x + "_scales"] = torch.zeros(pool, hkv, page, dim // 32, dtype=torch.uint8, device="cuda")
        return s
    lens = _lens(case)
    longest = max(lens)
    s.update(lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), longest=longest)
    if kind == "prompt":
        total = sum(lens)
        qk = _rows(g, total, (case["heads"] + 2 * hkv) * dim, dtype=dtype)  # q, k and v of a fused projection
        s.update(q=qk[:, :case["heads"] * dim].view(total, case["heads"], dim),
                 k=qk[:, case["heads"] * dim:(case["heads"] + hkv) * dim].view(total, hkv, dim),
                 cu=torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda(),
                 weights=torch.zeros(len(lens), hkv, max(longest, 1), device="cuda"))
        return s
    pool, s["tables"] = _pages(g, case, lens)
    for x in "kv":
        rows = _rows(g, pool, hkv, case["page"], dim, dtype=dtype)
        if case["format"] == "mxfp4":
            s[x], s[x + "_scales"] = _to_mxfp4(rows)
        else:
            s[x] = rows
    if kind == "decode":
        s["q"] = torch.randn(len(lens), case["heads"], dim, generator=g, device="cuda").to(dtype)
        if case["tracked"]:  # what some fifty steps have left
            s["weights"] = _weights(g, lens, longest, hkv, 50.0 * case["heads"] / hkv / max(longest, 1))
    else:
        s["weights"] = _weights(g, lens, longest, hkv, 1.0)
    return s


# --- one pass -------------------------------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    kind = case["kind"]
    scales = {} if case.get("format") == "full" else {"k_scales": s.get("k_scales"), "v_scales": s.get("v_scales")}
    if own:
        ak = _ak()
        if kind == "write4":
            ak.reshape_and_cache_mxfp4(s["key"], s["value"], s["k"], s["k_scales"], s["v"], s["v_scales"], s["slots"])
            return ak.gather_cache_mxfp4(s["k"], s["k_scales"], s["v"], s["v_scales"], s["slots"], s["key"].dtype)
        if kind == "decode" and case["format"] == "mxfp4":
            out = ak.paged_decode_mxfp4(s["q"], s["k"], s["k_scales"], s["v"], s["v_scales"], s["tables"], s["lens"],
                                        s["longest"], weights=s.get("weights"))
            return (out, s["weights"]) if case["tracked"] else out
        if kind == "decode":
            return ak.paged_decode_weights(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["longest"],
                                           s["weights"]), s["weights"]
        if kind == "prompt":
            ak.prompt_weights(s["q"], s["k"], s["cu"], s["longest"], s["weights"], last=case["last"] or None)
            return s["weights"]
        lens, weights, kept = ak.evict_cache(s["k"], s["v"], s["tables"], s["lens"], s["weights"], case["budget"],
                                             case["recent"], **scales)
        return lens, weights, kept, [s[x] for x in ("k", "v", *scales)]
    if kind == "write4":
        return _plain_write(s)
    if kind == "decode":
        return _plain_decode(s)
    if kind == "prompt":
        return _plain_prompt(s)
    lens, weights, kept = _plain_evict(s)
    # Bytes that are moved, not computed: the 4-bit rows compare as they are.
    return lens, weights, kept, [s[x] for x in ("k", "v", *scales)]


def _to_mxfp4(x):
    """Codes (two to a byte, the even channel low) and scale exponents (biased by 127) of finite rows [..., D]."""
    x = x.float().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    scale = (((top.view(torch.int32) + (1 << 21)) >> 23) - 2).clamp_(1, 254)
    y = x * torch.ldexp(torch.ones_like(top), 127 - scale).unsqueeze(-1)
    a = y.abs()
    code = (a > 0.25).to(torch.uint8)
    code += a >= 0.75
    code += a > 1.25
    code += a >= 1.75
    code += a > 2.5
    code += a >= 3.5
    code += a > 5.0
    code += 8 * torch.signbit(x).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, scale.to(torch.uint8)


def _from_mxfp4(codes, scales):
    """The values that codes [..., D/2] and scales [..., D/32] stand for, in 32 bits."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=codes.device)
    x = table[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()]
    scale = torch.ldexp(torch.ones(scales.shape, device=codes.device), scales.int() - 127)
    return (x.unflatten(-1, (-1, 32)) * scale.unsqueeze(-1)).flatten(-2)


def _plain_write(s):
    page = s["case"]["page"]
    at, row = s["slots"] // page, s["slots"] % page

    def one(x, new):
        s[x][at, :, row], s[x + "_scales"][at, :, row] = _to_mxfp4(new)
        return _from_mxfp4(s[x][at, :, row], s[x + "_scales"][at, :, row]).to(new.dtype)

    return one("k", s["key"]), one("v", s["value"])


def _sequences(s, x):
    """[B, Hkv, longest, ...] rows of the cache s[x] along the block tables, padded by rows of page 0."""
    cache = s[x][s["tables"].long()].transpose(1, 2).flatten(2, 3)  # [B, Hkv, pages * page, ...]
    return cache[:, :, :s["longest"]]


def _plain_decode(s):
    case, q = s["case"], s["q"]
    if case["format"] == "mxfp4":
        k, v = (_from_mxfp4(_sequences(s, x), _sequences(s, x + "_scales")) for x in "kv")
    else:
        k, v = _sequences(s, "k").float(), _sequences(s, "v").float()
    inside = (torch.arange(s["longest"], device="cuda") < s["lens"][:, None])[:, None, None]
    grouped = q.float().unflatten(1, (case["kv_heads"], -1))  # [B, Hkv, G, D]
    score = grouped @ k.transpose(2, 3).contiguous() * case["dim"] ** -0.5
    score = torch.where(inside, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.where(inside, torch.exp(score - top), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp_(min=1e-30)  # an empty context: zeros
    out = (p @ torch.where(inside.transpose(2, 3), v, 0.0)).flatten(1, 2).to(q.dtype)
    if not case["tracked"]:
        return out
    s["weights"][:, :, :s["longest"]] += p.sum(2)
    return out, s["weights"]


def _plain_prompt(s):
    case, n = s["case"], s["lens"][:, None].long()
    last, longest, hkv, total = min(case["last"] or s["longest"], s["longest"]), s["longest"], case["kv_heads"], \
        s["q"].shape[0]
    start = s["cu"][:-1, None].long()
    j = torch.arange(longest, device="cuda")
    i = n - last + torch.arange(last, device="cuda")  # positions of the queries that count; negative: none
    k = s["k"].float()[(start + j).clamp_(max=total - 1)]  # [B, N, Hkv, D]
    q = s["q"].float()[(start + i).clamp_(0, total - 1)].unflatten(2, (hkv, -1))  # [B, last, Hkv, G, D]
    score = q.permute(0, 2, 3, 1, 4) @ k.permute(0, 2, 3, 1).unsqueeze(2).contiguous()
    score *= case["dim"] ** -0.5
    seen = ((j <= i[:, :, None]) & (j < n[:, :, None]))[:, None, None]
    score.masked_fill_(~seen, -math.inf)
    score -= score.amax(-1, keepdim=True)
    p = score.exp_().masked_fill_(~seen, 0.0)
    p /= p.sum(-1, keepdim=True).clamp_(min=1e-30)
    s["weights"][:, :, :longest] = p.sum(3).sum(2)
    s["weights"][:, :, longest:] = 0.0
    return s["weights"]


def _plain_evict(s):
    case, w, n = s["case"], s["weights"], s["lens"][:, None, None].long()
    length, budget, page = w.shape[2], case["budget"], case["page"]
    position = torch.arange(length, device="cuda").expand(w.shape)
    # First the last tokens (and all of a short sequence), then the others by weight, then what is past the end.
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    rank = torch.where(position >= n, 2, torch.where((position >= n - case["recent"]) | (n <= budget), 0, 1))
    order = order.gather(2, torch.sort(rank.gather(2, order), dim=-1, stable=True).indices)
    at = torch.arange(budget, device="cuda")
    taken = torch.full((*w.shape[:2], budget), length, device="cuda")
    taken[:, :, :min(budget, length)] = order[:, :, :budget]
    new = n.clamp(max=budget)
    kept = torch.where(at < new, taken, length).sort(dim=-1).values
    kept = torch.where(at < new, kept, -1)
    weights = torch.zeros_like(w)
    m = min(budget, length)
    weights[:, :, :m] = torch.where(at[:m] < new, w.gather(2, kept[:, :, :m].clamp(min=0)), 0.0)
    # Rows move within the sequence's own pages: row at[i] becomes what row kept[i] was.
    b, h, i = torch.nonzero((kept >= 0) & (kept != at), as_tuple=True)
    source = kept[b, h, i]
    table = s["tables"].long()

    def move(x):
        x[table[b, i // page], h, i % page] = x[table[b, source // page], h, source % page]

    move(s["k"])
    move(s["v"])
    if case["format"] == "mxfp4":
        move(s["k_scales"])
        move(s["v_scales"])
    return new[:, 0, 0].to(torch.int32), weights, kept.to(torch.int32)


# --- from the definition, in 64 bits ---------------------------------------------------------------------------------


def _nearest4(rows):
    """Rows [T, H, D] rounded to the format's nearest values, in 64 bits."""
    x = rows.double().reshape(*rows.shape[:-1], -1, 32)
    top = x.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [1/2, 1)
    exponent = exponent - 1 + (mantissa >= 0.875).to(exponent.dtype) - 2
    step = torch.ldexp(torch.ones_like(top), exponent)
    grid = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64, device=x.device)  # even first
    best = torch.zeros_like(x)
    far = torch.full_like(x, math.inf)
    for value in grid.tolist():
        off = (x.abs() / step - value).abs()
        best = torch.where(off < far, value, best)
        far = torch.minimum(far, off)
    best = torch.where(top > 0, best * step, 0.0)
    return torch.copysign(best, x).reshape(rows.shape)


def _values64(s, x, pages, h):
    """Rows [pages * page, D] of one head along its pages."""
    if s["case"]["format"] == "full":
        return s[x][pages, h].reshape(-1, s["case"]["dim"]).double()
    c = s[x][pages, h].reshape(-1, s["case"]["dim"] // 2).long()
    half = 2.0 ** (s[x + "_scales"][pages, h].reshape(c.shape[0], -1).double() - 127)
    code = torch.empty(c.shape[0], 2 * c.shape[1], dtype=torch.long, device=c.device)
    code[:, 0::2], code[:, 1::2] = c % 16, c // 16
    size = code % 8
    value = torch.where(size < 2, 0.5 * size, (1 + 0.5 * (size % 2)) * 2.0 ** (size // 2 - 1).double())
    value = torch.where(code >= 8, -value, value)
    return value * half.repeat_interleave(32, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    kind, hkv = case["kind"], case["kv_heads"]
    if kind == "write4":
        return _nearest4(s["key"]), _nearest4(s["value"])
    lens = _lens(case)
    if kind == "evict":
        return _exact_evict(s, lens)
    group = case["heads"] // hkv
    scale = case["dim"] ** -0.5
    if kind == "prompt":
        weights = torch.zeros(s["weights"].shape, dtype=torch.float64, device="cuda")
        start = 0
        for b, n in enumerate(lens):
            first = n - min(case["last"] or n, n)
            for h in range(case["heads"] if n else 0):
                k = s["k"][start:start + n, h // group].double()
                for r in range(first, n, 2048):
                    m = min(n, r + 2048)
                    score = s["q"][start + r:start + m, h].double() @ k[:m].t().contiguous() * scale
                    future = torch.arange(m, device="cuda") > torch.arange(r, m, device="cuda")[:, None]
                    weights[b, h // group, :m] += torch.softmax(score.masked_fill(future, -math.inf), 1).sum(0)
            start += n
        return weights
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if case["tracked"] else None
    for b, n in enumerate(lens):
        pages = s["tables"][b, :-(-n // case["page"])].long()
        for h in range(hkv if n else 0):
            heads = slice(h * group, (h + 1) * group)
            k, v = (_values64(s, x, pages, h)[:n] for x in "kv")
            p = torch.softmax(s["q"][b, heads].double() @ k.t().contiguous() * scale, dim=1)
            out[b, heads] = p @ v
            if case["tracked"]:
                weights[b, h, :n] += p.sum(0)
    return (out, weights) if case["tracked"] else out


def _exact_evict(s, lens):
    case = s["case"]
    budget, recent, page = case["budget"], case["recent"], case["page"]
    names = ("k", "v", "k_scales", "v_scales") if case["format"] == "mxfp4" else ("k", "v")
    before = {x: s[x].clone() for x in names}
    weights = torch.zeros_like(s["weights"], dtype=torch.float64)
    kept = torch.full((len(lens), case["kv_heads"], budget), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        for h in range(case["kv_heads"]):
            if n <= budget:
                keep = torch.arange(n, device="cuda")
            else:
                old = s["weights"][b, h, :n - recent].double()
                heavy = torch.argsort(-old, stable=True)[:budget - recent]
                keep = torch.cat((heavy.sort().values, torch.arange(n - recent, n, device="cuda")))
            kept[b, h, :len(keep)] = keep.int()
            weights[b, h, :len(keep)] = s["weights"][b, h, keep].double()
            to = torch.arange(len(keep), device="cuda")
            table = s["tables"][b].long()
            for x in names:
                s[x][table[to // page], h, to % page] = before[x][table[keep // page], h, keep % page]
    new = torch.tensor([min(n, budget) for n in lens], dtype=torch.int32, device="cuda")
    return new, weights, kept, [s[x].double() if s[x].is_floating_point() else s[x] for x in names]
