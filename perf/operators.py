"""Performance cases of the 8-bit serving operators: integer linears and the paged 8-bit KV cache.

Four kinds of work, each through the entry points that a server of such a model calls:

* ``linear``  ``w8a8_forward``: tokens quantized to int8 with a scale each, times int8 weights with a scale per output channel;
* ``tables``  ``plan_blocks``: block tables and slot maps of a step from the requests' lengths;
* ``update``  ``plan_blocks``, ``append_blocks`` and ``dense_blocks``: prompts (or pieces of prompts) into the cache, and the dense
  keys / values of every request back, as the attention of a long prompt takes them;
* ``attend``  ``plan_blocks``, then ``append_blocks`` and ``attend_blocks`` for each layer: one decode step's attention.

``own`` chooses between the package's kernels and the plain form of the same operators in elementary torch operations.  ``listed()``
are the cases to watch, ``draw(rng)`` gives more from the same ranges, ``exact`` is the definition in 64 bits.  Inputs are
synthetic: N(0, 1) activations, values and queries, keys with a few channels ten times as large.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_DEVICE = "cuda"


def listed() -> list[dict]:
    return [
        # one projection, one token: latency of a decode step's linear
        {"name": "linear_one_token", "kind": "linear", "rows": 1, "n": 4096, "k": 4096, "dtype": "fp16", "zero": False,
         "input_scale": False, "bias": False},
        # batched decode through the fused gate|up projection: weight streaming
        {"name": "linear_gate_up_16", "kind": "linear", "rows": 16, "n": 28672, "k": 4096, "dtype": "bf16", "zero": False,
         "input_scale": False, "bias": False},
        # a ragged chunk of a model with odd sizes: smoothed activations, asymmetric weights, bias
        {"name": "linear_odd_333", "kind": "linear", "rows": 333, "n": 3584, "k": 18944, "dtype": "fp16", "zero": True,
         "input_scale": True, "bias": True},
        # a long prompt through the largest projection: integer tensor-core rate
        {"name": "linear_prompt_2048", "kind": "linear", "rows": 2048, "n": 28672, "k": 4096, "dtype": "bf16", "zero": False,
         "input_scale": False, "bias": False},
        # the tables of a decode step of 64 running requests
        {"name": "tables_decode_64", "kind": "tables", "requests": 64, "ctx": 4096, "new": 1, "block": 32, "pad": 0},
        # the tables of 256 prompts arriving together, in small blocks, with a padded batch
        {"name": "tables_prompts_256", "kind": "tables", "requests": 256, "ctx": 300, "new": 251, "block": 16, "pad": 100},
        # a chunk of a few ragged prompts on top of what their requests hold already
        {"name": "update_chunks_8", "kind": "update", "requests": 8, "ctx": 300, "new": 257, "block": 32, "hkv": 8, "d": 128,
         "dtype": "bf16"},
        # long prompts into an empty cache
        {"name": "update_prompts_32k", "kind": "update", "requests": 4, "ctx": 0, "new": 8192, "block": 16, "hkv": 4, "d": 128,
         "dtype": "fp16"},
        # one sequence, eight layers: latency of the decode attention
        {"name": "attend_one_sequence_4k", "kind": "attend", "requests": 1, "ctx": 4096, "new": 1, "block": 32, "hq": 32, "hkv": 8,
         "d": 128, "layers": 8, "dtype": "bf16"},
        # a running batch of ragged requests
        {"name": "attend_ragged_64", "kind": "attend", "requests": 64, "ctx": 2000, "new": 1, "block": 16, "hq": 32, "hkv": 8,
         "d": 128, "layers": 2, "dtype": "bf16"},
        # a full batch of long contexts: cache streaming
        {"name": "attend_batch16_32k", "kind": "attend", "requests": 16, "ctx": 32768, "new": 1, "block": 64, "hq": 28, "hkv": 4,
         "d": 128, "layers": 1, "dtype": "fp16"},
        # three drafted tokens per request verified at once, small heads
        {"name": "attend_drafts_12", "kind": "attend", "requests": 12, "ctx": 1500, "new": 3, "block": 32, "hq": 32, "hkv": 8,
         "d": 64, "layers": 2, "dtype": "fp16"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer between lo and hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["linear", "linear", "tables", "update", "attend", "attend"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "linear":
        k = 16 * _log(rng, 16, 1184)
        n = _log(rng, 256, 28672)
        rows = _log(rng, 1, max(1, min(4096, 2048 * 28672 * 4096 // (n * k))))
        return {"kind": kind, "rows": rows, "n": n, "k": k, "dtype": dtype, "zero": rng.random() < 0.4,
                "input_scale": rng.random() < 0.3, "bias": rng.random() < 0.4}
    if kind == "tables":
        requests = _log(rng, 1, 256)
        new = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, 64000 // requests))
        return {"kind": kind, "requests": requests, "ctx": _log(rng, 16, 8192), "new": new, "block": rng.choice([16, 32, 64]),
                "pad": rng.choice([0, 0, 7])}
    d, block = rng.choice([64, 128, 128]), rng.choice([16, 32, 64])
    if kind == "update":
        requests, hkv = _log(rng, 1, 16), rng.choice([2, 4, 8])
        return {"kind": kind, "requests": requests, "ctx": rng.choice([0, _log(rng, 16, 1000)]),
                "new": _log(rng, 16, 131072 // (4 * hkv * requests) * 4), "block": block, "hkv": hkv, "d": d, "dtype": dtype}
    requests, hkv = _log(rng, 1, 96), rng.choice([2, 4, 8])
    new = rng.choice([1, 1, 1, 2, 4]) if requests <= 32 else 1
    return {"kind": kind, "requests": requests, "ctx": _log(rng, 16, min(60000, 2097152 // (hkv * requests * new))), "new": new,
            "block": block, "hq": hkv * rng.choice([1, 4, 7, 8]), "hkv": hkv, "d": d, "layers": rng.choice([1, 2]), "dtype": dtype}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------

def _spread(mean: int, n: int) -> list[int]:
    """``n`` lengths from a tenth of ``mean`` to almost twice it: the same ones, in whatever order, for every seed."""
    if n == 1 or mean < 2:
        return [mean] * n
    return [max(1, round(mean * (0.1 + 1.8 * i / (n - 1)))) for i in range(n)]


def _requests(case: dict, seed: int) -> dict:
    """Lengths, blocks and the stack of free blocks of a running server, as tensors on the GPU."""
    g = torch.Generator().manual_seed(seed)
    n, bs = case["requests"], case["block"]
    order = torch.randperm(n, generator=g)
    old = torch.tensor(_spread(case["ctx"], n) if case["ctx"] else [0] * n)[order]
    new = torch.tensor(_spread(case["new"], n) if case["kind"] != "attend" else [case["new"]] * n).roll(n // 3)[order]
    have, need = (old + bs - 1) // bs, (old + new + bs - 1) // bs
    width = int(need.max()) + 3
    blocks = int(need.sum()) + 17
    ids = torch.randperm(blocks, generator=g).to(torch.int32)
    table = torch.zeros(n, width, dtype=torch.int32)
    held = torch.arange(width)[None, :] < have[:, None]
    table[held] = ids[: int(have.sum())]
    free = torch.zeros(blocks, dtype=torch.int32)
    left = blocks - int(have.sum())
    free[:left] = ids[int(have.sum()):]
    on = lambda t: t.to(torch.int32).to(_DEVICE)  # noqa: E731
    return {"seq_lens": on(old), "new_lens": on(new), "block_table": on(table), "free_blocks": on(free),
            "free_count": on(torch.tensor([left])), "block": bs, "blocks": blocks, "tokens": int(new.sum()) + case.get("pad", 0),
            "context": int((old + new).sum())}


def _normal(shape, seed: int, dtype, outliers: bool = False) -> torch.Tensor:
    g = torch.Generator(device=_DEVICE).manual_seed(seed)
    x = torch.randn(shape, device=_DEVICE, generator=g, dtype=torch.float32 if math.prod(shape) < 1 << 28 else dtype)
    if outliers:
        x[..., torch.randperm(shape[-1], device=_DEVICE, generator=g)[: max(1, shape[-1] // 100)]] *= 10.0
    return x.to(dtype)


def _cached(case: dict, req: dict, seed: int) -> dict:
    """One layer's pool with every block filled, and the open blocks' rows."""
    dtype, h, d, bs = _DTYPES[case["dtype"]], case["hkv"], case["d"], req["block"]
    if case["ctx"]:
        kc, ks = _quantized(_normal((req["blocks"], h, bs, d), seed, dtype, outliers=True))
        vc, vs = _quantized(_normal((req["blocks"], h, bs, d), seed + 1, dtype))
    else:
        kc, vc = (torch.zeros(req["blocks"], h, bs, d, dtype=torch.int8, device=_DEVICE) for _ in range(2))
        ks, vs = (torch.zeros(req["blocks"], h, dtype=torch.float32, device=_DEVICE) for _ in range(2))
    n = case["requests"]
    return {"k_codes": kc, "v_codes": vc, "k_scale": ks, "v_scale": vs,
            "tail_k": _normal((n, h, bs, d), seed + 2, dtype, outliers=True), "tail_v": _normal((n, h, bs, d), seed + 3, dtype),
            "k": _normal((req["tokens"], h, d), seed + 4, dtype, outliers=True), "v": _normal((req["tokens"], h, d), seed + 5, dtype),
            "q": _normal((req["tokens"], case["hq"], d), seed + 6, dtype) if "hq" in case else None}


def prepare(case: dict, seed: int) -> dict:
    if case["kind"] == "linear":
        m, n, k, dtype = case["rows"], case["n"], case["k"], _DTYPES[case["dtype"]]
        g = torch.Generator(device=_DEVICE).manual_seed(seed)
        rand = lambda *s: torch.rand(*s, device=_DEVICE, generator=g)  # noqa: E731
        x = _normal((m, k), seed + 1, dtype)
        if case["input_scale"]:
            x[:, :: 97] *= 20.0           # the channels that smoothing is for
        return {"kind": "linear", "x": x,
                "q_weight": torch.randint(-127, 128, (n, k), device=_DEVICE, generator=g, dtype=torch.int8),
                "scale": (0.5 + rand(n)) * 3e-4,
                "zero": torch.randint(-20, 21, (n,), device=_DEVICE, generator=g).float() if case["zero"] else None,
                "input_scale": 0.5 + 2.0 * rand(k) if case["input_scale"] else None,
                "bias": _normal((n,), seed + 2, dtype) if case["bias"] else None}
    req = _requests(case, seed)
    state = {"kind": case["kind"], "req": req}
    if case["kind"] != "tables":
        state["layers"] = [_cached(case, req, seed * 64 + 8 * i) for i in range(case.get("layers", 1))]
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------------------

def run(state: dict):
    kind = state["kind"]
    if kind == "linear":
        s = state
        if own:
            from pare_b200.kernels import w8a8_forward

            return w8a8_forward(s["x"], s["q_weight"], s["scale"], s["zero"], bias=s["bias"], input_scale=s["input_scale"])
        return _plain_linear(s["x"], s["q_weight"], s["scale"], s["zero"], s["bias"], s["input_scale"])
    req = state["req"]
    if own:
        from pare_b200 import paged_cache as pc

        step = pc.plan_blocks(req["seq_lens"], req["new_lens"], req["block_table"], req["free_blocks"], req["free_count"],
                              req["block"], req["tokens"])
        if kind == "tables":
            return {"query_start": step.query_start, "token_request": step.token_request, "positions": step.positions,
                    "slots": step.slots, "seq_lens": step.seq_lens, "block_table": step.block_table, "free_count": step.free_count}
        if "own_layers" not in state:   # names for the buffers that a program holds, no copies
            state["own_layers"] = [pc.PagedLayer(*(y[n] for n in ("k_codes", "v_codes", "k_scale", "v_scale", "tail_k", "tail_v")))
                                   for y in state["layers"]]
        if kind == "update":
            y, layer = state["layers"][0], state["own_layers"][0]
            pc.append_blocks(layer, step, y["k"], y["v"])
            k, v = pc.dense_blocks(layer, step, req["context"])
            return {"k": k, "v": v, "k_scale": layer.k_scale, "v_scale": layer.v_scale, "tail_k": layer.tail_k, "tail_v": layer.tail_v}
        out = []
        for y, layer in zip(state["layers"], state["own_layers"]):
            pc.append_blocks(layer, step, y["k"], y["v"])
            out.append(pc.attend_blocks(layer, step, y["q"]))
        return out
    step = _plain_plan(req)
    if kind == "tables":
        return step
    if kind == "update":
        y = state["layers"][0]
        _plain_append(y, step, req["block"])
        k, v = _plain_dense(y, step, req["block"], req["context"])
        return {"k": k, "v": v, "k_scale": y["k_scale"], "v_scale": y["v_scale"], "tail_k": y["tail_k"], "tail_v": y["tail_v"]}
    out = []
    for y in state["layers"]:
        _plain_append(y, step, req["block"])
        out.append(_plain_attend(y, step, req["block"]))
    return out


# ---- plain forms -----------------------------------------------------------------------------------------------------------------

def _over_127(x):
    return x / torch.full_like(x, 127.0)      # a quotient: dividing by a Python number multiplies by its rounded reciprocal


def _plain_linear(x, q_weight, scale, zero, bias, input_scale):
    if input_scale is not None:
        x = (x.float() / input_scale).to(x.dtype)
    step = _over_127(x.float().abs().amax(dim=1, keepdim=True).clamp(min=1e-6))
    codes = torch.round(x.float() / step)
    w = q_weight.float() if zero is None else q_weight.float() - zero[:, None]
    y = codes @ w.t() * step * scale
    return (y if bias is None else y + bias.float()).to(x.dtype)


def _plain_plan(req: dict) -> dict:
    old, new, bs = req["seq_lens"].long(), req["new_lens"].long(), req["block"]
    end, zero = old + new, old.new_zeros(1)
    start = torch.cat([zero, new.cumsum(0)])
    t = torch.arange(req["tokens"], device=old.device)
    real = t < start[-1]
    r = torch.searchsorted(start[1:].contiguous(), t, right=True).clamp(max=old.numel() - 1)
    pos = old[r] + t - start[r]
    have, need = (old + bs - 1) // bs, (end + bs - 1) // bs
    first = (need - have).cumsum(0) - (need - have)       # blocks taken by the requests before this one
    col = torch.arange(req["block_table"].shape[1], device=old.device)[None, :]
    taken = (first - have)[:, None] + col
    fresh = (col >= have[:, None]) & (col < need[:, None])
    ids = req["free_blocks"][(req["free_count"].long() - 1 - taken).clamp(0, req["blocks"] - 1)]
    table = torch.where(fresh, ids, req["block_table"])
    slots = table[r, (pos // bs).clamp(max=table.shape[1] - 1)].long() * bs + pos % bs
    return {"query_start": start.int(), "token_request": torch.where(real, r, -1).int(), "positions": torch.where(real, pos, -1).int(),
            "slots": torch.where(real, slots, -1), "seq_lens": end.int(), "block_table": table,
            "free_count": (req["free_count"] - (need - have).sum()).int()}


def _quantized(x):
    """``[blocks, heads, tokens, channels]`` -> int8 codes, fp32 scales ``[blocks, heads]`` (in pieces of about a gigabyte)."""
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:2], dtype=torch.float32, device=x.device)
    piece = max(1, (1 << 28) // max(1, math.prod(x.shape[1:])))
    for a in range(0, x.shape[0], piece):
        f = x[a:a + piece].float()
        s = _over_127(f.abs().amax(dim=(2, 3)))
        codes[a:a + piece] = torch.where(s[..., None, None] > 0, torch.round(f / s[..., None, None]), 0.0).to(torch.int8)
        scale[a:a + piece] = s
    return codes, scale


def _plain_append(y: dict, step: dict, bs: int) -> None:
    """New tokens into the rows of their request's open block; blocks that are full now into the pool."""
    end, start, r, pos = step["seq_lens"].long(), step["query_start"].long(), step["token_request"].long(), step["positions"].long()
    old = end - (start[1:] - start[:-1])
    b0, b1 = old // bs, end // bs                                     # blocks that fill up: [b0, b1)
    n = -(-r.numel() // bs) + 2 * old.numel()                         # at most so many fill up or are open
    many = (b1 - b0 + 1).cumsum(0)
    i = torch.arange(n, device=r.device)
    ri = torch.searchsorted(many, i, right=True)
    live = ri < old.numel()
    ri = ri.clamp(max=old.numel() - 1)
    bi = b0[ri] + i - (many - (b1 - b0 + 1))[ri]                      # block i of the list: block bi of request ri
    full = live & (bi < b1[ri])
    p = bi[:, None] * bs + torch.arange(bs, device=r.device)          # its tokens' positions
    fresh = (p >= old[ri][:, None]) & (p < end[ri][:, None]) & live[:, None]
    row = (start[ri][:, None] + p - old[ri][:, None]).clamp(0, max(0, r.numel() - 1))
    held = fresh[..., None, None]
    at = step["block_table"][ri, bi.clamp(max=step["block_table"].shape[1] - 1)].long()[full]
    for new, tail, codes, scale in ((y["k"], y["tail_k"], y["k_codes"], y["k_scale"]), (y["v"], y["tail_v"], y["v_codes"], y["v_scale"])):
        x = torch.where(held, new[row], tail[ri].transpose(1, 2)).transpose(1, 2)    # [n, heads, bs, channels]
        codes[at], scale[at] = _quantized(x[full])
        some = live & (bi == b1[ri])                                  # the open block: only its new rows change
        tail[ri[some]] = torch.where(fresh[some][:, None, :, None], x[some], tail[ri[some]])


def _values(y: dict, step: dict, bs: int, r, pos):
    """fp32 keys and values at positions ``pos`` of requests ``r`` (any shape): ``[..., heads, channels]``."""
    end = step["seq_lens"].long()[r]
    inside = pos < end // bs * bs
    at = step["block_table"][r, (pos // bs).clamp(max=step["block_table"].shape[1] - 1)].long()
    off = pos % bs
    return tuple(torch.where(inside[..., None, None], y[c][at, :, off].float() * y[s][at][..., None], y[t][r, :, off].float())
                 for c, s, t in (("k_codes", "k_scale", "tail_k"), ("v_codes", "v_scale", "tail_v")))


def _plain_dense(y: dict, step: dict, bs: int, total: int):
    end = step["seq_lens"].long()
    first = end.cumsum(0) - end
    t = torch.arange(total, device=end.device)
    r = torch.searchsorted(end.cumsum(0), t, right=True)
    return tuple(x.to(y["k"].dtype) for x in _values(y, step, bs, r, t - first[r]))


def _plain_attend(y: dict, step: dict, bs: int):
    q, h = y["q"], y["k"].shape[1]
    T, hq, d = q.shape
    r, pos = step["token_request"].long(), step["positions"].long()
    width = step["block_table"].shape[1] * bs
    out = torch.empty_like(q)
    piece = max(1, (1 << 29) // (width * h * d))
    for a in range(0, T, piece):                                      # tokens at a time, for memory only
        rr, pp = r[a:a + piece], pos[a:a + piece]
        j = torch.arange(width, device=q.device).expand(rr.numel(), width)
        k, v = _values(y, step, bs, rr[:, None].expand_as(j), j)      # [t, width, heads, channels]
        qf = q[a:a + piece].float().view(rr.numel(), h, hq // h, d)
        s = qf @ k.permute(0, 2, 3, 1) / math.sqrt(d)
        seen = (j <= pp[:, None])[:, None, None, :]
        s = torch.where(seen, s, float("-inf"))
        e = torch.exp(s - s.amax(dim=-1, keepdim=True))
        v = torch.where((j <= pp[:, None])[..., None, None], v, 0.0)
        o = e @ v.permute(0, 2, 1, 3) / e.sum(dim=-1, keepdim=True)
        out[a:a + piece] = o.reshape(rr.numel(), hq, d).to(q.dtype)
    return out


# ---- work ------------------------------------------------------------------------------------------------------------------------

def work(case: dict) -> dict:
    """Bytes and operations that one pass cannot do without."""
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        extra = 4 * n * case["zero"] + 4 * k * case["input_scale"] + 2 * n * case["bias"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n + extra, "flops": 2 * m * n * k}
    n, bs = case["requests"], case["block"]
    old = _spread(case["ctx"], n) if case["ctx"] else [0] * n
    new = _spread(case["new"], n) if case["kind"] != "attend" else [case["new"]] * n
    t, ctx = sum(new), sum(old) + sum(new)
    tables = 4 * 4 * n + 16 * (t + case.get("pad", 0)) + 8 * (t // bs + n)
    if case["kind"] == "tables":
        return {"bytes": tables, "flops": 0}
    h, d = case["hkv"], case["d"]
    if case["kind"] == "update":
        return {"bytes": tables + 2 * t * h * d * 3 + 2 * ctx * h * d * 3, "flops": 2 * (t + ctx) * h * d}
    lay, hq = case["layers"], case["hq"]
    seen = sum((o + i + 1) for o, w in zip(old, new) for i in range(w))
    return {"bytes": tables + lay * (2 * ctx * h * d + 2 * t * h * d * 2 + 2 * t * hq * d * 2), "flops": lay * 4 * seen * hq * d}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------

def _codes64(x, step):
    return torch.where(step > 0, torch.round(x / step), torch.zeros_like(x))


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["kind"] == "linear":
        x, w = state["x"], state["q_weight"].double()
        if state["input_scale"] is not None:
            x = (x.double() / state["input_scale"].double()).to(x.dtype)     # the operator's own rounding of its input
        x = x.double()
        if state["zero"] is not None:
            w = w - state["zero"].double().unsqueeze(1)
        step = torch.clamp(x.abs().max(dim=1).values, min=1e-6) / 127
        y = torch.einsum("mk,nk->mn", _codes64(x, step.unsqueeze(1)), w) * torch.outer(step, state["scale"].double())
        return y if state["bias"] is None else y + state["bias"].double()
    req, bs = state["req"], case["block"]
    old, new, count = req["seq_lens"].tolist(), req["new_lens"].tolist(), int(req["free_count"])
    table, free = req["block_table"].tolist(), req["free_blocks"].tolist()
    rows, begin, tokens = [0], {}, []
    for i, (a, b) in enumerate(zip(old, new)):
        begin[i] = rows[-1]
        rows.append(rows[-1] + b)
        for blk in range(-(-a // bs), -(-(a + b) // bs)):
            count -= 1
            table[i][blk] = free[count]
        tokens += [(i, p, table[i][p // bs] * bs + p % bs) for p in range(a, a + b)]
    if case["kind"] == "tables":
        tokens += [(-1, -1, -1)] * (req["tokens"] - len(tokens))
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=_DEVICE)  # noqa: E731
        return {"query_start": i32(rows), "token_request": i32([x[0] for x in tokens]), "positions": i32([x[1] for x in tokens]),
                "slots": torch.tensor([x[2] for x in tokens], dtype=torch.int64, device=_DEVICE),
                "seq_lens": i32([a + b for a, b in zip(old, new)]), "block_table": i32(table), "free_count": i32([count])}

    def sequence(y, i, name):
        """Request i's tokens in 64 bits after the append, the scales of the blocks that filled up, and its open rows."""
        a, end = old[i], old[i] + new[i]
        x = y[name][begin[i]:begin[i] + new[i]].double().transpose(0, 1)                 # [heads, new, channels]
        keep, scales = a // bs * bs, {}
        ids = torch.tensor(table[i][: a // bs], dtype=torch.int64, device=_DEVICE)
        past = y[name + "_codes"][ids].double() * y[name + "_scale"][ids].double()[..., None, None]
        past = past.transpose(0, 1).reshape(case["hkv"], keep, case["d"])
        rest = torch.cat([y["tail_" + name][i, :, : a - keep].double(), x], dim=1)
        whole = (end // bs * bs - keep) // bs
        if whole:
            blocks = rest[:, : whole * bs].reshape(case["hkv"], whole, bs, case["d"])
            step = blocks.abs().amax(dim=(2, 3), keepdim=True) / 127
            scales = {table[i][keep // bs + w]: step[:, w, 0, 0] for w in range(whole)}
            rest = torch.cat([(_codes64(blocks, step) * step).reshape(case["hkv"], -1, case["d"]), rest[:, whole * bs:]], dim=1)
        return torch.cat([past, rest], dim=1), scales, end % bs, rest[:, rest.shape[1] - end % bs:] if end % bs else None

    if case["kind"] == "update":
        y, out = state["layers"][0], {}
        for name in ("k", "v"):
            got = [sequence(y, i, name) for i in range(len(old))]
            scale, tail = y[name + "_scale"].double(), y["tail_" + name].double()
            for i, (_, scales, n_open, open_rows) in enumerate(got):
                for at, s in scales.items():
                    scale[at] = s
                fresh = min(n_open, new[i])
                if fresh:
                    tail[i, :, n_open - fresh: n_open] = open_rows[:, n_open - fresh:]
            out.update({name: torch.cat([x[0] for x in got], dim=1).transpose(0, 1).contiguous(), name + "_scale": scale,
                        "tail_" + name: tail})
        return out
    result = []
    for y in state["layers"]:
        out = torch.zeros(y["q"].shape, dtype=torch.float64, device=_DEVICE)
        for i, n in enumerate(new):
            k, v = sequence(y, i, "k")[0], sequence(y, i, "v")[0]
            for w in range(n):
                seen, row = old[i] + w + 1, begin[i] + w
                q = y["q"][row].double().view(case["hkv"], -1, case["d"])
                p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, k[:, :seen]) / case["d"] ** 0.5, dim=-1)
                out[row] = torch.einsum("hgn,hnd->hgd", p, v[:, :seen]).reshape(-1, case["d"])
        result.append(out)
    return result
