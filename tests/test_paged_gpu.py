"""Paged 8-bit KV cache on the GPU: tables, append, dense reconstruction and attention against plain implementations in 64 bits.

Tables, codes and scales have to be equal.  Attention is held to a bound that is derived per output element (``_bound``)."""

import copy
import math
import random

import pytest
import torch

from pare_b200 import PagedKVCache, PagedKVConfig
from pare_b200 import paged_cache as pc

pytestmark = pytest.mark.gpu

DEV = "cuda"


# ---- plain implementations -------------------------------------------------------------------------------------------------------

def _ref_plan(old, new, table, free, count, bs, rows):
    """Python lists in, python lists out; ``None`` if the step does not fit."""
    table = [list(r) for r in table]
    need = sum(-(-(a + n) // bs) - -(-a // bs) for a, n in zip(old, new))
    if sum(new) > rows or need > count or any(a + n > len(table[0]) * bs for a, n in zip(old, new)):
        return None
    start, req, pos, slot, ctx = [0], [], [], [], [0]
    for r, (a, n) in enumerate(zip(old, new)):
        for b in range(-(-a // bs), -(-(a + n) // bs)):
            count -= 1
            table[r][b] = free[count]
        for p in range(a, a + n):
            req.append(r), pos.append(p), slot.append(table[r][p // bs] * bs + p % bs)
        start.append(start[-1] + n)
        ctx.append(ctx[-1] + (a + n if n else 0))
    pad = [-1] * (rows - len(req))
    return dict(query_start=start, token_request=req + pad, positions=pos + pad, slots=slot + pad,
                seq_lens=[a + n for a, n in zip(old, new)], free_count=[count], context_start=ctx, block_table=table)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class _Model:
    """A cache that remembers every token: what the pool has to hold and what attention has to give, in 64 bits."""

    def __init__(self, requests, h, d, bs, dtype):
        self.h, self.d, self.bs, self.dtype = h, d, bs, dtype
        self.k = [torch.empty(h, 0, d, dtype=dtype, device=DEV) for _ in range(requests)]
        self.v = [torch.empty(h, 0, d, dtype=dtype, device=DEV) for _ in range(requests)]

    def add(self, r, k, v):
        self.k[r] = torch.cat([self.k[r], k.transpose(0, 1)], 1)
        self.v[r] = torch.cat([self.v[r], v.transpose(0, 1)], 1)

    def blocks(self, x):
        """fp32 arithmetic of the definition: codes and scales of the full blocks of ``x [h, n, d]``."""
        full = x.shape[1] // self.bs
        f = x[:, : full * self.bs].float().reshape(self.h, full, self.bs, self.d)
        s = f.abs().amax(dim=(2, 3))
        s = s / torch.full_like(s, 127.0)      # a quotient: by a Python number torch multiplies by its rounded reciprocal
        c = torch.where(s[..., None, None] > 0, torch.round(f / s[..., None, None]), 0.0)
        return c, s

    def dense(self, x):
        c, s = self.blocks(x)
        done = (c.double() * s.double()[..., None, None]).reshape(self.h, -1, self.d)
        return torch.cat([done, x[:, done.shape[1]:].double()], 1)

    def attend(self, r, q, seen, scale):
        """``q [hq, d]`` over the first ``seen`` tokens -> output and the bound of its error, both float64."""
        k, v = self.dense(self.k[r])[:, :seen], self.dense(self.v[r])[:, :seen]
        qq = q.double().view(self.h, -1, self.d)
        s = qq @ k.transpose(1, 2) * scale
        p = torch.softmax(s, -1)
        o = p @ v
        # Error of a score: 2 d + 2 roundings of fp32 sums of |q| |k|, two scale products; doubled for the softmax's numerator and
        # denominator.  Probabilities: fp16 rounding 2^-11 for a bf16 result, two terms (2^-16 and less) in fp16 and for open rows;
        # ex2 and the rescales below 2^-19; those that are subnormal in fp16 lose at most 2^-25 each where the largest is at
        # least 2^4.  Sums of the products: fp32.
        mag = (qq.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * scale
        rel = (2.0 ** -11 if self.dtype is torch.bfloat16 else 2.0 ** -16) + 2 * ((2 * self.d + 8) * 2.0 ** -24 * mag) + 2.0 ** -18
        out_step = torch.finfo(self.dtype).eps / 2
        bound = rel * (p @ v.abs()) + seen * 2.0 ** -29 * v.abs().amax(1, keepdim=True) + out_step * o.abs() * 1.01 + 1e-30
        if self.dtype is torch.float16:
            bound = bound + 2.0 ** -25
        return o.reshape(-1, self.d), bound.reshape(-1, self.d)


def _rand(shape, seed, dtype, outliers=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(shape, device=DEV, generator=g)
    if outliers:
        x[..., 3] *= 12.0
    return x.to(dtype)


def _cache(requests, h, d, bs, dtype, blocks=200, max_len=2048, layers=1):
    return PagedKVCache(layers, h, d, PagedKVConfig(blocks, bs, requests, max_len), dtype=dtype, device=DEV)


def _feed(cache, model, new, seed, layer=0):
    """One step of ``new`` tokens per request, appended to the cache and to the model."""
    step = cache.plan(new)
    k = _rand((step.tokens, model.h, model.d), seed, model.dtype, outliers=True)
    v = _rand((step.tokens, model.h, model.d), seed + 1, model.dtype)
    cache.append(layer, step, k, v)
    row = 0
    for r, n in enumerate(new):
        if n:
            model.add(r, k[row:row + n], v[row:row + n])
            row += n
    return step, k, v


def _check_attend(model, step, new, q, out, scale=None):
    scale = scale or 1 / math.sqrt(model.d)
    row = 0
    for r, n in enumerate(new):
        for i in range(n):
            seen = model.k[r].shape[1] - n + i + 1
            want, bound = model.attend(r, q[row], seen, scale)
            off = (out[row].double() - want).abs()
            assert bool((off <= bound).all()), (r, i, seen, float((off / bound).max()))
            row += 1


# ---- tables ----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("requests,bs,rows_extra,most", [(1, 16, 0, 1), (1, 32, 3, 700), (5, 16, 0, 40), (64, 32, 8, 1), (64, 64, 0, 300),
                                                         (700, 16, 5, 30), (4096, 16, 0, 3)])
def test_plan_matches_plain(requests, bs, rows_extra, most, cuda_lib):
    rng = random.Random(requests * 100 + bs)
    for trial in range(4):
        old = [rng.choice([0, 0, 1, bs - 1, bs, bs + 1, rng.randrange(5 * bs)]) for _ in range(requests)]
        new = [rng.choice([0, 1, rng.randrange(most + 1)]) for _ in range(requests)]
        rows = sum(new) + rows_extra
        width = max(-(-(a + n) // bs) for a, n in zip(old, new)) + 2
        have = [-(-a // bs) for a in old]
        blocks = sum(-(-(a + n) // bs) for a, n in zip(old, new)) + trial      # trial 0: not one block to spare
        ids = list(range(blocks))
        rng.shuffle(ids)
        table, at = [], 0
        for n in have:
            table.append(ids[at:at + n] + [7777] * (width - n))
            at += n
        free = ids[at:]
        want = _ref_plan(old, new, table, free, len(free), bs, rows)
        dev_table = _i32(table).view(requests, width)
        args = (_i32(old), _i32(new), dev_table, _i32(free + [0] * 3), _i32([len(free)]))
        for again in range(2):                                   # planning again from the same lengths gives the same step
            step = pc.plan_blocks(*args, bs, rows)
            step.check()
            for name in ("query_start", "token_request", "positions", "slots", "seq_lens", "free_count", "context_start"):
                assert getattr(step, name).tolist() == want[name], (name, again)
            assert dev_table.tolist() == want["block_table"]


def test_plan_refuses_as_a_whole(cuda_lib):
    table = torch.full((3, 4), 9, dtype=torch.int32, device=DEV)
    free, bs = _i32([5, 6, 7, 8]), 16
    for old, new, count, rows, flag in (([16, 0, 3], [1, 1, 1], 1, 3, "free blocks"), ([16, 0, 3], [1, 1, 1], 4, 2, "rows"),
                                        ([64, 0, 3], [1, 0, 0], 4, 1, "block table"), ([1, -1, 3], [1, 0, 0], 4, 1, "negative"),
                                        ([1, 1, 3], [1, -2, 0], 4, 1, "negative"), ([1, 1, 3], [1, 0, 0], 5, 1, "free blocks"),
                                        ([1, 1, 3], [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], 4, 4, "rows")):
        step = pc.plan_blocks(_i32(old), _i32(new), table, free, _i32([count]), bs, rows)
        with pytest.raises(RuntimeError, match=flag):
            step.check()
        assert table.eq(9).all() and step.seq_lens.tolist() == old and step.free_count.tolist() == [count]
        assert step.token_request.eq(-1).all() and step.slots.eq(-1).all() and step.positions.eq(-1).all()
        assert step.query_start.eq(0).all() and step.context_start.eq(0).all()
        # and nothing is written by the calls that go on from it
        layer = pc.PagedLayer(*(torch.full((10, 1, bs, 64), 3, dtype=torch.int8, device=DEV) for _ in range(2)),
                              *(torch.full((10, 1), 3.0, device=DEV) for _ in range(2)),
                              *(torch.full((3, 1, bs, 64), 3.0, dtype=torch.float16, device=DEV) for _ in range(2)))
        x = torch.ones(rows, 1, 64, dtype=torch.float16, device=DEV)
        pc.append_blocks(layer, step, x, x)
        out = pc.attend_blocks(layer, step, x, out=torch.full_like(x, 5.0))
        assert all(t.eq(3).all() for t in layer) and out.eq(5).all()


# ---- append, dense ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h,d,bs", [(1, 64, 16), (2, 128, 16), (3, 128, 32), (2, 64, 64), (8, 128, 64), (2, 64, 32)])
def test_append_and_dense_are_exact(h, d, bs, dtype, cuda_lib):
    requests = 5
    cache, model = _cache(requests, h, d, bs, dtype), _Model(requests, h, d, bs, dtype)
    steps = ([1, 0, bs, bs - 1, 3 * bs + 5], [1, 1, 1, 1, 1], [bs, 2 * bs, 2 * bs + 1, bs - 1, 0], [0, 0, 0, 0, 1], [bs - 1, 3, bs + 7, 4 * bs, 200])
    for i, new in enumerate(steps):
        step, _, _ = _feed(cache, model, new, 10 * i)
        layer = cache.layers[0]
        live = [r for r in range(requests) if new[r]]
        dk, dv = pc.dense_blocks(layer, step, sum(model.k[r].shape[1] for r in live) + 3)
        at = 0
        for r in range(requests):
            n = model.k[r].shape[1]
            ids = cache.block_table[r, : n // bs].long()
            for x, codes, scale, tail, dense in ((model.k[r], layer.k_codes, layer.k_scale, layer.tail_k, dk),
                                                 (model.v[r], layer.v_codes, layer.v_scale, layer.tail_v, dv)):
                c, s = model.blocks(x)
                assert torch.equal(codes[ids].transpose(0, 1).float(), c), (i, r)
                assert torch.equal(scale[ids].t(), s)
                assert torch.equal(tail[r, :, : n % bs], x[:, n // bs * bs:])
                if r in live:
                    want = torch.cat([(c * s[..., None, None]).reshape(h, -1, d), x[:, n // bs * bs:].float()], 1)
                    assert torch.equal(dense[at:at + n], want.to(dtype).transpose(0, 1))
            at += n if r in live else 0
        assert dk[at:].eq(0).all() and dv[at:].eq(0).all()


def test_pieces_give_what_one_call_gives(cuda_lib):
    total, bs = 517, 32
    k, v = _rand((total, 2, 128), 1, torch.bfloat16, outliers=True), _rand((total, 2, 128), 2, torch.bfloat16)
    got = []
    for pieces in ([total], [1] * 40 + [total - 40], [31, 1, 32, 33, 95, 100, 225], [500, 17]):
        cache, at = _cache(2, 2, 128, bs, torch.bfloat16), 0
        for n in pieces:
            cache.append(0, cache.plan([0, n]), k[at:at + n], v[at:at + n])
            at += n
        ids = cache.block_table[1, : total // bs].long()
        got.append([t[ids] for t in cache.layers[0][:4]] + [t[1, :, : total % bs] for t in cache.layers[0][4:]])
    assert all(torch.equal(a, b) for other in got[1:] for a, b in zip(got[0], other))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_codes_at_ties_zeros_and_non_finite_blocks(dtype, cuda_lib):
    bs, d = 16, 64
    x = torch.zeros(8 * bs, 1, d, dtype=dtype, device=DEV)
    x[bs, 0, 0] = 254.0                                                  # step 2: every odd number is a tie
    x[bs:2 * bs, 0, 1:] = torch.arange(-7, 8, device=DEV).repeat(100)[: bs * (d - 1)].view(bs, d - 1).to(dtype)
    x[2 * bs:3 * bs] = _rand((bs, 1, d), 3, dtype) * 1e-6 if dtype is torch.float16 else _rand((bs, 1, d), 3, dtype) * 1e-38
    x[3 * bs:4 * bs] = _rand((bs, 1, d), 4, dtype)
    x[3 * bs + 5, 0, 7] = float("inf")
    x[4 * bs:5 * bs] = _rand((bs, 1, d), 5, dtype)
    x[4 * bs + 2, 0, 9] = float("nan")
    x[5 * bs:6 * bs] = (1143.0 / 9 * torch.randint(-18, 19, (bs, 1, d), device=DEV) / 2).to(dtype)   # ties where 1 / step rounds
    x[5 * bs, 0, 0] = 1143.0
    x[6 * bs:7 * bs] = _rand((bs, 1, d), 6, dtype).sign() * torch.finfo(dtype).max
    x[7 * bs:] = _rand((bs, 1, d), 7, dtype)
    cache = _cache(1, 1, d, bs, dtype)
    step = cache.plan([8 * bs])
    cache.append(0, step, x, x)
    model = _Model(1, 1, d, bs, dtype)
    c, s = model.blocks(x.transpose(0, 1))
    ids, layer = cache.block_table[0, :8].long(), cache.layers[0]
    for b in (0, 1, 2, 5, 6, 7):
        assert torch.equal(layer.k_codes[ids[b], 0].float(), c[0, b].clamp(-127, 127)), b
        assert torch.equal(layer.v_scale[ids[b], 0], s[0, b]), b
    dk, _ = pc.dense_blocks(layer, step, 8 * bs)
    for b in range(8):
        assert bool(dk[b * bs:(b + 1) * bs].isfinite().all()) == (b not in (3, 4)), b
    assert layer.k_scale[ids[0], 0] == 0 and dk[:bs].eq(0).all()


# ---- attention -------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h,group,d,bs", [(1, 1, 64, 16), (2, 4, 128, 16), (8, 4, 128, 32), (4, 7, 128, 64), (2, 8, 64, 32), (1, 9, 128, 32),
                                          (2, 16, 128, 16), (1, 28, 64, 64),
                                          (2, 1, 128, 16), (1, 2, 64, 32), (2, 3, 128, 32), (3, 5, 64, 16), (4, 2, 128, 64)])
def test_attend_ragged_steps(h, group, d, bs, dtype, cuda_lib):
    requests = 6
    cache, model = _cache(requests, h, d, bs, dtype, blocks=400), _Model(requests, h, d, bs, dtype)
    # lengths of one token, block borders, empty requests, several new tokens across a border, a long one
    steps = ([1, 0, bs - 1, bs, 2 * bs + 3, 700], [1, 1, 1, 1, 1, 1], [1, 0, 1, 1, 0, 1], [3, 5, 17, bs + 1, 2, 40], [1, 1, 1, 1, 1, 1])
    for i, new in enumerate(steps):
        step, _, _ = _feed(cache, model, new, 100 + 10 * i)
        q = _rand((step.tokens, h * group, d), 105 + 10 * i, dtype)
        out = pc.attend_blocks(cache.layers[0], step, q)
        if i:
            _check_attend(model, step, new, q, out)
        else:
            pick = [r for r in range(requests) if 0 < new[r] < 100]
            sub = [new[r] if r in pick else 0 for r in range(requests)]
            rows = torch.cat([torch.arange(sum(new[:r]), sum(new[:r]) + new[r]) for r in pick])
            _check_attend(model, step, sub, q[rows], out[rows])


@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 4095, 20000])
def test_attend_one_request_of_any_length(tokens, cuda_lib):
    cache, model = _cache(1, 2, 128, 32, torch.bfloat16, blocks=700, max_len=22000), _Model(1, 2, 128, 32, torch.bfloat16)
    if tokens > 1:
        _feed(cache, model, [tokens - 1], 7)
    step, _, _ = _feed(cache, model, [1], 8)
    q = _rand((1, 10, 128), 9, torch.bfloat16)
    _check_attend(model, step, [1], q, pc.attend_blocks(cache.layers[0], step, q))


def test_attend_peaked_and_flat_scores(cuda_lib):
    """A single far larger score, scores that grow from token to token (the reference value moves), and flat ones."""
    cache, model = _cache(3, 1, 128, 16, torch.float16, blocks=300), _Model(3, 1, 128, 16, torch.float16)
    n = 1000
    q = torch.zeros(3, 4, 128, dtype=torch.float16, device=DEV)
    q[..., 0] = 1.0
    step = cache.plan([n] * 3)
    k = torch.zeros(3 * n, 1, 128, dtype=torch.float16, device=DEV)
    k[300, 0, 0] = 2000.0
    k[n:2 * n, 0, 0] = torch.arange(n, device=DEV).half()
    v = _rand((3 * n, 1, 128), 5, torch.float16)
    cache.append(0, step, k, v)
    for r in range(3):
        model.add(r, k[r * n:(r + 1) * n], v[r * n:(r + 1) * n])
    step = cache.plan([1] * 3)
    k1, v1 = torch.zeros(3, 1, 128, dtype=torch.float16, device=DEV), _rand((3, 1, 128), 6, torch.float16)
    out = cache.attend(0, step, q, k1, v1, scale=1.0)
    for r in range(3):
        model.add(r, k1[r:r + 1], v1[r:r + 1])
    _check_attend(model, step, [1] * 3, q, out, scale=1.0)


@pytest.mark.parametrize("tokens", [5, 16, 100])
def test_attend_scores_far_below_zero(tokens, cuda_lib):
    cache, model = _cache(1, 1, 64, 16, torch.bfloat16), _Model(1, 1, 64, 16, torch.bfloat16)
    k = torch.full((tokens, 1, 64), 2.0 ** 54, dtype=torch.bfloat16, device=DEV)
    k[3] *= 0.25                                                       # all scores below -1e32, this one by far the largest
    v = _rand(k.shape, 1, torch.bfloat16)
    step = cache.plan([tokens])
    cache.append(0, step, k, v)
    model.add(0, k, v)
    out = pc.attend_blocks(cache.layers[0], step, torch.full((tokens, 1, 64), -(2.0 ** 53), dtype=torch.bfloat16, device=DEV))
    want = model.dense(model.v[0])[0, 3]
    # one probability is 1 and the others vanish: the result's rounding is below 2^-8 / (1 + 2^-8), those of an fp32 product and quotient below 2^-22
    assert bool(((out[3:, 0].double() - want).abs() <= 2.0 ** -8 * want.abs()).all())


@pytest.mark.parametrize("big", [3e4, 1e-6])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_query_magnitudes(big, dtype, cuda_lib):
    cache, model = _cache(1, 2, 128, 16, dtype), _Model(1, 2, 128, 16, dtype)
    _feed(cache, model, [99], 1)
    step, _, _ = _feed(cache, model, [1], 2)
    q = (_rand((1, 8, 128), 3, torch.float32) * big / 5).to(dtype)
    _check_attend(model, step, [1], q, pc.attend_blocks(cache.layers[0], step, q, scale=1 / (11 * big)), scale=1 / (11 * big))


def test_hidden_rows_do_not_reach_a_query(cuda_lib):
    """Leftovers behind the last open token and later tokens of the same step may be infinite or NaN."""
    for dtype in (torch.float16, torch.bfloat16):
        cache, model = _cache(2, 2, 128, 32, dtype), _Model(2, 2, 128, 32, dtype)
        for t in cache.layers[0][4:]:
            t.fill_(float("nan"))
        step = cache.plan([9, 40])
        k, v = _rand((49, 2, 128), 1, dtype), _rand((49, 2, 128), 2, dtype)
        k[8], v[8] = float("inf"), float("nan")                        # the last token of request 0
        k[47], v[48] = float("nan"), float("inf")                      # the last two of request 1, in its open block
        cache.append(0, step, k, v)
        model.add(0, k[:9], v[:9])
        model.add(1, k[9:], v[9:])
        q = _rand((49, 4, 128), 3, dtype)
        out = pc.attend_blocks(cache.layers[0], step, q)
        row = 0
        for r, n in ((0, 8), (1, 38)):
            for i in range(n):
                # what the query sees: the stored values of the tokens up to its own
                kk, vv = model.k[r][:, : i + 1], model.v[r][:, : i + 1]
                full = 32 if r == 1 else 0
                part = _Model(1, 2, 128, 32, dtype)
                part.k[0], part.v[0] = (x[r][:, :full] if i < full else s for x, s in ((model.k, kk), (model.v, vv)))
                want, bound = part.attend(0, q[row + i], i + 1, 1 / math.sqrt(128))
                assert bool(((out[row + i].double() - want).abs() <= bound).all()), (r, i)
            row += 9
        assert out[8].isnan().all() and out[47:].isnan().any(dim=-1).all()


@pytest.mark.parametrize("group", [1, 2, 4])
def test_blocks_that_fill_up_with_nan_do_not_reach_earlier_tokens(group, cuda_lib):
    """Tokens of a step that share a tile, on both sides of a block's border: the first ones do not see the block behind it."""
    for dtype, d in ((torch.float16, 128), (torch.bfloat16, 64)):
        cache, model = _cache(1, 2, d, 32, dtype), _Model(1, 2, d, 32, dtype)
        _feed(cache, model, [2 if group > 1 else 3], 5)
        n, old = 70, model.k[0].shape[1]
        step = cache.plan([n])
        k, v, q = _rand((n, 2, d), 1, dtype), _rand((n, 2, d), 2, dtype), _rand((n, 2 * group, d), 3, dtype)
        k[40], v[40] = float("nan"), float("inf")                      # in the second block, all of which has no scale any more
        cache.append(0, step, k, v)
        model.add(0, k, v)
        out = pc.attend_blocks(cache.layers[0], step, q)
        first = _Model(1, 2, d, 32, dtype)
        first.k[0], first.v[0] = model.k[0][:, :32], model.v[0][:, :32]
        for i in range(32 - old):
            want, bound = first.attend(0, q[i], old + i + 1, 1 / math.sqrt(d))
            assert bool(((out[i].double() - want).abs() <= bound).all()), i
        assert out[32 - old:].isnan().all()


def test_padded_rows_stay_and_strided_inputs(cuda_lib):
    h, group, d, bs = 2, 4, 128, 16
    cache, model = _cache(4, h, d, bs, torch.bfloat16), _Model(4, h, d, bs, torch.bfloat16)
    _feed(cache, model, [20, 0, 33, 5], 1)
    step = cache.plan({0: 1, 2: 1}, tokens=5)
    qkv = _rand((5, (group + 2) * h, d), 2, torch.bfloat16)             # a fused projection's rows
    q, k, v = qkv.split((group * h, h, h), dim=1)
    wide = torch.full((5, group * h, 2 * d), 7.0, dtype=torch.bfloat16, device=DEV)
    got = cache.attend(0, step, q, k, v, out=wide[..., :d])
    assert got.data_ptr() == wide.data_ptr()
    for i, r in enumerate((0, 2)):
        model.add(r, k[i:i + 1], v[i:i + 1])
    _check_attend(model, step, [1, 0, 1, 0], q, got)
    assert wide[2:].eq(7).all() and wide[..., d:].eq(7).all()
    # rows that are not 16-byte aligned are copied first
    odd = torch.zeros(5 * (h * d + 1) + 8, dtype=torch.bfloat16, device=DEV)
    crooked = odd[1:1 + 5 * (h * d + 1)].view(5, h * d + 1)[:, : h * d].unflatten(1, (h, d))
    crooked.copy_(k)
    again = cache.attend(0, step, q, crooked, v)
    assert torch.equal(again[:2], got[:2])


def test_a_block_that_is_not_in_the_pool_reads_as_nan(cuda_lib):
    cache, model = _cache(2, 2, 64, 16, torch.float16), _Model(2, 2, 64, 16, torch.float16)
    _feed(cache, model, [40, 40], 1)
    before = [t.clone() for t in cache.layers[0]]
    for bad in (-1, 200, 2 ** 31 - 1, -2 ** 31):
        cache.block_table[1, 0] = bad
        step = pc.plan_blocks(cache.seq_lens, _i32([1, 1]), cache.block_table, cache.free_blocks, cache.free_count, 16, 2)
        q = _rand((2, 4, 64), 2, torch.float16)
        k = _rand((2, 2, 64), 3, torch.float16)
        pc.append_blocks(cache.layers[0], step, k, k)
        out = pc.attend_blocks(cache.layers[0], step, q)
        assert out[0].isfinite().all() and out[1].isnan().all()
        dk, dv = pc.dense_blocks(cache.layers[0], step, 82)
        assert dk[:41].isfinite().all() and dk[41:57].isnan().all() and dv[41:57].isnan().all() and dv[57:].isfinite().all()
    # appends leave such a block alone
    cache.block_table[1, 2] = 12345
    step = pc.plan_blocks(cache.seq_lens, _i32([0, 10]), cache.block_table, cache.free_blocks, cache.free_count, 16, 10)
    x = _rand((10, 2, 64), 4, torch.float16)
    pc.append_blocks(cache.layers[0], step, x, x)
    assert all(torch.equal(a, b) for a, b in zip(before[:4], cache.layers[0][:4]))


def test_offsets_beyond_32_bits(cuda_lib):
    h, d, bs, blocks = 8, 128, 64, 36000                                # 2.36e9 codes each for keys and values
    cache, model = _cache(2, h, d, bs, torch.bfloat16, blocks=blocks, max_len=4096), _Model(2, h, d, bs, torch.bfloat16)
    cache.free_blocks.copy_(torch.arange(blocks, dtype=torch.int32))     # the highest ids first
    _feed(cache, model, [200, 130], 1)
    step, _, _ = _feed(cache, model, [1, 1], 2)
    assert int(cache.block_table[0, 0]) * h * bs * d > 2 ** 31
    q = _rand((2, 32, d), 3, torch.bfloat16)
    _check_attend(model, step, [1, 1], q, pc.attend_blocks(cache.layers[0], step, q))
    dk, _ = pc.dense_blocks(cache.layers[0], step, 332)
    assert torch.equal(dk[:201], model.dense(model.k[0]).float().to(torch.bfloat16).transpose(0, 1))


# ---- the class -------------------------------------------------------------------------------------------------------------------

def test_requests_come_and_go(cuda_lib):
    rng = random.Random(3)
    requests, h, d, bs = 5, 2, 128, 16
    cache, model = _cache(requests, h, d, bs, torch.bfloat16, blocks=40, max_len=400), _Model(requests, h, d, bs, torch.bfloat16)
    for i in range(25):
        if i % 4 == 3:
            gone = [r for r in range(requests) if rng.random() < 0.4]
            cache.release(gone)
            for r in gone:
                model.k[r], model.v[r] = (x[:, :0] for x in (model.k[r], model.v[r]))
        new = [rng.choice([0, 1, 1, 2]) if model.k[r].shape[1] else rng.randrange(1, 60) for r in range(requests)]
        need = sum(-(-(model.k[r].shape[1] + n) // bs) for r, n in enumerate(new))
        if need > 40:
            with pytest.raises(RuntimeError, match="blocks needed"):
                cache.plan(new)
            cache.release([0, 1, 2, 3, 4])
            model = _Model(requests, h, d, bs, torch.bfloat16)
            continue
        step, _, _ = _feed(cache, model, new, 1000 + 10 * i)
        step.check()
        assert [cache.seq_len(r) for r in range(requests)] == [x.shape[1] for x in model.k] == cache.seq_lens.tolist()
        assert cache.free_block_count() == 40 - need == int(cache.free_count)
        used = [b for r in range(requests) for b in cache.block_table[r, : -(-model.k[r].shape[1] // bs)].tolist()]
        assert sorted(used + cache.free_blocks[: 40 - need].tolist()) == list(range(40))     # every block exactly once
        q = _rand((step.tokens, 4 * h, d), 1005 + 10 * i, torch.bfloat16)
        _check_attend(model, step, new, q, pc.attend_blocks(cache.layers[0], step, q))


def test_release_of_many_blocks(cuda_lib):
    """More requests than threads and a long one among them: the stack holds their blocks in request order, each once."""
    requests, bs = 700, 16
    cache = _cache(requests, 1, 64, bs, torch.float16, blocks=3000, max_len=20000)
    new = [(17 * r) % 40 for r in range(requests)]
    new[5] = 15000
    cache.plan(new)
    table, free = cache.block_table.tolist(), cache.free_blocks.tolist()
    count = cache.free_block_count()
    assert count == int(cache.free_count) == 3000 - sum(-(-n // bs) for n in new)
    ending = [r for r in range(requests) if r % 3 or r == 699]
    cache.release(ending + ending[:7])
    back = [b for r in ending for b in table[r][: -(-new[r] // bs)]]
    assert cache.free_blocks.tolist() == free[:count] + back + free[count + len(back):]
    assert cache.free_block_count() == int(cache.free_count) == count + len(back)
    assert cache.seq_lens.tolist() == [0 if r in set(ending) else n for r, n in enumerate(new)]
    cache.release(ending)
    assert int(cache.free_count) == count + len(back)


def test_copies_of_a_cache_are_caches_of_their_own(cuda_lib):
    cache, model = _cache(2, 2, 64, 16, torch.float16), _Model(2, 2, 64, 16, torch.float16)
    _feed(cache, model, [40, 9], 1)
    twin = copy.deepcopy(cache)
    layer = pc.PagedLayer._make(cache.layers[0])
    assert twin.layers[0]._c != cache.layers[0]._c != layer._c and layer._replace(tail_k=twin.layers[0].tail_k).tail_k is twin.layers[0].tail_k
    before = [t.clone() for t in (*twin.layers[0], twin.seq_lens, twin.block_table, twin.free_blocks, twin.free_count)]
    _feed(cache, model, [30, 30], 5)
    assert all(torch.equal(a, b) for a, b in zip(before, (*twin.layers[0], twin.seq_lens, twin.block_table, twin.free_blocks, twin.free_count)))
    step = twin.plan([0, 1])
    twin.append(0, step, *(_rand((1, 2, 64), i, torch.float16) for i in (8, 9)))
    assert twin.seq_lens.tolist() == [40, 10] and cache.seq_lens.tolist() == [70, 39]


def test_prefill_then_decode(cuda_lib):
    h, group, d = 2, 4, 128
    cache, model = _cache(3, h, d, 32, torch.bfloat16, layers=2), _Model(3, h, d, 32, torch.bfloat16)
    other = _Model(3, h, d, 32, torch.bfloat16)
    for i, new in enumerate(([70, 0, 129], [33, 200, 0], [1, 1, 1])):
        step = cache.plan(new) if i != 1 else cache.plan(_i32(new), tokens=sum(new))
        for layer, m in ((0, model), (1, other)):
            q, k, v = (_rand((step.tokens, n * h, d), 50 * i + 10 * layer + n, torch.bfloat16) for n in (group, 1, 1))
            v = v.flip(0)
            old = [x.shape[1] for x in m.k]
            past = [(m.dense(m.k[r]), m.dense(m.v[r])) for r in range(3)]
            row = 0
            for r, n in enumerate(new):
                m.add(r, k[row:row + n], v[row:row + n])
                row += n
            if i == 2:
                _check_attend(m, step, new, q, cache.attend(layer, step, q, k, v))
                continue
            out = cache.prefill(layer, step, q, k, v)
            row = 0
            for r, n in enumerate(new):
                if n:
                    # older tokens as they are held (rounded to bf16 by the dense form), the new ones as they came
                    kk = torch.cat([past[r][0].float().bfloat16().double(), k[row:row + n].double().transpose(0, 1)], 1) if old[r] else k[row:row + n].double().transpose(0, 1)
                    vv = torch.cat([past[r][1].float().bfloat16().double(), v[row:row + n].double().transpose(0, 1)], 1) if old[r] else v[row:row + n].double().transpose(0, 1)
                    if old[r]:   # the open block's older tokens may have been quantized by this step's append
                        held = m.dense(m.k[r])[:, : old[r]].float().bfloat16().double(), m.dense(m.v[r])[:, : old[r]].float().bfloat16().double()
                        kk, vv = torch.cat([held[0], kk[:, old[r]:]], 1), torch.cat([held[1], vv[:, old[r]:]], 1)
                    qq = q[row:row + n].double().transpose(0, 1).view(h, group, n, d)
                    s = qq @ kk[:, None].transpose(2, 3) / math.sqrt(d)
                    hide = torch.arange(old[r] + n, device=DEV)[None] > torch.arange(n, device=DEV)[:, None] + old[r]
                    want = (torch.softmax(s.masked_fill(hide, float("-inf")), -1) @ vv[:, None]).reshape(h * group, n, d).transpose(0, 1)
                    off = (out[row:row + n].double() - want).abs()
                    # the prompt attention's probabilities have two bf16 terms: the output's own rounding dominates
                    assert bool((off <= 2.0 ** -8 * want.abs() + 2.0 ** -9).all()), float(off.max())
                row += n


def test_captured_steps_replay(cuda_lib):
    """Planning, append and attention in a graph, lengths on the GPU; two graphs replayed on two streams at once."""
    h, group, d, bs, requests = 2, 4, 128, 16, 4
    streams = [torch.cuda.Stream() for _ in range(2)]
    runs = []
    for w in range(2):
        cache, model = _cache(requests, h, d, bs, torch.float16), _Model(requests, h, d, bs, torch.float16)
        _feed(cache, model, [300 * (w + 1), 15, 16, 0], 11 + w)
        new = _i32([1, 1, 1, 1])
        q, k, v = (torch.zeros(requests, n * h, d, dtype=torch.float16, device=DEV) for n in (group, 1, 1))
        keep = cache._state.clone()
        warm = cache.plan(new, tokens=requests)
        cache.attend(0, warm, q, k, v)
        cache._state.copy_(keep)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step = cache.plan(new, tokens=requests)
            out = cache.attend(0, step, q, k, v)
        runs.append((cache, model, q, k, v, out, step, graph, new))     # a graph reads its inputs where they were
    for i in range(20):
        for w, (cache, model, q, k, v, *_) in enumerate(runs):
            for j, t in enumerate((q, k, v)):
                t.copy_(_rand(t.shape, 1000 * w + 10 * i + j, torch.float16))
        torch.cuda.synchronize()
        for run, stream in zip(runs, streams):
            with torch.cuda.stream(stream):
                run[7].replay()
        torch.cuda.synchronize()
        for cache, model, q, k, v, out, step, _, _ in runs:
            for r in range(requests):
                model.add(r, k[r:r + 1], v[r:r + 1])
            step.check()
            _check_attend(model, step, [1] * requests, q, out)


def test_a_captured_plan_takes_the_lengths_from_the_host(cuda_lib):
    """A replay moves lengths that the host had counted: after it was captured the host asks the GPU, a reset included."""
    cache, model = _cache(2, 1, 128, 16, torch.float16), _Model(2, 1, 128, 16, torch.float16)
    new = _i32([20, 3])
    q, k, v = (_rand((23, n, 128), 7 + n, torch.float16) for n in (2, 1, 1))
    cache.attend(0, cache.plan(new, tokens=23), q, k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(0, cache.plan(new, tokens=23), k, v)
    cache.reset()
    assert cache.seq_len(0) == 0 and cache.free_block_count() == 200
    graph.replay()
    assert cache.seq_len(0) == 20 and cache.free_block_count() == 197
    for r, rows in enumerate((slice(0, 20), slice(20, 23))):
        model.add(r, k[rows], v[rows])
    step = cache.plan([0, 1])
    q1, k1, v1 = (_rand((1, n, 128), 70 + n, torch.float16) for n in (2, 1, 1))
    out = cache.prefill(0, step, q1, k1, v1)
    model.add(1, k1, v1)
    want, bound = model.attend(1, q1[0], 4, 128 ** -0.5)
    assert bool(((out[0].double() - want).abs() <= bound + 2.0 ** -11 * want.abs()).all())       # four open rows: nothing is in 8 bits


def test_two_streams_at_once(cuda_lib):
    h, d, bs = 2, 128, 16
    cache, model = _cache(2, h, d, bs, torch.bfloat16), _Model(2, h, d, bs, torch.bfloat16)
    _feed(cache, model, [900, 333], 1)
    step, _, _ = _feed(cache, model, [1, 1], 2)
    q = [_rand((2, 8, d), 10 + i, torch.bfloat16) for i in range(2)]
    want = [pc.attend_blocks(cache.layers[0], step, x) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(30):
        got = []
        for x, s in zip(q, streams):
            with torch.cuda.stream(s):
                got.append(pc.attend_blocks(cache.layers[0], step, x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))      # and the same bits every time
