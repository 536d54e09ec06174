"""The 8-bit operators together, as a server uses them: a block's projections as integer products, its attention over the paged
cache, requests that come and go.  Every stage is held to its own bound from the inputs that it got."""

import math
import threading

import pytest
import torch
import torch.nn as nn

from pare_b200 import PagedKVCache, PagedKVConfig, QuantConfig, QuantizedLinear
from pare_b200 import paged_cache as pc
from pare_b200.kernels import w8a8_forward
from pare_b200.kv_cache import apply_rope, rope_table
from test_paged_gpu import _check_attend, _i32, _Model, _rand
from test_w8a8_gpu import _check as _check_linear

pytestmark = pytest.mark.gpu

DEV = "cuda"
HIDDEN, HQ, HKV, D = 512, 8, 2, 128


def _layer(n, k, seed):
    torch.manual_seed(seed)
    layer = QuantizedLinear.from_linear(nn.Linear(k, n), QuantConfig(bits=8, scheme="smoothquant", granularity="per_channel", sym=True)).cuda()
    layer.quantize_inputs, layer.use_kernel, layer.int8_kernel = True, True, True
    return layer


def _linear(layer, x):
    y = layer(x)
    n = layer.out_features
    _check_linear(y, x, layer.q_weight, layer.scale.reshape(-1), None, layer.bias)
    assert y.shape == (x.shape[0], n)
    return y


class _Block:
    def __init__(self, dtype, requests=4):
        self.qkv, self.o, self.dtype = _layer((HQ + 2 * HKV) * D, HIDDEN, 1), _layer(HIDDEN, HQ * D, 2), dtype
        self.cache = PagedKVCache(1, HKV, D, PagedKVConfig(60, 16, requests, 300), dtype=dtype, device=DEV)
        self.model = _Model(requests, HKV, D, 16, dtype)
        self.rope = rope_table(300, D, device=DEV)

    def __call__(self, h, step, prompt):
        rows = self.qkv(h) if prompt is None else _linear(self.qkv, h)
        q, k, v = rows.view(-1, HQ + 2 * HKV, D).split((HQ, HKV, HKV), dim=1)
        turn = self.rope[step.positions.long().clamp(min=0)]
        q, k = (apply_rope(x.transpose(0, 1).unsqueeze(0), turn)[0].transpose(0, 1) for x in (q, k))
        a = self.cache.prefill(0, step, q, k, v) if prompt else self.cache.attend(0, step, q, k, v)
        flat = a.reshape(-1, HQ * D)
        return q, k, v, a, (self.o(flat) if prompt is None else _linear(self.o, flat))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompts_decode_and_new_requests(dtype, cuda_lib):
    block = _Block(dtype)
    cache, model = block.cache, block.model
    steps = [([37, 5, 0, 0], True), ([1, 1, 0, 0], False), ([0, 0, 130, 0], True), ([1, 1, 1, 0], False), (None, False), ([64, 0, 0, 9], True),
             ([1, 1, 1, 1], False), ([2, 1, 3, 1], False), ([1, 1, 1, 1], False)]
    for i, (new, prompt) in enumerate(steps):
        if new is None:      # request 0 ends; its number is used again
            cache.release([0])
            model.k[0], model.v[0] = model.k[0][:, :0], model.v[0][:, :0]
            continue
        step = cache.plan(new)
        h = _rand((step.tokens, HIDDEN), 100 + i, dtype)
        q, k, v, a, y = block(h, step, prompt)
        row = 0
        for r, n in enumerate(new):
            assert step.positions[row:row + n].tolist() == list(range(model.k[r].shape[1], model.k[r].shape[1] + n))
            model.add(r, k[row:row + n], v[row:row + n])
            row += n
        if not prompt:
            _check_attend(model, step, new, q, a)
        else:                # the prompts here begin their requests: full precision among themselves
            row = 0
            for n in new:
                if n:
                    qq, kk, vv = (x[row:row + n].double().transpose(0, 1) for x in (q, k, v))
                    s = qq @ kk.repeat_interleave(HQ // HKV, 0).transpose(1, 2) / math.sqrt(D)
                    s = s.masked_fill(torch.ones(n, n, device=DEV, dtype=torch.bool).triu(1), float("-inf"))
                    want = (torch.softmax(s, -1) @ vv.repeat_interleave(HQ // HKV, 0)).transpose(0, 1)
                    # half a step of the result, and as much again of the largest value for the probabilities' rounding
                    half = torch.finfo(dtype).eps / 2
                    assert bool(((a[row:row + n].double() - want).abs() <= half * (want.abs() + vv.abs().max())).all())
                row += n
        assert bool(y.isfinite().all())


def test_a_captured_decode_step_is_the_eager_one(cuda_lib):
    blocks = [_Block(torch.bfloat16) for _ in range(2)]
    for b in blocks:
        b(_rand((60, HIDDEN), 5, torch.bfloat16), b.cache.plan([20, 31, 9, 0]), True)
    new = _i32([1, 1, 1, 0])
    h = _rand((3, HIDDEN), 6, torch.bfloat16)
    eager, captured = blocks
    keep = captured.cache._state.clone()
    captured(h, captured.cache.plan(new, tokens=3), None)          # buffers that are made on the first call
    captured.cache._state.copy_(keep)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = captured(h, captured.cache.plan(new, tokens=3), None)[4]
    for i in range(40):                                             # over several blocks' borders
        h.copy_(_rand((3, HIDDEN), 50 + i, torch.bfloat16))
        graph.replay()
        want = eager(h, eager.cache.plan([1, 1, 1, 0]), None)[4]
        assert torch.equal(y, want), i
    assert torch.equal(captured.cache._state, eager.cache._state)


def test_threads_on_one_stream(cuda_lib):
    """Calls of several threads land in turn on the same stream; each keeps what it works in."""
    cache, model = PagedKVCache(1, 2, 128, PagedKVConfig(300, 16, 2, 4000), dtype=torch.bfloat16, device=DEV), _Model(2, 2, 128, 16, torch.bfloat16)
    step = cache.plan([2000, 1500])
    k, v = _rand((3500, 2, 128), 1, torch.bfloat16), _rand((3500, 2, 128), 2, torch.bfloat16)
    cache.append(0, step, k, v)
    step = cache.plan([1, 1])
    cache.append(0, step, k[:2], v[:2])
    x = [_rand((m, 1024), 10 + m, torch.bfloat16) for m in (40, 100)]
    w = torch.randint(-127, 128, (700, 1024), device=DEV, dtype=torch.int8)
    scale = torch.rand(700, device=DEV)
    q = [_rand((2, 8, 128), 20 + i, torch.bfloat16) for i in range(2)]
    want = [(w8a8_forward(x[i], w, scale), pc.attend_blocks(cache.layers[0], step, q[i])) for i in range(2)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        for _ in range(200):
            got = (w8a8_forward(x[i], w, scale), pc.attend_blocks(cache.layers[0], step, q[i]))
            if not (torch.equal(got[0], want[i][0]) and torch.equal(got[1], want[i][1])):
                wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_an_empty_step(cuda_lib):
    cache = PagedKVCache(1, 2, 64, PagedKVConfig(10, 16, 3, 100), dtype=torch.float16, device=DEV)
    for tokens in (0, 4):
        step = cache.plan([0, 0, 0], tokens=tokens)
        step.check()
        x = torch.ones(tokens, 2, 64, dtype=torch.float16, device=DEV)
        out = cache.attend(0, step, torch.ones(tokens, 4, 64, dtype=torch.float16, device=DEV), x, x,
                           out=torch.full((tokens, 4, 64), 3.0, dtype=torch.float16, device=DEV))
        assert out.shape == (tokens, 4, 64) and out.eq(3).all() and cache.free_block_count() == 10
        k, v = pc.dense_blocks(cache.layers[0], step, 0)
        assert k.shape == v.shape == (0, 2, 64) and step.positions.tolist() == [-1] * tokens


def test_refusals(cuda_lib):
    cache = PagedKVCache(1, 2, 64, PagedKVConfig(10, 16, 3, 100), dtype=torch.float16, device=DEV)
    layer = cache.layers[0]
    for bad in ([1, 2], [1, -1, 0], {3: 1}, [101, 0, 0]):
        with pytest.raises(ValueError):
            cache.plan(bad)
    with pytest.raises(RuntimeError, match="blocks needed"):
        cache.plan([80, 80, 10])
    with pytest.raises(ValueError, match="rows"):
        cache.plan([1, 1, 1], tokens=2)
    with pytest.raises(ValueError, match="rows is needed"):
        cache.plan(_i32([1, 1, 1]))
    with pytest.raises(ValueError):
        cache.release([3])
    assert cache.seq_lens.tolist() == [0, 0, 0] and cache.free_block_count() == 10
    step = cache.plan([1, 1, 0])
    good = torch.zeros(2, 2, 64, dtype=torch.float16, device=DEV)
    for bad in (good[:1], good.bfloat16(), good.cpu(), good[..., :32], good.expand(2, 2, 64)[:, :1]):
        with pytest.raises(ValueError, match="k must be"):
            cache.append(0, step, bad, good)
    for bad in (good[:, :1], good[:, :0], good[:1], good[0], good.float()):
        with pytest.raises(ValueError):
            pc.attend_blocks(layer, step, bad)
    with pytest.raises(ValueError, match="out must be"):
        pc.attend_blocks(layer, step, good, out=good.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="prefill needs"):
        cache.prefill(0, step, good, good, good)
    other = PagedKVCache(1, 2, 64, PagedKVConfig(10, 32, 3, 100), dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match="do not belong together"):
        other.append(0, step, good, good)
    with pytest.raises(ValueError, match="paged layer"):
        pc.PagedLayer(*layer[:4], layer.tail_k, layer.tail_v[:1])
    with pytest.raises(ValueError, match="paged layer"):
        pc.PagedLayer(layer.k_codes.transpose(0, 1), *layer[1:])
    lens = (cache.seq_lens, _i32([1, 1, 0]), cache.block_table, cache.free_blocks, cache.free_count)
    for i, bad in ((0, lens[0].long()), (1, lens[1][:2]), (2, cache.block_table.t()), (2, cache.block_table[:2]), (3, cache.free_blocks[::2]),
                   (4, cache.free_count.expand(2)), (2, cache.block_table[:, :0])):
        with pytest.raises(ValueError):
            pc.plan_blocks(*(bad if i == j else t for j, t in enumerate(lens)), 16, 2)
    for bs, rows in ((8, 2), (128, 2), (16, -1)):
        with pytest.raises(ValueError):
            pc.plan_blocks(*lens, bs, rows)
    long = PagedKVCache(1, 2, 128, PagedKVConfig(10, 16, 3, 100), dtype=torch.float16, device=DEV)
    step, rows = long.plan([3, 0, 0]), torch.zeros(3, 2, 128, dtype=torch.float16, device=DEV)
    for bad in (rows[:2], rows[0], rows.float(), rows.cpu()):
        with pytest.raises((ValueError, IndexError)):
            long.prefill(0, step, bad, rows, rows)
    many = PagedKVCache(1, 1, 64, PagedKVConfig(300, 16, 1, 4800), dtype=torch.float16, device=DEV)
    step = many.plan([4097])
    with pytest.raises(ValueError, match="at most 4096"):
        pc.attend_blocks(many.layers[0], step, torch.zeros(4097, 1, 64, dtype=torch.float16, device=DEV))


def test_outputs_beyond_32_bits(cuda_lib):
    m, n, k = 70000, 32768, 64                                       # 2.3e9 outputs
    x, w = _rand((m, k), 1, torch.bfloat16), torch.randint(-127, 128, (n, k), device=DEV, dtype=torch.int8)
    scale = torch.rand(n, device=DEV) + 0.1
    y = w8a8_forward(x, w, scale)
    pick = torch.tensor([0, 1, 40000, 65535, 65536, 69999], device=DEV)
    _check_linear(y[pick], x[pick], w, scale)
    _check_linear(y[-300:], x[-300:], w, scale)
