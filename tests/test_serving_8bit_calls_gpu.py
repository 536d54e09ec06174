"""Calls of the 8-bit operators that the tests of each operator do not make: precision between roundings, steps and layers that change
under a program, calls that are refused half way, other streams."""

import math

import pytest
import torch
import torch.nn as nn

from pare_b200 import QuantConfig, QuantizedLinear
from pare_b200 import paged_cache as pc
from pare_b200.kernels import w8a8_forward
from test_paged_gpu import _cache, _check_attend, _feed, _Model, _rand
from test_w8a8_gpu import _check as _check_linear

pytestmark = pytest.mark.gpu

DEV = "cuda"


# ---- attention: nothing but the result is rounded to 16 bits ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h,group,d,new", [(2, 4, 128, 1), (8, 4, 128, 1), (4, 7, 128, 1), (2, 8, 64, 1), (2, 1, 128, 4), (2, 2, 64, 3)])
def test_probabilities_keep_more_than_the_result(h, group, d, new, dtype, cuda_lib):
    """A probability rounded to one 16-bit number would change a tenth of the bf16 results."""
    cache, model = _cache(2, h, d, 16, dtype, blocks=400), _Model(2, h, d, 16, dtype)
    _feed(cache, model, [1500, 333], 1)
    step, _, _ = _feed(cache, model, [new, new], 2)
    q = _rand((2 * new, h * group, d), 3, dtype)
    out = pc.attend_blocks(cache.layers[0], step, q)
    wrong = total = 0
    for row in range(2 * new):
        r = row // new
        seen = model.k[r].shape[1] - new + row % new + 1
        k, v = model.dense(model.k[r])[:, :seen], model.dense(model.v[r])[:, :seen]
        qq = q[row].double().view(h, group, d)
        s = qq @ k.transpose(1, 2) / math.sqrt(d)
        p = torch.softmax(s, -1)
        want = (p @ v).reshape(-1, d)
        # Before the result's own rounding.  Scores: sums of d products in fp32, 2 d + 8 roundings of the magnitudes at most, twice (numerator and
        # denominator).  Probabilities in two terms: 2^-16 of them; ex2 and the rescales 2^-18; what is subnormal in fp16 loses at most
        # 2^-25 where the largest is 2^4 or more.
        mag = (qq.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) / math.sqrt(d)
        rel = 2.0 ** -16 + 2 * ((2 * d + 8) * 2.0 ** -24 * mag) + 2.0 ** -18
        bound = (rel * (p @ v.abs()) + seen * 2.0 ** -29 * v.abs().amax(1, keepdim=True)).reshape(-1, d)
        half = torch.finfo(dtype).eps / 2 * want.abs() * (1 + torch.finfo(dtype).eps) + (2.0 ** -25 if dtype is torch.float16 else 0)
        assert bool(((out[row].double() - want).abs() <= half + bound).all())
        wrong += int((out[row] != want.to(dtype)).sum())
        total += want.numel()
    # An error of `bound` crosses a border between two results with a probability of 2 bound / step; the errors are far smaller than
    # their bounds, so one result in fifty is more than what two terms can change and less than what one term does.
    assert wrong <= total / 50 if dtype is torch.bfloat16 else wrong <= total / 10


# ---- a cache's tensors --------------------------------------------------------------------------------------------------------------

def test_a_new_cache_holds_numbers(cuda_lib):
    """Copies and comparisons of a cache's tensors do not meet what other tensors left in their memory."""
    shape = (4, 2, 16, 128)
    left = [torch.full(shape, float("nan"), dtype=torch.float16, device=DEV) for _ in range(400)]
    del left                                                # their memory is what the next small tensors get
    layer = _cache(4, 2, 128, 16, torch.float16).layers[0]
    assert layer.tail_k.shape == shape and all(t.eq(0).all() for t in layer[2:])


# ---- steps that a graph writes again ------------------------------------------------------------------------------------------------

def _prompt(q, k, v):
    """Causal attention of a prompt's rows ``[n, heads, d]`` among themselves in 64 bits, and the bound of a 16-bit result's error."""
    qq, kk, vv = (x.double().transpose(0, 1) for x in (q, k, v))
    n, group = q.shape[0], q.shape[1] // k.shape[1]
    s = qq @ kk.repeat_interleave(group, 0).transpose(1, 2) / math.sqrt(q.shape[2])
    s = s.masked_fill(torch.ones(n, n, device=DEV, dtype=torch.bool).triu(1), float("-inf"))
    want = (torch.softmax(s, -1) @ vv.repeat_interleave(group, 0)).transpose(0, 1)
    # half a step of the result, and as much again of the largest value for the probabilities' rounding
    return want, torch.finfo(q.dtype).eps / 2 * (want.abs() + vv.abs().max())


@pytest.mark.parametrize("planned_by", ["class", "function"])
def test_prefill_after_replays_of_a_captured_plan(planned_by, cuda_lib):
    """Every replay gives the step other lengths; prefill has to go by those of the last one."""
    cache = _cache(3, 2, 128, 16, torch.float16, blocks=100, layers=2)
    new = torch.tensor([20, 0, 3], dtype=torch.int32, device=DEV)
    rows = 40

    def plan():
        if planned_by == "class":
            return cache.plan(new, tokens=rows)
        return pc.plan_blocks(cache.seq_lens, new, cache.block_table, cache.free_blocks, cache.free_count, 16, rows)

    plan()
    cache.reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = plan()
    for i, lens in enumerate(([20, 0, 3], [5, 30, 2], [0, 0, 40], [40, 0, 0], [1, 1, 1])):
        cache.reset()
        new.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        for layer in range(2):
            q, k, v = (_rand((rows, n, 128), 100 * i + 10 * layer + n, torch.float16) for n in (8, 2, 1))
            v = v.expand(rows, 2, 128)
            out = cache.prefill(layer, step, q, k, v)
            at = 0
            for n in lens:
                if n:
                    want, bound = _prompt(q[at:at + n], k[at:at + n], v[at:at + n])
                    assert bool(((out[at:at + n].double() - want).abs() <= bound).all()), (i, layer, n)
                at += n
    new.copy_(torch.tensor([41, 0, 0], dtype=torch.int32))
    graph.replay()
    with pytest.raises(RuntimeError, match="refused"):
        cache.prefill(0, step, q, k, v)


def test_prefill_reads_an_eager_step_once(cuda_lib):
    cache = _cache(2, 2, 128, 16, torch.float16, blocks=20, layers=2)
    step = cache.plan(torch.tensor([5, 0], dtype=torch.int32, device=DEV), tokens=5)
    q = _rand((5, 2, 128), 1, torch.float16)
    assert step.lengths is None
    cache.prefill(0, step, q, q, q)
    assert step.lengths == [(0, 5), (0, 0)]


# ---- refusals half way --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("call", ["attend", "prefill"])
def test_a_refused_call_has_stored_nothing(call, cuda_lib):
    """A block fills up and the rows behind it are written again: what a refused call had stored could not be stored a second time."""
    cache, model = _cache(2, 2, 128, 16, torch.float16, blocks=100), _Model(2, 2, 128, 16, torch.float16)
    _feed(cache, model, [10, 3], 1)
    new = [30, 1]
    step = cache.plan(new)
    q, k, v = (_rand((31, n, 128), 5 + n, torch.float16) for n in (8, 2, 1))
    v = v.expand(31, 2, 128).contiguous()
    before = [t.clone() for t in cache.layers[0]]
    go = getattr(cache, call)
    bad_out = [] if call == "prefill" else [lambda: go(0, step, q, k, v, out=q.transpose(1, 2).contiguous().transpose(1, 2)),
                                            lambda: go(0, step, q, k, v, out=q.float())]
    for refused in (lambda: go(0, step, q[:, :7], k, v), lambda: go(0, step, q[:, :0], k, v), lambda: go(0, step, q[:30], k, v),
                    lambda: go(0, step, q.float(), k, v), lambda: go(0, step, q, k[:30], v), lambda: go(0, step, q, k, v[:, :1]),
                    lambda: go(0, step, q, k, v, scale="?"), *bad_out):
        with pytest.raises((ValueError, IndexError)):
            refused()
        assert all(torch.equal(a, b) for a, b in zip(before, cache.layers[0]))
    out = go(0, step, q, k, v)
    model.add(0, k[:30], v[:30])
    model.add(1, k[30:], v[30:])
    if call == "attend":
        _check_attend(model, step, new, q, out)
    for r in range(2):
        n = model.k[r].shape[1] // 16
        ids = cache.block_table[r, :n].long()
        assert torch.equal(cache.layers[0].k_codes[ids].transpose(0, 1).float(), model.blocks(model.k[r])[0])


def test_too_many_rows_for_attention_are_not_stored(cuda_lib):
    cache = _cache(1, 1, 64, 16, torch.float16, blocks=300, max_len=4800)
    step = cache.plan([4097])
    q, k = torch.ones(4097, 1, 64, dtype=torch.float16, device=DEV), torch.ones(4097, 1, 64, dtype=torch.float16, device=DEV)
    before = [t.clone() for t in cache.layers[0]]
    with pytest.raises(ValueError, match="at most 4096"):
        cache.attend(0, step, q, k, k)
    assert all(torch.equal(a, b) for a, b in zip(before, cache.layers[0]))


# ---- integer layers -----------------------------------------------------------------------------------------------------------------

def _layer(k=500, n=300, seed=0, sym=False, granularity="per_channel", input_scale=False):
    torch.manual_seed(seed)
    layer = QuantizedLinear.from_linear(nn.Linear(k, n), QuantConfig(bits=8, scheme="smoothquant", granularity=granularity, sym=sym))
    if input_scale:
        layer.input_scale = 0.5 + torch.rand(k)
    layer.quantize_inputs, layer.use_kernel, layer.int8_kernel = True, True, True
    return layer.cuda()


def _as_defined(layer, x):
    n = layer.out_features
    ins = None if layer.input_scale is None else layer.input_scale.float()
    y = layer(x)
    _check_linear(y, x, layer.q_weight, layer.scale.float().reshape(-1).expand(n), layer.zero.float().reshape(-1).expand(n), layer.bias, ins)
    return y


@pytest.mark.parametrize("k", [500, 512])
@pytest.mark.parametrize("granularity", ["per_channel", "per_tensor"])
def test_layer_follows_its_tensors(granularity, k, cuda_lib):
    """Weights, scales and zero-points that are replaced or written to between calls."""
    x = torch.randn(5, k, device=DEV, dtype=torch.float16)
    layer = _layer(k, granularity=granularity, sym=True)
    _as_defined(layer, x)
    layer.zero.copy_(torch.tensor(7.0))                     # a zero-point where there was none
    _as_defined(layer, x)
    layer.scale.mul_(3.0)
    _as_defined(layer, x)
    layer.q_weight.copy_(layer.q_weight.flip(0))
    _as_defined(layer, x)
    layer.zero.zero_()
    _as_defined(layer, x)
    made = layer._int8_made
    _as_defined(layer, x)
    assert layer._int8_made is made                         # nothing is made again while nothing changes
    old = layer.scale.clone(), layer.q_weight.clone()
    gone = layer.scale, layer.q_weight
    layer.scale, layer.zero = layer.scale * 2, layer.zero - 3.0
    _as_defined(layer, x)
    layer.q_weight = -layer.q_weight.clamp(-127, 127)
    _as_defined(layer, x)
    assert torch.equal(gone[0], old[0]) and torch.equal(gone[1], old[1])      # what was replaced is left alone


def test_a_captured_layer_follows_a_loaded_state(cuda_lib):
    """Loading writes into the layer's tensors; after the next call a graph that was captured before reads them too."""
    first, other = _layer(seed=1), _layer(seed=2)
    x = torch.randn(5, 500, device=DEV, dtype=torch.float16)
    first(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = first(x)
    first.load_state_dict(other.state_dict())
    want = _as_defined(first, x)
    torch.empty(1 << 20, dtype=torch.uint8, device=DEV).fill_(77)             # freed memory would be in use again
    graph.replay()
    assert torch.equal(y, want) and torch.equal(want, other(x))


@pytest.mark.parametrize("first", [torch.inference_mode, torch.no_grad])
@pytest.mark.parametrize("then", [torch.inference_mode, torch.no_grad, torch.enable_grad])
def test_layer_follows_a_loaded_state_across_modes(first, then, cuda_lib):
    layer, other = _layer(granularity="per_tensor", seed=1, input_scale=True), _layer(granularity="per_tensor", seed=2, input_scale=True)
    x = torch.randn(5, 500, device=DEV, dtype=torch.float16)
    with first():
        _as_defined(layer, x)
    layer.load_state_dict(other.state_dict())
    with then():
        assert torch.equal(_as_defined(layer, x), other(x))


def test_a_captured_layer_stays_where_a_move_moves_nothing(cuda_lib):
    layer = _layer(input_scale=True)
    x = torch.randn(20, 500, device=DEV, dtype=torch.float16)
    want = _as_defined(layer, x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
    names = ("_q_weight_int8", "_scale_int8", "_zero_int8", "_input_scale_int8")
    read = [layer._buffers[name] for name in names]
    for move in (lambda: layer.cuda(), lambda: layer.to(DEV), lambda: layer.to(torch.float32)):
        assert move() is layer
        assert all(layer._buffers[name] is t for name, t in zip(names, read))
    y.zero_()
    graph.replay()
    assert torch.equal(y, want) and torch.equal(layer(x), want)
    keys = set(layer.state_dict())
    layer.half()
    assert not any(name in layer._buffers for name in names) and set(layer.state_dict()) == keys
    _as_defined(layer, x)
    assert set(layer.state_dict()) == keys


def test_a_layer_that_two_streams_call_first(cuda_lib, monkeypatch):
    """The first call makes the derived tensors on its stream; the next one, on another stream, finds them made."""
    from pare_b200.layers import linear

    copy = linear.aligned_rows

    def late(q_weight):
        torch.cuda._sleep(200_000_000)                      # a tenth of a second: the copy ends long after the call has returned
        return copy(q_weight)

    layer, same = _layer(seed=3), _layer(seed=3)
    x = torch.randn(20, 500, device=DEV, dtype=torch.float16)
    want = same(x)
    torch.cuda.synchronize()
    monkeypatch.setattr(linear, "aligned_rows", late)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(layer(x))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 20])
def test_a_smoothed_layer_in_a_16_bit_model(rows, dtype, cuda_lib):
    """A cast of the module rounds input_scale too; the product then divides by the rounded one in float32, as the eager branch does."""
    layer = _layer(512, input_scale=True)
    x = torch.randn(rows, 512, device=DEV).to(dtype)
    _as_defined(layer, x)
    layer.to(dtype)
    assert layer.input_scale.dtype is dtype
    _as_defined(layer, x)
    layer.input_scale.mul_(2.0)
    _as_defined(layer, x)
    layer.input_scale = (0.5 + torch.rand(1024, device=DEV))[::2]
    _as_defined(layer, x)
    layer.input_scale = None
    _as_defined(layer, x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_activations_of_more_than_16_bits_stay_what_they_are(dtype, cuda_lib):
    layer = _layer(512, input_scale=True)
    x = torch.randn(4, 512, device=DEV, dtype=dtype)
    x[1, 7], x[2] = 3e5, x[2] * 1e-9                        # beyond float16, on either side
    layer.int8_kernel = False
    if dtype is torch.float64:
        layer.double()
    want = layer(x)
    layer.int8_kernel = True
    y = layer(x)
    assert y.dtype is dtype and bool(y.isfinite().all()) and torch.equal(y, want)


def test_layer_refuses_what_it_was_changed_to(cuda_lib):
    """A layer that has run and then stops quantizing its inputs, or gets an order of columns, is not the integer product's any more."""
    layer, x = _layer(), torch.randn(3, 500, device=DEV, dtype=torch.float16)
    _as_defined(layer, x)
    layer.quantize_inputs = False
    with pytest.raises(ValueError, match="int8_kernel needs"):
        layer(x)
    layer.quantize_inputs = True
    _as_defined(layer, x)
    layer.g_idx = torch.arange(500, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="int8_kernel needs"):
        layer(x)


# ---- linear -------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", [24064, 24072, 24448, 24456, 24560, 24568, 24576, 24584])
@pytest.mark.parametrize("m", [12, 300, 600, 1300])
def test_rows_of_about_48_kilobytes(m, k, dtype, cuda_lib):
    """A row waits in shared memory between maximum and codes: beside it there is the kernel's static shared memory."""
    g = torch.Generator(device=DEV).manual_seed(m + k)
    x = torch.randn(m, k, device=DEV, generator=g).to(dtype)
    w = torch.randint(-128, 128, (130, k), device=DEV, generator=g, dtype=torch.int8)
    scale, ins = torch.rand(130, device=DEV, generator=g) * 1e-3, 0.5 + torch.rand(k, device=DEV, generator=g)
    _check_linear(w8a8_forward(x, w, scale), x, w, scale)
    _check_linear(w8a8_forward(x, w, scale, input_scale=ins), x, w, scale, None, None, ins)
