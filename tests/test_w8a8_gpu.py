"""W8A8 linear on the GPU against the definition: codes in the float32 arithmetic it names, sums in 64-bit integers, the rest in float64."""

import copy

import pytest
import torch
import torch.nn as nn

from pare_b200 import QuantConfig, QuantizedLinear
from pare_b200.kernels import w8a8_forward

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _codes(x, input_scale=None):
    """``(codes int64, step float32)`` of the definition."""
    if input_scale is not None:
        x = (x.float() / input_scale).to(x.dtype)
    f = x.float()
    step = f.abs().amax(1, keepdim=True).clamp(min=1e-6)
    step = step / torch.full_like(step, 127.0)
    return torch.round(f / step).clamp(-127, 127).long(), step


def _check(got, x, w, scale, zero=None, bias=None, input_scale=None):
    c, step = _codes(x, input_scale)
    acc = (c.double() @ w.double().t())                       # exact: below 2^53
    xs = c.sum(1, keepdim=True).double()
    z = torch.zeros_like(scale).double() if zero is None else zero.double()
    s = step.double() * scale.double()
    want = (acc - z * xs) * s + (0 if bias is None else bias.to(x.dtype).double())
    # one rounding each: int -> float, step * scale, the last product and sum; a zero-point that is not whole (or beyond 128) adds
    # the product and difference of its rest
    exact_z = (z == z.round()) & (z.abs() <= 128)
    mag = (acc - z * xs).abs() + torch.where(exact_z, 0.0, 2 * acc.abs() + 2 * (z * xs).abs())
    bound = torch.finfo(x.dtype).eps / 2 * want.abs() * 1.01 + 2.0 ** -22 * (mag * s.abs() + want.abs()) + 1e-30
    if x.dtype is torch.float16:
        bound = bound + 2.0 ** -25
    off = (got.double() - want).abs()
    # Rounding to nearest gives an infinity from half a step above the type's largest number on (float16: 65504 + 16): there `got` is
    # infinite with the sign of `want`, and no finite bound says anything about the difference.
    top = torch.finfo(x.dtype).max
    over = want.abs() + bound >= top * (1 + torch.finfo(x.dtype).eps / 4)
    assert bool(((off <= bound) | (over & (got.double() == want.sign() * float("inf")))).all())


def _data(m, n, k, seed, dtype):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(m, k, device=DEV, generator=g).to(dtype)
    w = torch.randint(-128, 128, (n, k), device=DEV, generator=g, dtype=torch.int8)
    scale = (0.5 + torch.rand(n, device=DEV, generator=g)) * 1e-3
    return x, w, scale, g


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 16), (2, 129, 100), (15, 257, 130), (16, 512, 4096), (17, 300, 1000), (63, 128, 128),
                                   (129, 1000, 2064), (255, 130, 384), (257, 384, 1111), (333, 3584, 2368), (600, 640, 5000),
                                   (20, 300, 8200), (65, 1500, 16384), (250, 200, 8192), (513, 300, 9000)])
def test_sizes(m, n, k, dtype, cuda_lib):
    x, w, scale, g = _data(m, n, k, m + n + k, dtype)
    _check(w8a8_forward(x, w, scale), x, w, scale)
    zero = torch.randint(-128, 128, (n,), device=DEV, generator=g).float()
    bias = torch.randn(n, device=DEV, generator=g)
    ins = 0.3 + 3 * torch.rand(k, device=DEV, generator=g)
    _check(w8a8_forward(x, w, scale, zero, bias=bias, input_scale=ins), x, w, scale, zero, bias, ins)


@pytest.mark.parametrize("m", [1, 16, 40, 130])
def test_long_rows_and_split_sums(m, cuda_lib):
    """One or two weight tiles over a long K: every thread block has a part of the same tile."""
    x, w, scale, _ = _data(m, 200, 18944, m, torch.bfloat16)
    y = w8a8_forward(x, w, scale)
    _check(y, x, w, scale)
    assert all(torch.equal(y, w8a8_forward(x, w, scale)) for _ in range(20))


def test_largest_sums(cuda_lib):
    k = 65536
    x = torch.ones(3, k, dtype=torch.float16, device=DEV)
    x[1] = -1
    w = torch.full((130, k), -128, dtype=torch.int8, device=DEV)
    scale = torch.full((130,), 1e-6, device=DEV)
    zero = torch.full((130,), 128.0, device=DEV)
    _check(w8a8_forward(x, w, scale), x, w, scale)
    _check(w8a8_forward(x, w, scale, zero), x, w, scale, zero)


def test_zero_points_of_any_value(cuda_lib):
    x, w, scale, g = _data(20, 256, 300, 1, torch.bfloat16)
    zero = torch.randn(256, device=DEV, generator=g) * torch.logspace(-3, 4, 256, device=DEV)
    _check(w8a8_forward(x, w, scale, zero), x, w, scale, zero)


@pytest.mark.parametrize("m", [3, 40, 700])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_smoothing_divides_exactly(dtype, m, cuda_lib):
    """Every code by itself (the weights are 127 times the identity): scales of any size, powers of two and their neighbours, signs."""
    k, span = 512, 6 if dtype is torch.float16 else 100
    g = torch.Generator(device=DEV).manual_seed(m)
    e = torch.randint(-span, span + 1, (k,), device=DEV, generator=g).double()
    u = 0.5 + torch.rand(k, device=DEV, generator=g).double()
    u[::7], u[1::7], u[2::7], u[3::7] = 1.0, 1.0 + 2.0 ** -23, 1.0 - 2.0 ** -24, -1.5
    ins = (u * 2.0 ** e).float()
    x = (torch.randn(m, k, device=DEV, generator=g).double().clamp(-3, 3) * 2.0 ** e).to(dtype)
    x[0, ::5], x[1, 7] = 0.0, float("inf")
    w = 127 * torch.eye(k, dtype=torch.int8, device=DEV)
    got = w8a8_forward(x, w, torch.ones(k, device=DEV), input_scale=ins)
    assert got[1].isnan().all()
    keep = [i for i in range(m) if i != 1]
    _check(got[keep], x[keep], w, torch.ones(k, device=DEV), None, None, ins)


def test_ties_tiny_and_non_finite_rows(cuda_lib):
    for dtype in (torch.float16, torch.bfloat16):
        x, w, scale, g = _data(8, 128, 256, 2, dtype)
        x[0] = 0
        x[1] = torch.arange(-128, 128, device=DEV).to(dtype)
        x[1, 0] = 254.0                                                    # step 2: odd numbers are ties
        x[2] = (1143.0 / 9 * torch.randint(-18, 19, (256,), device=DEV) / 2).to(dtype)
        x[2, 5] = 1143.0                                                   # step 9 (fp16): ties where 1 / step is rounded
        x[3] = (x[3].float() * 1e-7).to(dtype)                             # below the smallest step
        x[4] = x[4].sign() * torch.finfo(dtype).max
        x[5, 17] = float("inf")
        x[6, 18] = float("nan")
        x[7, 19] = float("-inf")
        y = w8a8_forward(x, w, scale)
        _check(y[:5], x[:5], w, scale)
        assert y[5:].isnan().all()


def test_strides_and_alignments(cuda_lib):
    m, n, k = 37, 200, 328
    x, w, scale, g = _data(m, n, k, 3, torch.float16)
    want = w8a8_forward(x, w, scale)
    wide = torch.zeros(m, 3 * k, dtype=torch.float16, device=DEV)
    wide[:, k:2 * k] = x
    odd = torch.zeros(m, k + 1, dtype=torch.float16, device=DEV)
    odd[:, 1:] = x
    flipped = x.t().contiguous().t()
    for other in (wide[:, k:2 * k], odd[:, 1:], flipped):
        assert torch.equal(w8a8_forward(other, w, scale), want)
    assert torch.equal(w8a8_forward(x[:1].expand(4, k), w, scale), want[:1].expand(4, n))
    assert torch.equal(w8a8_forward(wide[3:4, k:2 * k], w, scale), want[3:4])
    w_odd = torch.zeros(n, k + 5, dtype=torch.int8, device=DEV)
    w_odd[:, 2:2 + k] = w
    w_pad = torch.full((n, 352), 99, dtype=torch.int8, device=DEV)          # what lies behind a row is not read
    w_pad[:, :k] = w
    for other in (w_odd[:, 2:2 + k], w_pad[:, :k], w.t().contiguous().t()):
        assert torch.equal(w8a8_forward(x, other, scale), want)
    big = torch.full((m + 2, n + 7), 5.0, dtype=torch.float16, device=DEV)
    for cols in (slice(0, n), slice(3, n + 3)):
        big.fill_(5.0)
        w8a8_forward(x, w, scale, out=big[1:-1, cols])
        assert torch.equal(big[1:-1, cols], want)
        big[1:-1, cols] = 5.0
        assert big.eq(5).all()
    assert w8a8_forward(x[:0], w, scale).shape == (0, n)


def test_layer_takes_the_integer_path_when_asked(cuda_lib):
    torch.manual_seed(0)
    lin = nn.Linear(500, 300)
    for sym, granularity in ((True, "per_channel"), (False, "per_channel"), (True, "per_tensor")):
        cfg = QuantConfig(bits=8, scheme="smoothquant", granularity=granularity, sym=sym)
        layer = QuantizedLinear.from_linear(lin, cfg).cuda()
        layer.quantize_inputs = True
        x = torch.randn(2, 7, 500, device=DEV, dtype=torch.float16)
        eager = layer(x)
        layer.use_kernel = True
        assert torch.equal(layer(x), eager)                                 # what ran before keeps its results
        keys = set(layer.state_dict())
        layer.int8_kernel = True
        y = layer(x)
        assert y.shape == (2, 7, 300) and y.dtype is torch.float16 and set(layer.state_dict()) == keys
        n = layer.out_features
        _check(y.reshape(14, n), x.reshape(14, 500), layer.q_weight, layer.scale.reshape(-1).expand(n), layer.zero.reshape(-1).expand(n), layer.bias)
        # the eager branch in float32 rounds neither the step nor the weights: what is left are sums in float32
        exact = torch.nn.functional.linear(_codes(x.reshape(14, 500))[0].float() * _codes(x.reshape(14, 500))[1], layer.dequantize(), layer.bias)
        assert (y.reshape(14, n).float() - exact).abs().max() <= 2.0 ** -11 * exact.abs().max() + 1e-4
        assert layer(x.float()).dtype is torch.float32
        layer.input_scale = torch.rand(500, device=DEV) + 0.5
        _check(layer(x).reshape(14, n), x.reshape(14, 500), layer.q_weight, layer.scale.reshape(-1).expand(n), layer.zero.reshape(-1).expand(n),
               layer.bias, layer.input_scale)


@pytest.mark.parametrize("m,n,k", [(1, 264, 2048), (16, 264, 6144), (20, 264, 2048), (40, 136, 8192), (300, 520, 256), (513, 1032, 512)])
def test_outputs_stay_inside_their_rows(m, n, k, cuda_lib):
    x, w, scale, _ = _data(m, n, k, m, torch.bfloat16)
    want = w8a8_forward(x, w, scale)
    _check(want, x, w, scale)
    for pad, left in ((8, 0), (16, 8), (6, 2), (7, 1)):              # rows of 16-byte pieces, of 4-byte pieces, of neither
        big = torch.full((m + 2, n + pad), 5.0, dtype=torch.bfloat16, device=DEV)
        w8a8_forward(x, w, scale, out=big[1:-1, left:left + n])
        assert torch.equal(big[1:-1, left:left + n], want)
        big[1:-1, left:left + n] = 5.0
        assert big.eq(5).all()


@pytest.mark.parametrize("granularity", ["per_channel", "per_tensor"])
def test_layer_follows_loaded_states_and_moves(granularity, cuda_lib):
    def layer(seed, sym):
        torch.manual_seed(seed)
        cfg = QuantConfig(bits=8, scheme="smoothquant", granularity=granularity, sym=sym)
        one = QuantizedLinear.from_linear(nn.Linear(500, 300), cfg).cuda()
        one.quantize_inputs, one.use_kernel, one.int8_kernel = True, True, True
        return one

    x = torch.randn(5, 500, device=DEV, dtype=torch.float16)
    first, other = layer(0, True), layer(1, False)
    first(x)
    first.load_state_dict(other.state_dict())                               # a zero-point where there was none
    want = other(x)
    assert torch.equal(first(x), want)
    moved = first.cpu().cuda()
    assert torch.equal(moved(x), want) and moved._buffers["_q_weight_int8"].stride(0) == 512
    assert torch.equal(copy.deepcopy(first)(x), want)
    half = other.half()                                                     # rounds its scales, which the product then has in float32
    n = half.out_features
    _check(half(x), x, half.q_weight, half.scale.float().reshape(-1).expand(n), half.zero.float().reshape(-1).expand(n), half.bias)


def test_layer_refuses_what_the_integers_cannot_do(cuda_lib):
    lin = nn.Linear(256, 128)
    x = torch.randn(3, 256, device=DEV, dtype=torch.float16)
    for cfg, inputs in ((QuantConfig(bits=8, scheme="rtn", granularity="per_group", group_size=64), True),
                        (QuantConfig(bits=8, scheme="rtn", granularity="per_channel"), False)):
        layer = QuantizedLinear.from_linear(lin, cfg).cuda()
        layer.quantize_inputs, layer.use_kernel, layer.int8_kernel = inputs, True, True
        with pytest.raises(ValueError, match="int8_kernel needs"):
            layer(x)


def test_two_streams_and_two_graphs_at_once(cuda_lib):
    work = [(*_data(m, 1000, 4096, m, torch.bfloat16)[:3],) for m in (3, 40)]
    want = [w8a8_forward(*a) for a in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for a in work:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(w8a8_forward(*a))
        graphs.append(g)
    for _ in range(30):
        got = []
        for a, s, g in zip(work, streams, graphs):
            with torch.cuda.stream(s):
                got.append(w8a8_forward(*a))
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(got, want, outs))
