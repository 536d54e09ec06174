"""Refusals of the 8-bit operators, checked without a GPU: the Python faces and the C entries (whose checks come before any launch)."""

import ctypes
import re

import pytest
import torch

import pare_b200
from pare_b200 import PagedKVCache, PagedKVConfig
from pare_b200 import paged_cache as pc
from pare_b200.kernels import _lib, w8a8_forward
from pare_b200.kernels.matmul_int8 import aligned_rows


def _fake(n=4096):
    """An aligned host buffer: an address that is not NULL.  Nothing reads it: every call below is refused first."""
    buf = (ctypes.c_char * (n + 64))()
    return buf, (ctypes.addressof(buf) + 63) // 64 * 64


def test_public_names():
    assert pare_b200.PagedKVCache is PagedKVCache and "PagedKVConfig" in pare_b200.__all__
    from pare_b200 import kernels
    assert "w8a8_forward" in kernels.__all__


def test_cuda_tensors_only():
    x = torch.zeros(2, 16, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        w8a8_forward(x, torch.zeros(3, 16, dtype=torch.int8), torch.ones(3))
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedKVCache(1, 2, 128, PagedKVConfig(10), device="cpu")
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        pc.plan_blocks(one, one, torch.zeros(1, 4, dtype=torch.int32), one, one, 16, 1)


@pytest.mark.parametrize("config,heads,dim,dtype", [(PagedKVConfig(10, 24), 2, 128, torch.float16), (PagedKVConfig(10, 128), 2, 128, torch.float16),
                                                    (PagedKVConfig(10), 2, 96, torch.float16), (PagedKVConfig(10), 2, 128, torch.float32),
                                                    (PagedKVConfig(0), 2, 128, torch.float16), (PagedKVConfig(10, max_requests=4097), 2, 128, torch.float16),
                                                    (PagedKVConfig(10, max_requests=0), 2, 128, torch.float16), (PagedKVConfig(10, max_seq_len=0), 2, 128, torch.float16),
                                                    (PagedKVConfig(10), 0, 128, torch.float16)])
def test_cache_configurations_refused(config, heads, dim, dtype):
    with pytest.raises(ValueError, match="PagedKVCache"):
        PagedKVCache(1, heads, dim, config, dtype=dtype, device="cuda")


def test_step_layout():
    L = _lib.lib()
    for bad in ((0, 1, 16), (4097, 1, 16), (1, -1, 16), (1, (1 << 22) + 1, 16), (1, 1, 8), (1, 1, 24), (1, 1, 128)):
        assert L.pare_paged_step_bytes(*bad) == 0 and L.pare_paged_step_offset(0, *bad) == -1
    assert L.pare_paged_step_offset(7, 1, 1, 16) == -1 and L.pare_paged_step_offset(-1, 1, 1, 16) == -1
    for sizes in ((1, 0, 16), (3, 7, 32), (4096, 5000, 64)):
        at = [L.pare_paged_step_offset(f, *sizes) for f in range(7)]
        assert all(a % 16 == 0 for a in at) and max(at) < L.pare_paged_step_bytes(*sizes)
        size = {0: 16, 1: 4 * (sizes[0] + 1), 2: 4 * (sizes[0] + 1), 3: 8 * (sizes[0] + 1), 4: 8 * sizes[1], 5: 4 * sizes[1], 6: 4 * sizes[1]}
        spans = sorted((a, a + size[f]) for f, a in enumerate(at))
        assert all(e <= b for (_, e), (b, _) in zip(spans, spans[1:]))


def test_c_entries_refuse():
    L = _lib.lib()
    buf, p = _fake()
    OK, SHAPE, DTYPE, ALIGN, SPACE, UNSUPPORTED = 0, 1, 2, 3, 4, 5

    def plan(R=2, ld=4, width=4, capacity=8, bs=16, T=2, size=1 << 20, step=p):
        return L.pare_paged_plan(p, p, R, p, ld, width, p, capacity, p, bs, T, step, size, None)
    assert plan(R=0) == plan(R=4097) == plan(T=-1) == plan(width=0) == plan(ld=3) == plan(capacity=-1) == plan(width=1 << 28, ld=1 << 28) == SHAPE
    assert plan(bs=8) == plan(bs=128) == UNSUPPORTED and plan(size=64) == SPACE and plan(step=p + 4) == ALIGN
    assert L.pare_paged_plan(None, p, 2, p, 4, 4, p, 8, p, 16, 2, p, 1 << 20, None) == SHAPE

    def release(R=2, ld=4, bs=16, mask=p):
        return L.pare_paged_release(mask, p, R, p, ld, 4, p, 8, p, bs, None)
    assert release(R=0) == release(ld=3) == release(mask=None) == SHAPE and release(bs=17) == UNSUPPORTED

    def layer(dtype=0, NB=4, H=2, D=128, bs=16, R=2, tail=p, codes=p):
        return _lib.PagedLayerStruct(codes, p, p, p, tail, p, NB, R, H, bs, D, dtype)

    def tables(T=2, ld=4, width=4, bs=16, R=2, step=p):
        return _lib.PagedTablesStruct(step, p, ld, width, R, T, bs)

    calls = (lambda l, t: L.pare_paged_append(p, p, 256, 128, 256, 128, ctypes.addressof(l), ctypes.addressof(t), None),
             lambda l, t: L.pare_paged_dense(ctypes.addressof(l), ctypes.addressof(t), p, p, 3, None),
             lambda l, t: L.pare_paged_attn(p, 1024, 128, ctypes.addressof(l), ctypes.addressof(t), 8, p, 1024, 128, 0.1, p, 1 << 26, None))
    for call in calls:
        for l, t in ((layer(NB=0), tables()), (layer(H=0), tables()), (layer(H=70000), tables()), (layer(tail=None), tables()), (layer(), tables(T=-1)),
                     (layer(), tables(ld=3)), (layer(), tables(width=0)), (layer(), tables(R=3)), (layer(), tables(bs=32)), (layer(), tables(step=None)),
                     (layer(R=0), tables(R=0))):
            assert call(l, t) == SHAPE
        assert call(layer(dtype=2), tables()) == DTYPE
        assert call(layer(D=96), tables()) == call(layer(bs=8), tables(bs=8)) == call(layer(bs=128), tables(bs=128)) == UNSUPPORTED
        assert call(layer(codes=p + 8), tables()) == call(layer(tail=p + 2), tables()) == call(layer(), tables(step=p + 4)) == ALIGN
    ok, some = layer(), tables()
    lp, tp, none = ctypes.addressof(ok), ctypes.addressof(some), tables(T=0)

    def append(k=p, st=256):
        return L.pare_paged_append(k, p, st, 128, st, 128, lp, tp, None)
    assert append(k=None) == SHAPE and append(k=p + 2) == append(st=130) == ALIGN
    assert L.pare_paged_append(p, p, 256, 128, 256, 128, None, tp, None) == L.pare_paged_append(p, p, 256, 128, 256, 128, lp, None, None) == SHAPE
    assert L.pare_paged_append(None, None, 256, 128, 256, 128, lp, ctypes.addressof(none), None) == OK

    def dense(total=3, out=p):
        return L.pare_paged_dense(lp, tp, out, p, total, None)
    assert dense(total=-1) == dense(out=None) == SHAPE and dense(out=p + 2) == ALIGN and dense(total=0) == OK

    need = 1 << 26

    many = tables(T=4097)

    def attend(q=p, t=tp, Hq=8, ws=p, size=need, sh=128):
        return L.pare_paged_attn(q, 1024, sh, lp, t, Hq, p, 1024, 128, 0.1, ws, size, None)
    assert attend(q=None) == attend(Hq=7) == attend(Hq=0) == SHAPE and attend(t=ctypes.addressof(many)) == UNSUPPORTED
    assert attend(size=16) == attend(ws=None) == SPACE and attend(q=p + 4) == attend(sh=130) == attend(ws=p + 8) == ALIGN
    assert attend(t=ctypes.addressof(none)) == OK
    wide = tables(T=256, ld=1 << 23, width=1 << 23)          # more units than 32 bits count
    assert attend(t=ctypes.addressof(wide)) == UNSUPPORTED
    assert L.pare_paged_attn_workspace_bytes(96) == 0

    def linear(M=2, N=4, K=32, ldw=32, ldx=32, ldy=4, dtype=0, x=p, w=p, ws=p, size=need):
        return L.pare_w8a8_forward(x, dtype, ldx, w, ldw, p, None, None, None, p, ldy, M, N, K, ws, size, None)
    assert linear(M=0) == linear(N=0) == linear(K=0) == linear(ldw=16) == linear(ldx=31) == linear(ldy=3) == linear(x=None) == SHAPE
    assert linear(dtype=2) == DTYPE and linear(K=65537, ldx=70000, ldw=70000) == UNSUPPORTED
    assert linear(w=p + 8) == linear(ldw=40) == linear(ws=p + 4) == linear(x=p + 2) == linear(ldx=36) == ALIGN
    assert linear(M=20, size=8) == linear(M=20, ws=None) == SPACE
    assert L.pare_w8a8_workspace_bytes(0, 1, 1) == L.pare_w8a8_workspace_bytes(1, 1, 65537) == 0
    del buf


def test_workspace_covers_the_codes():
    L = _lib.lib()
    for m, n, k in ((1, 1, 1), (3, 5, 4097), (17, 4096, 4096), (333, 3584, 18944), (5000, 100, 65536)):
        assert L.pare_w8a8_workspace_bytes(m, n, k) >= m * k + 8 * m


def test_a_few_rows_need_no_workspace():
    L = _lib.lib()
    assert all(L.pare_w8a8_workspace_bytes(m, n, k) == 0 for m in (1, 4) for n, k in ((1, 8), (4096, 4096), (28672, 4096)))
    assert L.pare_w8a8_workspace_bytes(1, 60000, 65536) > 0      # too long a row to keep its codes beside the weights


def test_aligned_rows():
    w = torch.arange(5 * 32, dtype=torch.int32).to(torch.int8).view(5, 32)
    assert aligned_rows(w).data_ptr() == w.data_ptr()
    for cols in (slice(0, 30), slice(3, 32)):
        a = aligned_rows(w[:, cols])
        assert torch.equal(a, w[:, cols]) and a.stride(0) % 16 == 0


def test_every_paged_entry_is_documented():
    header = (_lib.LIB_PATH.parent.parent.parent / "include" / "pare_b200.h").read_text()
    for name in (n for n in _lib.SIGNATURES if n.startswith(("pare_paged", "pare_w8a8"))):
        assert re.search(rf"\b{name}\s*\(", header)
