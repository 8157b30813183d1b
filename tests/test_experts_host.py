"""Host-side checks of the expert operators: they answer without touching a GPU."""
import ctypes
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))
import prism_b200 as pb  # noqa: E402
from prism_b200 import _lib  # noqa: E402

P = ctypes.c_void_p(1 << 20)      # never dereferenced: every call below is refused or empty
ODD = ctypes.c_void_p((1 << 20) + 2)


@pytest.fixture
def lib():
    lib = _lib.load()
    yield lib
    lib.prism_b200_clear_error()


def test_route_workspace(lib):
    size = lambda t, e, k: pb.route_workspace_size(t, e, k)  # noqa: E731
    assert size(0, 8, 2) == size(1, 1024, 32) == size(64, 64, 8) == 0
    assert size(65, 64, 8) == 3 * 64 * 4
    assert size(1 << 20, 64, 8) == 148 * 64 * 4
    for bad in ((-1, 8, 2), (1, 0, 1), (1, 1025, 2), (1, 8, 9), (1, 64, 33), (1 << 29, 64, 4)):
        with pytest.raises(pb.PrismB200Error):
            size(*bad)
    assert lib.prism_b200_route_workspace_size(1, 8, 2, None) == 1


def test_route_refusals(lib):
    assert lib.prism_b200_route_topk(4, 8, 2, 0, None, 8, 1, P, P, P, P, P, None, None) == 1
    assert lib.prism_b200_route_topk(4, 8, 2, 3, P, 8, 1, P, P, P, P, P, None, None) == 1       # unknown type
    assert lib.prism_b200_route_topk(4, 8, 2, 0, P, 7, 1, P, P, P, P, P, None, None) == 1       # rows overlap
    assert lib.prism_b200_route_topk(500, 8, 2, 0, P, 8, 1, P, P, P, P, P, None, None) == 1     # no workspace
    assert lib.prism_b200_route_topk_grad(4, 8, 2, 0, P, 8, 1, P, P, P, None, None) == 1
    assert lib.prism_b200_route_topk_grad(0, 8, 2, 0, None, 8, 1, None, None, None, None, None) == 0
    assert lib.prism_b200_route_gather(1, 4, 2, 64, P, 64, P, 8, P, 64, None) == 1               # x and out overlap
    assert "overlap" in _lib.last_error()[1]
    assert lib.prism_b200_route_gather(1, 4, 0, 64, P, 64, P, 8, P, 64, None) == 2
    assert lib.prism_b200_route_gather(1, 4, 2, 0, None, 0, None, 8, None, 0, None) == 0
    assert lib.prism_b200_route_combine(1, 0, 2, 64, None, 64, 0, None, None, None, 64, None) == 0
    assert lib.prism_b200_route_combine(1, 4, 33, 64, P, 64, 8, P, None, P, 64, None) == 2
    assert lib.prism_b200_route_combine_grad(1, 4, 2, 64, P, 64, P, 64, 8, P, P, P, 64, P, None) == 1
    big = (1 << 30) + 8
    assert lib.prism_b200_route_gather(1, 4, 2, big, P, big, P, 8, P, big, None) == 6
    assert lib.prism_b200_route_combine(1, 4, 2, big, P, big, 8, P, None, P, big, None) == 6
    assert lib.prism_b200_route_combine_grad(1, 4, 2, big, P, big, P, big, 8, P, P, P, big, P, None) == 6
    assert lib.prism_b200_route_combine_grad(1, 1 << 29, 4, 64, P, 64, P, 64, 8, P, P, P, 64, P, None) == 6


def test_grouped_refusals(lib):
    f, d, w = lib.prism_b200_grouped_gemm_bf16, lib.prism_b200_grouped_gemm_bf16_dgrad, lib.prism_b200_grouped_gemm_bf16_wgrad
    assert f(0, 8, 64, 64, None, 64, None, None, None, 64, None) == 0
    assert f(2, 0, 64, 64, None, 64, None, None, None, 64, None) == 0
    assert f(2, -1, 64, 64, P, 64, P, P, P, 64, None) == 1
    assert f(2, 8, 60, 64, P, 64, P, P, P, 64, None) == 2
    assert f(2, 8, 64, 0, P, 0, P, P, P, 64, None) == 2
    assert f(1025, 8, 64, 64, P, 64, P, P, P, 64, None) == 2
    assert f(2, 8, 64, 64, P, 64, P, None, P, 64, None) == 1
    assert f(2, 8, 64, 64, ODD, 64, P, P, P, 64, None) == 3
    assert f(2, 8, 64, 64, P, 68, P, P, P, 64, None) == 3
    assert f(2, 8, 64, 64, P, 56, P, P, P, 64, None) == 1
    assert f(2, 8, 64, 64, P, 64, P, P, P, 64, None) == 1 and "overlap" in _lib.last_error()[1]
    assert f(1024, 1 << 30, 1 << 20, 64, P, 64, P, P, P, 1 << 20, None) == 6
    big = (1 << 30) + 8
    assert f(1, 1, 8, big, P, big, P, P, P, 8, None) == 6 and d(1, 1, big, 8, P, big, P, P, P, 8, None) == 6
    assert w(1, 1, 8, big, P, 8, P, big, P, 1, P, None) == 6
    assert d(2, 8, 0, 64, P, 0, P, P, P, 64, None) == 2
    assert w(2, 8, 64, 64, P, 64, P, 64, P, 2, P, None) == 1                                      # fp16 result
    assert w(2, 8, 64, 64, P, 64, P, 64, P, 0, P, None) == 1 and "overlap" in _lib.last_error()[1]


def test_w4_refusals(lib):
    g = lib.prism_b200_gemv_w4
    ok = dict(dtype=1, rows=2, experts=1, n=64, k=256, group=64, x=P, ldx=256, q=P, scales=P, zeros=None, offsets=None, out=P, ldo=64, stream=None)
    call = lambda **kw: g(*{**ok, **kw}.values())  # noqa: E731
    assert call(rows=0) == 0 and call(n=0) == 0 and call(experts=0) == 0
    assert call(dtype=0) == 1 and call(rows=-1) == 1 and call(experts=2) == 1 and call(x=None) == 1 and call(ldx=128) == 1
    assert call(group=16) == 2 and call(k=200) == 2 and call(k=0) == 2 and call(experts=1025, offsets=P) == 2
    assert call(x=ODD) == 3 and call(ldx=260) == 3 and call(q=ODD) == 3
    assert call() == 1 and "overlap" in _lib.last_error()[1]
    big = (1 << 30) + 128
    assert call(k=big, ldx=big) == 6 and call(n=big, ldo=big) == 6 and call(rows=big) == 6
    assert call(ldo=63) == 1 and call(scales=ctypes.c_void_p((1 << 20) + 1)) == 3


def test_python_layer_has_no_cpu_path():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    pos, off = torch.zeros((4, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: pb.route_topk(x, 2), lambda: pb.route_gather(x, pos), lambda: pb.route_combine(x, pos),
                 lambda: pb.grouped_gemm_bf16(x, torch.zeros((2, 64, 64), dtype=torch.bfloat16), off),
                 lambda: pb.grouped_gemm_bf16_wgrad(x, x, off),
                 lambda: pb.gemv_w4(x, torch.zeros((8, 32), dtype=torch.uint8), torch.zeros((8, 1), dtype=torch.bfloat16))):
        with pytest.raises(TypeError):
            call()


def test_public_names():
    for name in ("route_topk", "route_topk_grad", "route_gather", "route_combine", "route_combine_grad", "grouped_gemm_bf16",
                 "grouped_gemm_bf16_dgrad", "grouped_gemm_bf16_wgrad", "gemv_w4", "Routing"):
        assert name in pb.__all__ and hasattr(pb, name)
