"""CPU tests of the mixture-of-experts and distillation operators: what their C
ABI and Python entry points refuse before any device work, and the shapes of
their Meta kernels."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import bcjr
    return bcjr.load_library()


P = ctypes.c_void_p(4096)  # never dereferenced: the checks fail first


def _said(lib):
    return lib.bcjr_last_error().decode()


@pytest.mark.parametrize("dtype,ld,T,E,k,status,msg", [
    (3, 8, 4, 8, 2, -1, "element type 3"),
    (0, 8, 4, 0, 1, -1, "E=0"),
    (0, 2048, 4, 2048, 2, -2, "E=2048"),
    (0, 8, 4, 8, 0, -1, "k=0"),
    (0, 8, 4, 8, 9, -1, "k=9"),
    (0, 128, 4, 128, 65, -1, "k=65"),
    (0, 8, -1, 8, 2, -1, "T=-1"),
    (0, 8, 1 << 30, 8, 2, -1, "T*k"),
    (0, 4, 4, 8, 2, -1, "row stride 4"),
])
def test_route_refusals(lib, dtype, ld, T, E, k, status, msg):
    assert lib.bcjr_moe_route(P, dtype, ld, None, T, E, k, 0, P, P, P, P, P, None, 0, None) == status
    assert msg in _said(lib)
    assert lib.bcjr_moe_route_backward(P, dtype, ld, None, T, E, k, 0, P, P, P, P, None) == status
    assert msg in _said(lib)


def test_route_gradient_refuses_more_tokens_than_a_launch_holds(lib):
    assert lib.bcjr_moe_route_backward(P, 0, 8, None, 1 << 26, 8, 2, 0, P, P, P, P, None) == -2
    assert "fewer than 2^26" in _said(lib)


@pytest.mark.parametrize("E,M,N,K", [
    (1, (1 << 30) - (1 << 17), 1, 1),    # row tiles of 64, 256 threads each
    (1024, 8, 256, 1 << 20),             # the weights' gradient's tiles, in eights over the dies
])
def test_grouped_refuses_more_than_a_launch_holds(lib, E, M, N, K):
    assert lib.bcjr_grouped_matmul(P, 1, K, M, None, P, K, 1, P, E, M, N, K, 0, P, None) == -2
    assert "more tiles" in _said(lib)
    assert lib.bcjr_grouped_wgrad(P, 1, N, P, K, M, None, P, E, M, N, K, 0, 1, P, None) == -2
    assert "more tiles" in _said(lib)


def test_route_workspace(lib):
    n = ctypes.c_size_t(7)
    assert lib.bcjr_moe_route_workspace(8, 64, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.bcjr_moe_route_workspace(16384, 64, ctypes.byref(n)) == 0 and n.value == 257 * 64 * 4
    assert lib.bcjr_moe_route_workspace(8, 64, None) == -1
    assert lib.bcjr_moe_route(P, 0, 64, None, 16384, 64, 8, 0, P, P, P, P, P, P, 257 * 64 * 4 - 1, None) == -3
    assert "65792 bytes" in _said(lib)
    assert lib.bcjr_moe_route(P, 0, 64, None, 16384, 64, 8, 0, P, P, P, P, P, None, 1 << 20, None) == -1
    assert lib.bcjr_moe_route(None, 0, 64, None, 8, 64, 8, 0, P, P, P, P, P, None, 0, None) == -1
    assert "non-NULL" in _said(lib)


@pytest.mark.parametrize("dtype,E,M,N,K,status,msg", [
    (0, 4, 8, 16, 16, -2, "bfloat16 and float16"),
    (5, 4, 8, 16, 16, -1, "element type 5"),
    (1, 0, 8, 16, 16, -1, "E=0"),
    (1, 1025, 8, 16, 16, -2, "E=1025"),
    (1, 4, -1, 16, 16, -1, "M=-1"),
    (1, 4, 1 << 31, 16, 16, -1, "M=2147483648"),
    (2, 4, 8, 0, 16, -1, "N=0"),
    (2, 4, 8, 16, 1 << 21, -1, "K=2097152"),
    (1, 4, 1 << 30, 16, 16, -2, "more tiles"),
    (1, 1024, 8, 1 << 20, 1 << 20, -2, "more tiles"),
])
def test_grouped_refusals(lib, dtype, E, M, N, K, status, msg):
    assert lib.bcjr_grouped_matmul(P, dtype, K, M, None, P, K, 1, P, E, M, N, K, 0, P, None) == status
    assert msg in _said(lib)
    assert lib.bcjr_grouped_wgrad(P, dtype, N, P, K, M, None, P, E, M, N, K, 0, 1, P, None) == status
    assert msg in _said(lib)


def test_grouped_refuses_rows_and_strides(lib):
    assert lib.bcjr_grouped_matmul(P, 1, 16, 7, None, P, 16, 1, P, 4, 8, 16, 16, 0, P, None) == -1
    assert "a has 7 rows for M=8" in _said(lib)
    assert lib.bcjr_grouped_matmul(P, 1, 15, 8, None, P, 16, 1, P, 4, 8, 16, 16, 0, P, None) == -1
    assert "row stride 15" in _said(lib)
    assert lib.bcjr_grouped_matmul(P, 1, 16, 8, None, P, 15, 1, P, 4, 8, 16, 16, 0, P, None) == -1
    assert "row stride 15 of b" in _said(lib)
    assert lib.bcjr_grouped_matmul(P, 1, 16, 8, None, None, 16, 1, P, 4, 8, 16, 16, 0, P, None) == -1
    assert "non-NULL" in _said(lib)
    assert lib.bcjr_grouped_matmul(None, 1, 16, 0, None, None, 16, 1, None, 4, 0, 16, 16, 0, None, None) == 0
    assert lib.bcjr_grouped_wgrad(P, 1, 16, P, 15, 8, None, P, 4, 8, 16, 16, 0, 0, P, None) == -1
    assert lib.bcjr_grouped_wgrad(P, 1, 15, P, 16, 8, None, P, 4, 8, 16, 16, 0, 0, P, None) == -1
    assert lib.bcjr_grouped_wgrad(P, 1, 16, P, 16, 7, None, P, 4, 8, 16, 16, 0, 0, P, None) == -1
    # rows said to be padded that have no room for it
    assert lib.bcjr_grouped_matmul(P, 1, 15, 8, None, P, 16, 1, P, 4, 8, 16, 15, 1, P, None) == -1
    assert lib.bcjr_grouped_matmul(P, 1, 16, 8, None, P, 15, 1, P, 4, 8, 16, 15, 1, P, None) == -1
    assert "in eights" in _said(lib)
    assert lib.bcjr_grouped_wgrad(P, 1, 15, P, 16, 8, None, P, 4, 8, 15, 16, 1, 0, P, None) == -1


def test_float32_weights_refusals(lib):
    Q = ctypes.c_void_p(1 << 20)
    assert lib.bcjr_grouped_matmul_f32w(P, 0, 16, 8, None, Q, 16, P, 4, 8, 16, 16, P, None, None) == -2
    assert lib.bcjr_grouped_matmul_f32w(P, 1, 16, 7, None, Q, 16, P, 4, 8, 16, 16, P, None, None) == -1
    for lda, ldb, K in [(16, 16, 12), (12, 16, 8), (16, 17, 16)]:
        assert lib.bcjr_grouped_matmul_f32w(P, 1, lda, 8, None, Q, ldb, P, 4, 8, 16, K, P, None, None) == -2
        assert "16-byte chunks" in _said(lib)
    assert lib.bcjr_grouped_matmul_f32w(P, 1, 16, 8, None, ctypes.c_void_p(4100), 16, P, 4, 8, 16, 16, P, None, None) == -2
    assert lib.bcjr_grouped_matmul_f32w(P, 1, 16, 8, None, Q, 16, P, 4, 8, 16, 16, P, ctypes.c_void_p(4100), None) == -2
    assert lib.bcjr_grouped_matmul_f32w(P, 1, 16, 8, None, Q, 15, P, 4, 8, 16, 16, P, None, None) == -1
    assert lib.bcjr_grouped_matmul_f32w(None, 1, 16, 0, None, None, 16, None, 4, 0, 16, 16, None, None, None) == 0


def test_pad_rows_refusals(lib):
    assert lib.bcjr_pad_rows(P, 0, 16, 4, 16, 0, P, 16, None) == -2
    assert lib.bcjr_pad_rows(P, 2, 16, 4, 16, 1, P, 16, None) == -2
    assert lib.bcjr_pad_rows(P, 0, 16, -1, 16, 1, P, 16, None) == -1
    assert lib.bcjr_pad_rows(P, 0, 15, 4, 16, 1, P, 16, None) == -1
    assert lib.bcjr_pad_rows(P, 0, 16, 4, 16, 1, P, 20, None) == -1
    assert lib.bcjr_pad_rows(P, 0, 16, 4, 16, 1, P, 8, None) == -1
    assert lib.bcjr_pad_rows(P, 0, 16, 4, 16, 1, ctypes.c_void_p(4104), 16, None) == -1
    assert lib.bcjr_pad_rows(None, 0, 16, 4, 16, 1, P, 16, None) == -1
    assert lib.bcjr_pad_rows(None, 0, 16, 0, 16, 1, None, 16, None) == 0


def test_combine_refusals(lib):
    assert lib.bcjr_moe_combine(P, 9, 16, P, P, 4, 2, 8, 16, P, None) == -1
    assert lib.bcjr_moe_combine(P, 0, 16, P, P, 4, 0, 8, 16, P, None) == -1
    assert "k=0" in _said(lib)
    assert lib.bcjr_moe_combine(P, 0, 15, P, P, 4, 2, 8, 16, P, None) == -1
    assert lib.bcjr_moe_combine(P, 0, 16, P, None, 4, 2, 8, 16, P, None) == -1
    assert lib.bcjr_moe_combine(None, 0, 16, None, None, 0, 2, 0, 16, None, None) == 0
    assert lib.bcjr_moe_combine_backward(P, 0, 16, P, P, P, P, 16, 4, 2, 9, 16, P, P, None) == -1
    assert "M=9 rows for T*k=8" in _said(lib)
    assert lib.bcjr_moe_combine_backward(P, 0, 16, P, P, P, P, 15, 4, 2, 8, 16, P, P, None) == -1


@pytest.mark.parametrize("dtype,ld,tau,T,V,K,status,msg", [
    (7, 32, 1.0, 4, 32, 4, -1, "element type 7"),
    (0, 32, 0.0, 4, 32, 4, -1, "temperature 0"),
    (0, 32, -1.0, 4, 32, 4, -1, "temperature -1"),
    (0, 32, float("nan"), 4, 32, 4, -1, "temperature"),
    (0, 32, float("inf"), 4, 32, 4, -1, "temperature"),
    (0, 32, 1e-45, 4, 32, 4, -1, "temperature"),
    (0, 32, 1.0, -1, 32, 4, -1, "T=-1"),
    (0, 32, 1.0, 1 << 22, 32, 4, -2, "2^22"),
    (0, 32, 1.0, 4, 0, 0, -1, "V=0"),
    (0, 1 << 21, 1.0, 4, 1 << 21, 4, -2, "V=2097152"),
    (0, 32, 1.0, 4, 32, 33, -1, "K=33"),
    (0, 31, 1.0, 4, 32, 4, -1, "row stride 31"),
])
def test_distill_refusals(lib, dtype, ld, tau, T, V, K, status, msg):
    assert lib.bcjr_topk_distill(P, dtype, ld, P, P, None, tau, T, V, K, P, None, None) == status
    assert msg in _said(lib)
    assert lib.bcjr_topk_distill_backward(P, dtype, ld, P, P, tau, T, V, K, P, P, P, None) == status
    assert lib.bcjr_topk_distill_both(P, dtype, ld, P, P, None, tau, T, V, K, P, P, P, None) == status


def test_distill_null_and_alignment(lib):
    assert lib.bcjr_topk_distill(P, 0, 32, None, P, None, 1.0, 4, 32, 4, P, None, None) == -1
    assert "non-NULL" in _said(lib)
    assert lib.bcjr_topk_distill(P, 0, 32, P, P, None, 1.0, 4, 32, 4, P, ctypes.c_void_p(4100), None) == -1
    assert "16-byte" in _said(lib)
    assert lib.bcjr_topk_distill(None, 0, 32, None, None, None, 1.0, 0, 32, 4, None, None, None) == 0


def test_python_surface_refuses_before_the_device():
    import bcjr
    x = torch.zeros(4, 8)
    with pytest.raises(AssertionError, match="GPU"):
        bcjr.moe_route(x, 2)
    with pytest.raises(AssertionError, match="GPU"):
        bcjr.grouped_matmul(x, torch.zeros(2, 8, 8), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(AssertionError, match="GPU"):
        bcjr.moe_combine(x, torch.ones(2, 2), torch.zeros(4, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(AssertionError, match="GPU"):
        bcjr.topk_distill_loss(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32))


def test_meta_shapes():
    import bcjr
    ops = bcjr.moe._ops
    l = torch.empty(10, 6, device="meta", dtype=torch.bfloat16)
    w, e, o, r, s = ops.moe_route(l, None, 3, False)
    assert w.shape == (10, 3) and w.dtype == torch.float32 and e.dtype == o.dtype == r.dtype == s.dtype == torch.int32
    assert o.shape == (7,) and r.shape == (30,) and s.shape == e.shape == (10, 3)
    x = torch.empty(10, 16, device="meta", dtype=torch.bfloat16, requires_grad=True)
    W = torch.empty(6, 24, 16, device="meta", requires_grad=True)
    y = ops.grouped_matmul(x, W, o, r, s)
    assert y.shape == (30, 24) and y.dtype == torch.bfloat16
    assert ops.pad_rows(torch.empty(3, 5, device="meta"), l).stride() == (8, 1)
    gx, gw = torch.autograd.grad(y, (x, W), torch.empty_like(y))
    assert gx.shape == x.shape and gx.dtype == x.dtype and gw.shape == W.shape and gw.dtype == torch.float32
    wr = torch.empty(10, 3, device="meta", requires_grad=True)
    out = ops.moe_combine(y, wr, r, s)
    assert out.shape == (10, 24)
    gy, gwr = torch.autograd.grad(out, (y, wr), torch.empty_like(out))
    assert gy.shape == y.shape and gwr.shape == wr.shape
    lg = torch.empty(5, 100, device="meta", dtype=torch.float16, requires_grad=True)
    v, i = torch.empty(5, 4, device="meta"), torch.empty(5, 4, device="meta", dtype=torch.int32)
    loss = ops.topk_distill_loss(lg, v, i, None, 2.0)
    assert loss.shape == (5,) and loss.dtype == torch.float32
    (g,) = torch.autograd.grad(loss, lg, torch.empty_like(loss))
    assert g.shape == lg.shape and g.dtype == torch.float16
