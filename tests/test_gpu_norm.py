"""Layer norm, counter-based dropout and both joined against their definitions in 64 bits (norm_reference.py), on the GPU."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

import norm_reference as R
from artifact_b200 import _native, graphs, norm, search
from artifact_b200.models import ROF_GCN, ROF_GIN, ROF_inputInfo, SumAggregate
from artifact_b200.plan import AggregationPlan, empty_padded
from conftest import load_golden

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = {F32: 0, BF16: 1, F16: 2}                     # enum rof_dtype


def randn(*shape, seed=0, dtype=F32, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).to(DEV)


def calm_gradient(dy, x, w, b, eps):
    """no gradient comes in next to the ReLU's border, where a rounding decides which one-sided gradient holds"""
    z = R.z_of(x, w, b, eps)
    return dy.masked_fill(torch.from_numpy(np.abs(z) < 1e-3).to(DEV), 0.0)


def check_norm(x, w, b, dy, eps=1e-5, relu=False, p=0.0, what="", **drop):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = norm.layer_norm(*leaves, eps, relu=relu, p=p, **drop)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    given = [t for t in leaves if t is not None]
    grads = dict(zip([k for k, t in zip(("dx", "dw", "db"), leaves) if t is not None],
                     torch.autograd.grad(y, given, dy)))
    with torch.no_grad():
        assert torch.equal(norm.layer_norm(x, w, b, eps, relu=relu, p=p, **drop), y)
    d = x.size(-1)
    want = R.norm_reference(x.reshape(-1, d), w, b, eps, relu, p, dy=dy.reshape(-1, d), **drop)
    R.assert_within(y.reshape(-1, d), want["y"], what + " y")
    for k, g in grads.items():
        assert g.shape == dict(dx=x, dw=w, db=b)[k].shape and g.dtype == dict(dx=x, dw=w, db=b)[k].dtype
        R.assert_within(g, want[k], what + " " + k)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, dim", [(1, 1), (3, 2), (5, 3), (1, 8), (33, 16), (2, 31), (129, 47), (7, 64), (65, 100), (300, 128),
                                       (17, 200), (9, 257), (40, 602), (3, 1000), (5, 1024), (4, 1031), (6, 2048), (3, 2050),
                                       (2, 4096), (2, 5001), (3, 8192), (1, 20000), (2, 33000)])
def test_layer_norm(dtype, rows, dim):
    x = randn(rows, dim, seed=1, scale=1.5, shift=0.4, dtype=dtype)
    dy = randn(rows, dim, seed=2, dtype=dtype)
    w, b = randn(dim, seed=3, scale=0.3, shift=1.0), randn(dim, seed=4, scale=0.3)
    check_norm(x, w, b, dy, what="affine")
    check_norm(x, w, b, calm_gradient(dy, x, w, b, 1e-5), relu=True, p=0.3, seed=2 ** 63 + 11, step=5, what="hidden")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, dim", [(3000, 16), (5000, 47), (2708, 64), (1500, 300), (1111, 602), (600, 2048)])
def test_layer_norm_many_rows(dtype, rows, dim):
    x, dy = randn(rows, dim, seed=1, scale=2.0, dtype=dtype), randn(rows, dim, seed=2, dtype=dtype)
    w, b = randn(dim, seed=3, shift=1.0), randn(dim, seed=4)
    check_norm(x, w, b, dy, what="norm")
    check_norm(x, w, b, calm_gradient(dy, x, w, b, 1e-5), relu=True, p=0.5, seed=3, step=2 ** 40 + 1, row_offset=12345, what="hidden")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [4, 12, 15, 17, 20, 28, 32, 33, 40, 48, 49, 56, 63, 65, 79, 80, 95, 96, 97, 127, 129, 160, 161, 191, 192, 193, 255, 256,
                                 259, 320, 383, 385, 509, 511, 512, 513, 640, 641, 644, 767, 768, 1023, 1025, 1028, 2047, 2049, 4095, 4097, 8191,
                                 8193, 8200])
def test_widths_next_to_every_border(dtype, dim):
    """the kernels change shape with the width: seven rows each, in both passes, with and without what is fused"""
    x, dy = randn(7, dim, seed=1, scale=1.5, dtype=dtype), randn(7, dim, seed=2, dtype=dtype)
    w, b = randn(dim, seed=3, scale=0.3, shift=1.0), randn(dim, seed=4, scale=0.3)
    check_norm(x, w, b, dy, what="norm")
    check_norm(x, w, b, calm_gradient(dy, x, w, b, 1e-5), relu=True, p=0.3, seed=12, step=5, what="hidden")
    check_dropout(x, b, dy, relu=True, p=0.3, seed=12, what="dropout relu")
    check_dropout(x, b, dy, p=0.3, seed=12, row_offset=1, what="dropout")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, dim", [(100003, 16), (120001, 47), (60000, 50), (30011, 130), (20003, 301), (9001, 501), (12001, 256), (7001, 602),
                                       (4003, 1024), (2503, 2048), (1203, 4097)])
def test_many_rows_per_block(dtype, rows, dim):
    """more rows than one round of the grid takes: rings and tiles go round, the column sums run over many rows"""
    x, dy = randn(rows, dim, seed=1, dtype=dtype), randn(rows, dim, seed=2, dtype=dtype)
    w, b = randn(dim, seed=3, scale=0.3, shift=1.0), randn(dim, seed=4, scale=0.3)
    check_norm(x, w, b, calm_gradient(dy, x, w, b, 1e-5), relu=True, p=0.3, seed=5, what="hidden")
    check_norm(x, w, b, dy, what="norm")
    check_dropout(x, b, dy, p=0.3, seed=5, what="dropout")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, dim", [(300, 47), (9001, 50), (77, 130), (64, 301), (700, 602), (33, 1001), (20, 2050), (12, 5001), (9, 9001)])
def test_padded_rows(dtype, rows, dim):
    """rows padded to whole vectors, as the framework's own buffers have them, beside contiguous ones"""
    per = 16 // torch.empty(0, dtype=dtype).element_size()

    def padded(t, more=0):
        buf = torch.full((rows, -(-dim // per) * per + more), float("nan"), dtype=dtype, device=DEV)
        buf[:, :dim] = t
        return buf[:, :dim]

    x, dy = randn(rows, dim, seed=1, dtype=dtype), randn(rows, dim, seed=2, dtype=dtype)
    w, b = randn(dim, seed=3, scale=0.3, shift=1.0), randn(dim, seed=4, scale=0.3)
    hidden = dict(relu=True, p=0.3, seed=5, row_offset=2)
    calm = calm_gradient(dy.clone(), x, w, b, 1e-5)
    for xs, gs in ((padded(x), padded(dy)), (padded(x), dy), (x, padded(dy)), (padded(x, 3), padded(dy, 8)), (padded(x, per), padded(dy))):
        check_norm(xs, w, b, gs, what="norm")
        check_norm(xs, w, b, padded(calm) if gs is not dy else calm, what="hidden", **hidden)
        check_dropout(xs, b, gs, what="dropout", **hidden)
        check_dropout(xs, None, gs, what="dropout without bias", p=0.3, seed=5, row_offset=3)


def _c_norm(x, w, b, dy, y, dx, relu, drop):
    """both passes through the C ABI into given outputs -> (dw, db)"""
    lib, d = _native.cuda(), DTYPES[x.dtype]
    rows, dim = x.shape
    stats = torch.full((rows, 2), float("nan"), device=DEV)
    dw, db = torch.full((dim,), float("nan"), device=DEV), torch.full((dim,), float("nan"), device=DEV)
    n = lib.rof_layer_norm_workspace_bytes(rows, dim)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=DEV)          # whatever was there before
    s = torch.cuda.current_stream().cuda_stream
    _native.check(lib.rof_layer_norm_forward(d, x.data_ptr(), x.stride(0), rows, dim, 0, w.data_ptr(), b.data_ptr(), 1e-5, relu, drop,
                                             y.data_ptr(), y.stride(0), stats.data_ptr(), s))
    _native.check(lib.rof_layer_norm_backward(d, dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), rows, dim, 0, w.data_ptr(),
                                              b.data_ptr(), stats.data_ptr(), relu, drop, dx.data_ptr(), dx.stride(0), dw.data_ptr(),
                                              db.data_ptr(), ws.data_ptr(), n, s))
    return dw, db


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [8, 47, 64, 130, 301, 602, 1001])
def test_outputs_with_strides_through_the_c_abi(dtype, dim):
    """every mix of how the four matrices lie; what lies between and behind the rows stays as it was"""
    rows, w, b = 37, randn(dim, seed=3, scale=0.3, shift=1.0), randn(dim, seed=4, scale=0.3)
    x0, dy0 = randn(rows, dim, seed=1, dtype=dtype), randn(rows, dim, seed=2, dtype=dtype)
    calm_gradient(dy0, x0, w, b, 1e-5)

    def laid(t, lead, ld):
        buf = torch.full((lead + rows * ld + 8,), 7.0, dtype=dtype, device=DEV)
        view = buf.as_strided((rows, dim), (ld, 1), lead)
        if t is not None:
            view.copy_(t)
        return buf, view

    up = -(-dim // 8) * 8
    want = R.norm_reference(x0, w, b, relu=True, p=0.3, seed=9, step=3, row_offset=4, dy=dy0)
    plain = R.dropout_reference(x0, b, True, 0.3, 9, 3, 4, dy=dy0)
    lib, s = _native.cuda(), torch.cuda.current_stream().cuda_stream
    drop = _native.Dropout(0.3, 9, 3, None, 4)
    layouts = ((0, up), (0, dim), (1, dim + 1), (8, up + 8), (3, up))
    for i, lx in enumerate(layouts):
        for ly in (layouts[i], layouts[(i + 1) % 5], layouts[(i + 3) % 5]):
            x, dy = laid(x0, *lx)[1], laid(dy0, *ly)[1]
            (ybuf, y), (gbuf, dx) = laid(None, *ly), laid(None, *lx)
            dw, db = _c_norm(x, w, b, dy, y, dx, 1, drop)
            for got, n in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
                R.assert_within(got, want[n], f"{lx} {ly} {n}")
            for buf, view in ((ybuf, y), (gbuf, dx)):
                view.fill_(7.0)
                assert (buf == 7.0).all(), (lx, ly)
            n = lib.rof_layer_norm_workspace_bytes(rows, dim)
            ws = torch.full((n,), 255, dtype=torch.uint8, device=DEV)
            d = DTYPES[dtype]
            _native.check(lib.rof_dropout_forward(d, x.data_ptr(), x.stride(0), rows, dim, 0, b.data_ptr(), 1, drop, y.data_ptr(), y.stride(0), s))
            _native.check(lib.rof_dropout_backward(d, dy.data_ptr(), dy.stride(0), y.data_ptr(), y.stride(0), rows, dim, 0, 1, drop,
                                                   dx.data_ptr(), dx.stride(0), db.data_ptr(), ws.data_ptr(), n, s))
            for got, name in ((y, "y"), (dx, "dx"), (db, "db")):
                R.assert_within(got, plain[name], f"dropout {lx} {ly} {name}")
            for buf, view in ((ybuf, y), (gbuf, dx)):
                view.fill_(7.0)
                assert (buf == 7.0).all(), (lx, ly)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows, dim", [(5, 64), (5, 47), (3, 1001), (40000, 33), (1, 4097)])
def test_dropout_in_place_through_the_c_abi(dtype, rows, dim):
    """y may be x itself, and dx dy"""
    x, dy, b = randn(rows, dim, seed=1, dtype=dtype), randn(rows, dim, seed=2, dtype=dtype), randn(dim, seed=3)
    lib, d, s = _native.cuda(), DTYPES[dtype], torch.cuda.current_stream().cuda_stream
    drop = _native.Dropout(0.4, 9, 3, None, 0)
    for bias in (None, b):
        want = R.dropout_reference(x, bias, True, 0.4, 9, 3, dy=dy)
        y, dx = x.clone(), dy.clone()
        _native.check(lib.rof_dropout_forward(d, y.data_ptr(), dim, rows, dim, 0, bias.data_ptr() if bias is not None else None, 1, drop, y.data_ptr(), dim, s))
        _native.check(lib.rof_dropout_backward(d, dx.data_ptr(), dim, y.data_ptr(), dim, rows, dim, 0, 1, drop, dx.data_ptr(), dim, None,
                                               None, 0, s))
        R.assert_within(y, want["y"])
        R.assert_within(dx, want["dx"])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_without_weight_or_bias_and_weights_of_x_type(dtype):
    x, dy = randn(50, 96, seed=1, dtype=dtype), randn(50, 96, seed=2, dtype=dtype)
    w, b = randn(96, seed=3, shift=1.0), randn(96, seed=4)
    check_norm(x, None, None, dy, what="bare")
    check_norm(x, w, None, dy, what="no bias")
    check_norm(x, None, b, dy, what="no weight")
    check_norm(x, w.to(dtype), b.to(dtype), dy, what="x's type")
    check_norm(x, w.to(dtype), b, dy, what="mixed")
    check_norm(x, None, None, dy, p=0.4, seed=1, what="dropout without relu")


def test_mixed_vector_types_in_the_bound():
    # weight in bf16 beside a 32-bit bias: both are widened, nothing is rounded on the way
    x = randn(4, 40, dtype=BF16)
    w, b = randn(40, seed=1, dtype=BF16), randn(40, seed=2)
    assert torch.equal(norm.layer_norm(x, w, b), norm.layer_norm(x, w.float(), b))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_strides_and_alignment(dtype):
    w, b = randn(47, seed=3, shift=1.0), randn(47, seed=4)
    base, gbase = randn(70, 60, seed=1, dtype=dtype), randn(70, 64, seed=2, dtype=dtype)
    for x, dy in ((base[:, 3:50], gbase[:, 1:48]), (base[::2, :47], gbase[1::2, 17:]), (base[:, 4:51], gbase[:, 8:55]),
                  (base[:47, :].t(), gbase[:60, :47]), (base[:, :47], gbase[:, :47].contiguous())):
        check_norm(x, w, b, dy, what="norm")
        z = dict(relu=True, p=0.25, seed=8)
        check_norm(x, w, b, calm_gradient(dy, x, w, b, 1e-5), what="hidden", **z)
        check_dropout(x, b, dy, what="dropout", **z)
        check_dropout(x, None, dy, p=0.25, seed=8, what="dropout")
    x = empty_padded(31, 47, DEV)
    x.copy_(base[:31, :47].float())
    check_norm(x, w, b, gbase[:31, :47].float(), what="padded")
    x3 = randn(3, 5, 47, seed=5, dtype=dtype)
    check_norm(x3, w, b, randn(3, 5, 47, seed=6, dtype=dtype), what="3-D")
    check_norm(x3[0, 0], w, b, randn(47, seed=6, dtype=dtype), what="1-D")
    check_norm(x3, w, b, randn(1, 1, 47, seed=6, dtype=dtype).expand(3, 5, 47), what="expanded gradient")
    w0 = randn(94, seed=7, shift=1.0)[1::2]                                         # a strided weight
    check_norm(x3, w0, b, randn(3, 5, 47, seed=6, dtype=dtype), what="strided weight")


def check_dropout(x, bias, dy, relu=False, p=0.0, what="", **drop):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, bias)]
    y = norm.dropout(leaves[0], p, bias=leaves[1], relu=relu, **drop)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    grads = dict(zip(("dx", "db"), torch.autograd.grad(y, [t for t in leaves if t is not None], dy)))
    with torch.no_grad():
        assert torch.equal(norm.dropout(x, p, bias=bias, relu=relu, **drop), y)
    d = x.size(-1)
    want = R.dropout_reference(x.reshape(-1, d), bias, relu, p, dy=dy.reshape(-1, d), **drop)
    zero = want["y"][0] == 0
    assert ((y.reshape(-1, d) == 0).cpu().numpy() == zero).all() or x.dtype != F32, what   # the mask itself, element by element
    R.assert_within(y.reshape(-1, d), want["y"], what + " y")
    for k, g in grads.items():
        assert g.shape == dict(dx=x, db=bias)[k].shape and g.dtype == dict(dx=x, db=bias)[k].dtype
        R.assert_within(g, want[k], what + " " + k)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, dim", [(1, 1), (1, 7), (3, 2), (5, 3), (33, 16), (129, 47), (65, 100), (300, 128), (9, 257), (3000, 20),
                                       (40, 602), (5, 1031), (2, 4096), (1, 70001), (4000, 33)])
def test_dropout(dtype, rows, dim):
    x = randn(rows, dim, seed=1, shift=0.2, dtype=dtype)
    dy, b = randn(rows, dim, seed=2, dtype=dtype), randn(dim, seed=3).to(dtype)
    check_dropout(x, None, dy, p=0.3, seed=5, what="plain")
    check_dropout(x, b, dy, relu=True, p=0.5, seed=2 ** 64 - 1, step=2 ** 64 - 1, row_offset=9, what="bias relu")
    check_dropout(x, b, dy, p=0.1, seed=6, step=7, what="bias")
    check_dropout(x, b.float(), dy, relu=True, what="no dropout")
    check_dropout(x, None, dy, relu=True, p=0.9, seed=7, what="relu")


def test_dropout_extremes():
    x = randn(64, 33)
    assert torch.equal(norm.dropout(x, 0.0), x) and torch.equal(norm.dropout(x, 0.7, training=False), x)
    assert torch.equal(norm.dropout(x, 1e-12, seed=1), x)                            # below a step of the border: nothing is dropped
    bad = x.clone()
    bad[0, 0], bad[1, 1], bad[2, 2] = float("nan"), float("inf"), -float("inf")
    for kw in (dict(), dict(relu=True)):
        leaf = bad.clone().requires_grad_(True)
        y = norm.dropout(leaf, 1.0, seed=3, **kw)
        assert (y == 0).all()                                                       # a dropped NaN or infinity is zero
        assert (torch.autograd.grad(y, leaf, torch.full_like(y, float("inf")))[0] == 0).all()
    keep = torch.from_numpy(R.keep_mask(64, 33, 0.5, 3)).to(DEV)
    y = norm.dropout(bad, 0.5, seed=3)
    assert (y[~keep] == 0).all() and torch.equal(torch.isnan(y), torch.isnan(bad) & keep)
    y = norm.dropout(bad, 0.5, seed=3, relu=True)
    assert torch.equal(torch.isnan(y), torch.isnan(bad) & keep)                     # a ReLU keeps a NaN
    xs = torch.full((3, 5), float("nan"), device=DEV, requires_grad=True)
    g, = torch.autograd.grad(norm.dropout(xs, relu=True), xs, torch.ones(3, 5, device=DEV))
    assert (g == 1).all() == (torch.autograd.grad(F.relu(xs), xs, torch.ones(3, 5, device=DEV))[0] == 1).all()


def test_layer_norm_extremes():
    w, b = randn(40, seed=1, shift=1.0), randn(40, seed=2)
    # a constant row: no deviation, whatever its size; the gradient is finite
    x = torch.tensor([0.0, 1.0, -1e4, 12345.678, 3e-30], device=DEV)[:, None].expand(5, 40).contiguous().requires_grad_(True)
    y = norm.layer_norm(x, w, b)
    assert torch.equal(y, b.expand(5, 40))
    assert torch.isfinite(torch.autograd.grad(y.sum(), x)[0]).all()
    # a row far from zero keeps its deviations: the mean is corrected after the first sum
    x = (torch.arange(40, device=DEV, dtype=F32) + 2.0 ** 20).expand(3, 40)
    check_norm(x, w, b, randn(3, 40, seed=5), what="far from zero")
    # rows with infinities or NaN turn to NaN, the others do not notice
    x = randn(6, 40, seed=3)
    good = norm.layer_norm(x, w, b)
    x2 = x.clone()
    x2[1, 3], x2[4, 39] = float("inf"), float("nan")
    y2 = norm.layer_norm(x2, w, b, relu=True)
    assert torch.isnan(y2[1]).all() and torch.isnan(y2[4]).all()
    assert torch.equal(y2[[0, 2, 3, 5]], good.relu()[[0, 2, 3, 5]])
    # values whose squares pass the range of float16
    x = randn(4, 64, seed=4, scale=20000.0).clamp(-60000, 60000).to(F16)
    check_norm(x, None, None, randn(4, 64, seed=5, dtype=F16), what="large float16")
    # eps = 0 and one column
    check_norm(randn(9, 12, seed=6), None, None, randn(9, 12, seed=7), eps=0.0, what="eps 0")


def test_refusals():
    x, v = torch.zeros(4, 8, device=DEV), torch.zeros(8, device=DEV)
    for bad in (torch.zeros(7, device=DEV), torch.zeros(1, 8, device=DEV), torch.zeros(8), v.double(), v.half()):
        with pytest.raises(RuntimeError, match="weight must be"):
            norm.layer_norm(x, bad)
        with pytest.raises(RuntimeError, match="bias must be"):
            norm.layer_norm(x, v, bad)
        with pytest.raises(RuntimeError, match="bias must be"):
            norm.dropout(x, bias=bad)
    norm.layer_norm(x.half(), v.half(), v)                                            # either type beside the other
    for f in (norm.layer_norm, norm.dropout):
        with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
            f(x.double())
        with pytest.raises(RuntimeError, match="at least one dimension"):
            f(torch.zeros((), device=DEV))
        for step in (torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int64)):
            with pytest.raises(RuntimeError, match="step must be"):
                f(x, p=0.5, seed=1, step=step)
    for eps in (-1e-9, float("nan")):
        with pytest.raises(ValueError):
            norm.layer_norm(x, eps=eps)


def test_no_rows_and_no_columns():
    for shape in ((0, 16), (4, 0), (2, 0, 8), (0, 0)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        w, b = (torch.ones(shape[-1], device=DEV, requires_grad=True) for _ in range(2))
        y = norm.layer_norm(x, w, b, relu=True, p=0.5, seed=1)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert y.shape == gx.shape == shape and (gw == 0).all() and (gb == 0).all()
        y = norm.dropout(x, 0.5, seed=1, bias=b)
        gx, gb = torch.autograd.grad(y, (x, b), torch.zeros_like(y))
        assert y.shape == gx.shape == shape and (gb == 0).all()


def test_only_the_gradients_asked_for():
    x, w, b, dy = randn(70, 48, seed=1), randn(48, seed=2), randn(48, seed=3), randn(70, 48, seed=4)
    want = R.norm_reference(x, w, b, dy=dy)
    for names in (("dx",), ("dw",), ("db",), ("dx", "db"), ("dw", "db")):
        leaves = dict(dx=x.clone(), dw=w.clone(), db=b.clone())
        for k in names:
            leaves[k].requires_grad_(True)
        y = norm.layer_norm(leaves["dx"], leaves["dw"], leaves["db"])
        for k, g in zip(names, torch.autograd.grad(y, [leaves[k] for k in names], dy)):
            R.assert_within(g, want[k], k)
    bias = b.clone().requires_grad_(True)
    g, = torch.autograd.grad(norm.dropout(x, 0.5, seed=1, bias=bias, relu=True), bias, dy)
    R.assert_within(g, R.dropout_reference(x, b, True, 0.5, 1, dy=dy)["db"])


def test_row_blocks_drop_what_the_whole_matrix_drops():
    x = randn(101, 47, seed=1)
    whole = norm.dropout(x, 0.4, seed=9, step=3)
    parts = [norm.dropout(x[a:e], 0.4, seed=9, step=3, row_offset=a) for a, e in ((0, 1), (1, 38), (38, 101))]
    assert torch.equal(torch.cat(parts), whole)
    w, b = randn(47, seed=2), randn(47, seed=3)
    # (a block that starts off a 16-byte boundary adds its rows in another order: the same within the roundings of the sums)
    want = R.norm_reference(x, w, b, p=0.4, seed=9)["y"]
    whole = norm.layer_norm(x, w, b, p=0.4, seed=9)
    parts = torch.cat([norm.layer_norm(x[a:e], w, b, p=0.4, seed=9, row_offset=a) for a, e in ((0, 50), (50, 101))])
    assert torch.equal(parts == 0, whole == 0)
    R.assert_within(whole, want)
    R.assert_within(parts, want)
    # an element index beyond 2^34: the counter's second word counts
    far = 2 ** 34 // 47 + 5
    check_dropout(x, None, randn(101, 47, seed=4), p=0.5, seed=4, row_offset=far, what="far rows")
    check_norm(x, w, None, randn(101, 47, seed=4), p=0.5, seed=4, row_offset=far, what="far rows")


def test_results_repeat_bit_for_bit_and_graphs_are_kept():
    x, w, b, dy = randn(5000, 130, seed=1), randn(130, seed=2), randn(130, seed=3), randn(5000, 130, seed=4)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = norm.layer_norm(x, w, b, relu=True, p=0.5, seed=1)
    first = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)))
    with pytest.raises(RuntimeError):                                # a second derivative is refused, not wrong
        g, = torch.autograd.grad(norm.layer_norm(x, w, b).sum(), x, create_graph=True)
        g.sum().backward()
    y = norm.dropout(x, 0.5, seed=1, relu=True)
    y.mul_(2.0)                                                      # the backward pass reads y
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_seeds_come_from_torchs_generator():
    x = randn(50, 40)
    torch.manual_seed(3)
    a = norm.dropout(x, 0.5), norm.dropout(x, 0.5)
    torch.manual_seed(3)
    b = norm.dropout(x, 0.5), norm.dropout(x, 0.5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not torch.equal(a[0], a[1])
    # recomputation under checkpointing draws the same mask
    w = randn(40, 40, seed=1).requires_grad_(True)
    f = lambda t: norm.dropout(t @ w, 0.5, relu=True)  # noqa: E731
    torch.manual_seed(4)
    g1, = torch.autograd.grad(f(x).square().sum(), w)
    torch.manual_seed(4)
    g2, = torch.autograd.grad(torch.utils.checkpoint.checkpoint(f, x, use_reentrant=False).square().sum(), w)
    assert torch.equal(g1, g2)


def test_step_tensor_in_a_captured_graph():
    x = randn(64, 96, seed=1)
    w, b, dy = randn(96, seed=2), randn(96, seed=3), randn(64, 96, seed=4)
    step = torch.tensor([7], device=DEV)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]

    def work():
        y = norm.layer_norm(*leaves, p=0.5, seed=5, step=step)
        d = norm.dropout(leaves[0], 0.3, seed=6, step=step)
        out = (y, *torch.autograd.grad(y, leaves, dy), d, *torch.autograd.grad(d, leaves[0], dy))
        step.add_(1)
        return tuple(t.detach() for t in out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for k in (8, 9, 10):
        assert int(step) == k
        graph.replay()
        torch.cuda.synchronize()
        want = R.norm_reference(x, w, b, p=0.5, seed=5, step=k, dy=dy)
        for g, n in zip(got, ("y", "dx", "dw", "db")):
            R.assert_within(g, want[n], f"replay {k} {n}")
        want = R.dropout_reference(x, p=0.3, seed=6, step=k, dy=dy)
        R.assert_within(got[4], want["y"])
        R.assert_within(got[5], want["dx"])
    with pytest.raises(RuntimeError, match="seed"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            norm.dropout(x, 0.5)
    # changed between forward and backward: autograd refuses
    y = norm.dropout(leaves[0], 0.3, seed=6, step=step)
    step.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_capture_beside_a_living_eager_graph():
    """a step captured while an eager graph of the same tensors waits for its backward pass, which still works afterwards.  The
    captured one has leaves of its own on them: torch ties a leaf's node to the stream of the graph that lives, and refuses to capture
    across (for every operation alike)"""
    x, w, b, dy = randn(300, 100, seed=1), randn(100, seed=2, shift=1.0), randn(100, seed=3), randn(300, 100, seed=4)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def forward(leaves=leaves):
        return norm.dropout(norm.layer_norm(*leaves, relu=True, p=0.2, seed=1), 0.3, seed=2, bias=leaves[2])

    want = torch.autograd.grad(forward(), leaves, dy)
    eager = forward()
    own = [t.detach().requires_grad_(True) for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(forward(own), own, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(forward(own), own, dy)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(eager, leaves, dy), want))


def test_streams_and_graphs_side_by_side():
    x, w, b, dy = randn(3000, 200, seed=1), randn(200, seed=2), randn(200, seed=3), randn(3000, 200, seed=4)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def work(p):
        y = norm.layer_norm(*leaves, relu=True, p=p, seed=5)
        return tuple(t.detach() for t in (y, *torch.autograd.grad(y, leaves, dy)))

    want = {p: work(p) for p in (0.2, 0.6)}
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], {}
    for _ in range(5):
        for s, p in zip(streams, (0.2, 0.6)):
            with torch.cuda.stream(s):
                got[p] = work(p)
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for p in want for a, e in zip(got[p], want[p]))
    made = {}
    for p in (0.2, 0.6):                               # two captured graphs, replayed on two streams at once
        made[p] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(made[p]):
            got[p] = work(p)
    torch.cuda.synchronize()
    for _ in range(5):
        for s, p in zip(streams, (0.2, 0.6)):
            with torch.cuda.stream(s):
                made[p].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for p in want for a, e in zip(got[p], want[p]))


def test_more_than_two_to_the_31_elements():
    rows, dim = 2 ** 23 + 3, 264                       # 2.2e9 elements in 16 bits
    x = torch.empty((rows, dim), dtype=F16, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    for i in range(0, rows, 2 ** 20):
        x[i:i + 2 ** 20].normal_(generator=gen)
    w, b = randn(dim, seed=2, shift=1.0), randn(dim, seed=3)
    y = norm.layer_norm(x, w, b, p=0.5, seed=4)
    d = norm.dropout(x, 0.5, seed=4)
    for r in (0, 2 ** 31 // dim - 1, rows - 5):
        R.assert_within(y[r:r + 5], R.norm_reference(x[r:r + 5], w, b, p=0.5, seed=4, row_offset=r)["y"], f"rows {r}")
        R.assert_within(d[r:r + 5], R.dropout_reference(x[r:r + 5], p=0.5, seed=4, row_offset=r)["y"], f"rows {r}")
    del y, d
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = norm.layer_norm(x, w, b)
    gx, gw = torch.autograd.grad(y, (x, w), y.detach())
    r = rows - 5
    want = R.norm_reference(x[r:], w, b, dy=y[r:].detach())
    R.assert_within(gx[r:], want["dx"], "dx of the last rows")
    sums = torch.zeros(dim, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(sums)
    for i in range(0, rows, 2 ** 18):                  # dw = sum of y (x - mean) rstd
        xs = x[i:i + 2 ** 18].detach().double()
        h = (xs - xs.mean(1, keepdim=True)) / (xs.var(1, correction=0, keepdim=True) + 1e-5).sqrt()
        t = y[i:i + 2 ** 18].detach().double() * h
        sums += t.sum(0)
        bound += t.abs().sum(0)
    assert ((gw.double() - sums).abs() <= (1100 + rows / 1024 + 32) * R.U * bound).all()


# ---- in the models --------------------------------------------------------------------------------
def _gcn_inputs():
    g = graphs.config1()
    info = ROF_inputInfo.from_layouts(g.indptr_dst, search.search_graph(g, 3), device=DEV)
    return g, info, randn(g.num_nodes, 40, seed=1)


@pytest.mark.parametrize("with_norm", [False, True])
def test_gcn_stack_equals_its_parts(with_norm):
    """the fused passes of the stack against torch's operations with the same masks"""
    g, info, x = _gcn_inputs()
    torch.manual_seed(0)
    model = ROF_GCN(40, 16, 7, 2, dropout=0.4, add_self_loops=False, reuse_size=info.reuse_size, dropout_source="counter",
                    norm="layer" if with_norm else None).to(DEV)
    for m in model.norms or ():
        m.weight.data.uniform_(0.5, 1.5)
        m.bias.data.uniform_(-0.5, 0.5)
    for m in model.layers:
        m.bias.data.uniform_(-0.1, 0.1)
    out = model(x, info, seed=11, step=4)
    h = x
    for i, layer in enumerate(model.layers):
        h = layer(h, info)
        if i < 2:
            if with_norm:
                h = F.layer_norm(h, (16,), model.norms[i].weight, model.norms[i].bias)
            mask = torch.from_numpy(R.keep_mask(g.num_nodes, 16, 0.4, 11, 4 + (i << 40))).to(DEV)
            h = F.relu(h) * mask / 0.6
    assert (out - h).abs().max() <= 2e-5 * h.abs().max()
    params = [p for p in model.parameters() if p.requires_grad and p.shape[0] != info.reuse_size]
    wt = randn(*out.shape, seed=5)
    for a, e in zip(torch.autograd.grad(out, params, wt), torch.autograd.grad(h, params, wt)):
        assert (a - e).norm() <= 1e-3 * e.norm()           # an element next to the ReLU's border may fall on its other side
    assert not torch.equal(model(x, info), model(x, info))             # a new seed each time
    model.eval()
    want = model(x, info)
    with torch.no_grad():
        assert (model(x, info) - want).abs().max() <= 2e-5 * want.abs().max()


def test_gcn_stack_by_default_is_what_it_was():
    g, info, x = _gcn_inputs()
    torch.manual_seed(0)
    model = ROF_GCN(40, 16, 7, 1, dropout=0.5, add_self_loops=False, reuse_size=info.reuse_size).to(DEV)
    torch.manual_seed(1)
    out = model(x, info)
    torch.manual_seed(1)
    h = F.relu(model.layers[0](x, info))
    assert torch.equal(out, model.layers[1](F.dropout(h, 0.5, True), info))


def test_gcn_stack_with_another_activation():
    g, info, x = _gcn_inputs()
    torch.manual_seed(0)
    model = ROF_GCN(40, 16, 7, 1, activation=torch.tanh, dropout=0.5, add_self_loops=False, reuse_size=info.reuse_size,
                    dropout_source="counter", norm="layer").to(DEV)
    out = model(x, info, seed=2)
    h = torch.tanh(F.layer_norm(model.layers[0](x, info), (16,)))
    h = h * torch.from_numpy(R.keep_mask(g.num_nodes, 16, 0.5, 2)).to(DEV) * 2
    h = model.layers[1](h, info)
    assert (out - h).abs().max() <= 2e-5 * h.abs().max()
    mixed = ROF_GCN(40, 16, 7, 1, dropout=0.5, add_self_loops=False, reuse_size=info.reuse_size, norm="layer").to(DEV)
    torch.manual_seed(1)
    out = mixed(x, info)
    torch.manual_seed(1)
    h = F.relu(F.layer_norm(mixed.layers[0](x, info), (16,)))
    h = mixed.layers[1](F.dropout(h, 0.5, True), info)
    assert (out - h).abs().max() <= 2e-5 * h.abs().max()


def test_gcn_training_step_in_a_captured_graph():
    """a whole step — aggregation, norm, ReLU, dropout, loss, gradients — captured while an eager graph of the same leaves lives"""
    g, info, x = _gcn_inputs()
    torch.manual_seed(0)
    model = ROF_GCN(40, 16, 7, 2, dropout=0.5, add_self_loops=False, reuse_size=info.reuse_size, dropout_source="counter",
                    norm="layer").to(DEV)
    params = [p for p in model.parameters() if p.shape[0] != info.reuse_size]
    labels = torch.randint(0, 7, (g.num_nodes,), device=DEV)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)

    def work():
        loss = F.cross_entropy(model(x, info, seed=3, step=step), labels)
        grads = torch.autograd.grad(loss, params)
        return (loss.detach(), *grads)

    eager = []
    for k in range(3):
        step.fill_(k)
        eager.append(work())
    step.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
        step.add_(1)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(got, eager[k]):
            assert torch.allclose(a, e, rtol=1e-4, atol=1e-6), k        # cuBLAS may pick another product under capture


def test_gin_stack_with_norm_and_dropout():
    g = load_golden("c3_n1500_ps3")
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)  # noqa: E731
    ptr = g["indptr_dst"]
    plan = AggregationPlan.from_parts(g["N"], t(g["indices_src"]), t(ptr), t(np.arange(g["N"])))
    torch.manual_seed(0)
    model = ROF_GIN(20, 32, 5, norm="layer", dropout=0.25).to(DEV)
    x = randn(g["N"], 20, seed=1)
    out = model(x, plan, seed=6, step=1)
    h = x
    for i, mlp in enumerate(model.mlps):
        h = mlp(SumAggregate.apply(h, plan, None, None, "sum", 1.0))
        if i < 2:
            mask = torch.from_numpy(R.keep_mask(g["N"], 32, 0.25, 6, 1 + (i << 40))).to(DEV)
            h = F.relu(F.layer_norm(h, (32,))) * mask / 0.75
    assert (out - h).abs().max() <= 5e-5 * h.abs().max()
    out.sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
    model = ROF_GIN(20, 32, 5, dropout=0.25).to(DEV).eval()
    h = x
    for i, mlp in enumerate(model.mlps):
        h = mlp(SumAggregate.apply(h, plan, None, None, "sum", 1.0))
        h = F.relu(h) if i < 2 else h
    assert torch.equal(model(x, plan), h)
