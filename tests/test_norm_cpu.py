"""Layer norm and dropout without a GPU: the generator against its published vectors, the refusals, the models' keywords."""
import ctypes

import numpy as np
import pytest
import torch

import norm_reference as R
from artifact_b200 import _native, norm
from artifact_b200.models import ROF_GCN, ROF_GIN


@pytest.mark.parametrize("rounds, ctr, key, words", [
    # the known answers that the authors of Philox publish with it (Random123, kat_vectors)
    (7, [0] * 4, (0, 0), (0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48)),
    (7, [0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF), (0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662)),
    (10, [0] * 4, (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    (10, [0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD))])
def test_generator_known_answers(rounds, ctr, key, words):
    assert tuple(int(v) for v in R.philox(ctr, key, rounds)) == words


def test_mask_follows_the_element_not_the_shape():
    whole = R.keep_mask(12, 10, 0.4, 77, 3)
    assert np.array_equal(whole.reshape(-1), R.keep_mask(8, 15, 0.4, 77, 3).reshape(-1))
    assert np.array_equal(whole[5:9], R.keep_mask(4, 10, 0.4, 77, 3, row_offset=5))
    assert not np.array_equal(whole, R.keep_mask(12, 10, 0.4, 77, 4)) and not np.array_equal(whole, R.keep_mask(12, 10, 0.4, 78, 3))
    share = R.keep_mask(1000, 100, 0.4, 1).mean()
    assert abs(share - 0.6) < 5 * np.sqrt(0.24 / 1e5)                 # five standard deviations


def test_reference_gradients_against_differences():
    gen = torch.Generator().manual_seed(3)
    x, dy = (torch.randn((5, 13), generator=gen, dtype=torch.float64) for _ in range(2))
    w, b, vw, vb = (torch.randn(13, generator=gen, dtype=torch.float64) for _ in range(4))
    v = torch.randn((5, 13), generator=gen, dtype=torch.float64)
    for kw in (dict(), dict(relu=True, p=0.3, seed=9, step=2)):
        r = R.norm_reference(x, w, b, 1e-5, dy=dy, **kw)
        f = lambda t: float((R.norm_reference(x + t * v, w + t * vw, b + t * vb, 1e-5, **kw)["y"][0] * dy.numpy()).sum())  # noqa: E731
        slope = (f(1e-6) - f(-1e-6)) / 2e-6
        want = (r["dx"][0] * v.numpy()).sum() + (r["dw"][0] * vw.numpy()).sum() + (r["db"][0] * vb.numpy()).sum()
        # second-order error 1e-12 and the roundings of f, about 1e-14, over 2e-6
        assert abs(slope - want) < 1e-6 * max(1.0, abs(want))
        r = R.dropout_reference(x, b, dy=dy, **kw)
        f = lambda t: float((R.dropout_reference(x + t * v, b + t * vb, **kw)["y"][0] * dy.numpy()).sum())  # noqa: E731
        want = (r["dx"][0] * v.numpy()).sum() + (r["db"][0] * vb.numpy()).sum()
        assert abs((f(1e-6) - f(-1e-6)) / 2e-6 - want) < 1e-6 * max(1.0, abs(want))


def test_no_cpu_path_and_no_other_types():
    x = torch.zeros(4, 8)
    for f in (norm.layer_norm, norm.dropout):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            f(x)
        with pytest.raises(TypeError):
            f([[1.0]])
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        norm.LayerNorm(8)(x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        norm.Dropout()(x)


@pytest.mark.parametrize("kw", [dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(p=0.5, seed=-1), dict(p=0.5, seed=2 ** 64),
                                dict(p=0.5, seed=1, step=-1), dict(p=0.5, seed=1, step=2 ** 64), dict(p=0.5, seed=1, row_offset=-1)])
def test_refused_dropout_arguments(kw):
    with pytest.raises(ValueError):
        norm.dropout(torch.zeros(2, 2), **kw)
    with pytest.raises(ValueError):
        norm.layer_norm(torch.zeros(2, 2), **kw)


def test_generator_arguments_and_seeds_from_torch():
    t = torch.zeros(1, dtype=torch.int64)
    assert norm._drop_args(0.5, 1, t, 0, True) == (0.5, 1, 0, 0, t)
    assert norm._drop_args(0.5, 2 ** 64 - 1, 2 ** 64 - 1, 3, True) == (0.5, 2 ** 64 - 1, 2 ** 64 - 1, 3, None)
    assert norm._drop_args(0.5, 1, 0, 0, False) == (0.0, 0, 0, 0, None) == norm._drop_args(0.0, None, 0, 0, True)
    torch.manual_seed(5)
    a = [norm.draw_seed() for _ in range(3)]
    torch.manual_seed(5)
    assert a == [norm.draw_seed() for _ in range(3)] and len(set(a)) == 3 and min(a) >= 0


def test_rows_views_and_copies():
    rows_of = _native.torch_ops().rows_of
    x = torch.arange(60.0).view(3, 4, 5)
    assert rows_of(x).shape == (12, 5) and rows_of(x).data_ptr() == x.data_ptr()
    assert rows_of(x[0, 0]).shape == (1, 5)
    assert rows_of(x.view(12, 5)[:, :3]).stride(0) == 5                           # padded rows stay where they are
    t = rows_of(torch.arange(12.0).view(3, 4).t())
    assert t.stride() == (3, 1) and torch.equal(t, torch.arange(12.0).view(3, 4).t())
    assert rows_of(torch.ones(1, 4).expand(3, 4)).stride() == (4, 1)              # an expanded gradient
    assert rows_of(torch.zeros(2, 3, 0)).shape == (6, 0) and rows_of(torch.zeros(0, 4)).shape == (0, 4)


def test_matrices_are_laid_alike():
    """a gradient whose rows lie differently against the 16-byte boundaries is copied, one that lies alike is not"""
    laid_like = _native.torch_ops().laid_like
    gen = torch.Generator().manual_seed(1)
    for dtype in (torch.float32, torch.bfloat16):
        per = 16 // torch.empty(0, dtype=dtype).element_size()
        flat = torch.randn(4096, generator=gen).to(dtype)
        start = -flat.data_ptr() // flat.element_size() % per         # an element on a boundary
        for off in (0, 1, 3):
            for ld in (12, 13, 14, 16, 40):
                v = flat.as_strided((7, 11), (ld, 1), start + off)
                for t in (v, v.contiguous(), flat.as_strided((7, 11), (24, 1), start), flat.as_strided((7, 11), (11, 1), start + 1)):
                    u = laid_like(t, v)
                    assert torch.equal(u, t) and u.stride(1) == 1 and u.stride(0) >= 11
                    for r in range(7):
                        assert (u[r].data_ptr() - v[r].data_ptr()) % 16 == 0
                assert laid_like(v, v).data_ptr() == v.data_ptr()
                one = flat.as_strided((1, 11), (3, 1), start + off)
                assert (laid_like(flat[start + 2:start + 13].view(1, 11), one).data_ptr() - one.data_ptr()) % 16 == 0


def test_c_entry_points_refuse_bad_arguments():
    """bad arguments come back as status codes before anything touches a device"""
    lib = _native.cuda()
    p = ctypes.cast((ctypes.c_double * 64)(), ctypes.c_void_p)
    p = ctypes.c_void_p((p.value + 15) // 16 * 16)
    odd = ctypes.c_void_p(p.value + 1)
    D = _native.Dropout

    def fwd(dtype=0, x=p, ldx=8, rows=4, dim=8, vt=0, w=p, b=p, eps=1e-5, drop=None, y=p, ldy=8, stats=p):
        return lib.rof_layer_norm_forward(dtype, x, ldx, rows, dim, vt, w, b, eps, 0, drop, y, ldy, stats, None)

    def bwd(dtype=0, dy=p, x=p, ldx=8, rows=4, dim=8, vt=0, stats=p, drop=None, dx=p, dw=p, db=p, ws=p, nws=0):
        return lib.rof_layer_norm_backward(dtype, dy, 8, x, ldx, rows, dim, vt, p, p, stats, 0, drop, dx, 8, dw, db, ws, nws, None)

    def drop_f(dtype=0, x=p, rows=4, dim=8, vt=0, b=p, drop=None, y=p, ldy=8):
        return lib.rof_dropout_forward(dtype, x, 8, rows, dim, vt, b, 0, drop, y, ldy, None)

    def drop_b(dtype=0, dy=p, y=p, rows=4, dim=8, relu=1, drop=None, dx=p, db=p, ws=p, nws=0):
        return lib.rof_dropout_backward(dtype, dy, 8, y, 8, rows, dim, 0, relu, drop, dx, 8, db, ws, nws, None)

    for f in (fwd, bwd, drop_f, drop_b):
        assert f(dtype=3) == 1 and f(dtype=-1) == 1 and f(rows=-1) == 1 and f(dim=-1) == 1
        assert f(rows=2 ** 62) == 1
        assert f(drop=D(1.5, 0, 0, None, 0)) == 1 and f(drop=D(float("nan"), 0, 0, None, 0)) == 1
        assert f(drop=D(0.5, 0, 0, None, -1)) == 1 and f(drop=D(0.5, 0, 0, None, 2 ** 62)) == 1
        assert f(drop=D(0.5, 0, 0, odd, 0)) == 1
        assert f(dim=0) == 0
    assert fwd(rows=0) == 0 and drop_f(rows=0) == 0
    for f in (fwd, drop_f):
        assert f(x=None) == 1 and f(y=None) == 1 and f(x=odd) == 1 and f(y=odd) == 1 and f(ldy=7) == 1 and f(vt=1) == 1 and f(b=odd) == 1
    assert fwd(ldx=7) == 1 and fwd(eps=-1.0) == 1 and fwd(eps=float("nan")) == 1 and fwd(w=odd) == 1 and fwd(stats=odd) == 1
    assert bwd(x=None) == 1 and bwd(dy=None) == 1 and bwd(stats=None) == 1 and bwd(ldx=7) == 1 and bwd(vt=2) == 1
    assert bwd(ws=None) == 4 and bwd(nws=8) == 4 and b"workspace" in lib.rof_last_error()
    assert bwd(dx=None, dw=None, db=None) == 0 and drop_b(dx=None, db=None) == 0
    assert drop_b(dy=None) == 1 and drop_b(y=None) == 1 and drop_b(ws=None) == 4
    assert lib.rof_layer_norm_workspace_bytes(-1, 8) == -1 and lib.rof_layer_norm_workspace_bytes(4, -1) == -1
    assert lib.rof_layer_norm_workspace_bytes(10 ** 9, 8) < 64 << 20


def test_model_keywords():
    with pytest.raises(ValueError):
        ROF_GCN(8, 4, 2, 1, norm="batch")
    with pytest.raises(ValueError):
        ROF_GCN(8, 4, 2, 1, dropout_source="curand")
    with pytest.raises(ValueError):
        ROF_GIN(8, 4, 2, norm="batch")
    plain, normed = ROF_GCN(8, 4, 2, 2, add_self_loops=False), ROF_GCN(8, 4, 2, 2, add_self_loops=False, norm="layer")
    extra = set(normed.state_dict()) - set(plain.state_dict())
    assert extra == {f"norms.{i}.{k}" for i in range(2) for k in ("weight", "bias")}
    assert set(ROF_GIN(8, 4, 2, 3, norm="layer").state_dict()) - set(ROF_GIN(8, 4, 2, 3).state_dict()) == extra
