"""Layer norm and dropout on the GPU at calls that the other tests do not make."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

import norm_reference as R
from artifact_b200 import _native, graphs, norm, search
from artifact_b200.models import ROF_GCN, ROF_GIN, ROF_inputInfo
from artifact_b200.plan import AggregationPlan
from conftest import load_golden
from test_gpu_norm import _c_norm, calm_gradient

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = {F32: 0, BF16: 1, F16: 2}                     # enum rof_dtype


def randn(*shape, seed=0, dtype=F32, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).to(DEV)


def padded(t, ld):
    """t with rows `ld` elements apart"""
    buf = torch.full((t.size(0), ld), 7.0, dtype=t.dtype, device=DEV)
    view = buf[:, :t.size(1)]
    view.copy_(t)
    return view


def c_dropout(x, bias, dy, y, dx, relu, drop):
    """both passes of rof_dropout_* into the given outputs -> dbias"""
    lib, d, s = _native.cuda(), DTYPES[x.dtype], torch.cuda.current_stream().cuda_stream
    rows, dim = x.shape
    vt = DTYPES[bias.dtype]
    db = torch.full((dim,), float("nan"), dtype=bias.dtype, device=DEV)
    n = lib.rof_layer_norm_workspace_bytes(rows, dim)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=DEV)          # whatever was there before
    _native.check(lib.rof_dropout_forward(d, x.data_ptr(), x.stride(0), rows, dim, vt, bias.data_ptr(), relu, drop, y.data_ptr(), y.stride(0), s))
    _native.check(lib.rof_dropout_backward(d, dy.data_ptr(), dy.stride(0), y.data_ptr() if relu else None, y.stride(0), rows, dim, vt, relu, drop,
                                           dx.data_ptr(), dx.stride(0), db.data_ptr(), ws.data_ptr(), n, s))
    return db


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("relu", [0, 1])
@pytest.mark.parametrize("rows, dim", [(1, 8), (5, 64), (70, 47), (9001, 47), (33, 602), (3, 1001)])
def test_dropout_gradients_in_place_with_a_bias_gradient(dtype, relu, rows, dim):
    """dx may be dy itself, on every path: dbias is the sum of what dy was"""
    x, b = randn(rows, dim, seed=1, dtype=dtype), randn(dim, seed=3)
    dy0 = randn(rows, dim, seed=2, dtype=dtype)
    want = R.dropout_reference(x, b, bool(relu), 0.4, 9, 3, dy=dy0)
    # y like dy, padded to whole vectors, and off by one element
    for ld in (dim, -(-dim // 8) * 8, dim + 1):
        dy = dy0.clone()
        y = padded(torch.zeros_like(x), ld)
        db = c_dropout(x, b, dy, y, dy, relu, _native.Dropout(0.4, 9, 3, None, 0))
        for got, name in ((y, "y"), (dy, "dx"), (db, "db")):
            R.assert_within(got, want[name], f"ld {ld} {name}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [1, 2, 3, 5, 7, 9])
def test_dropout_of_rows_shorter_than_a_vector(dtype, dim):
    """off the 16-byte boundaries: rows before the last reach the matrix's end too, and what lies around the outputs stays"""
    b = randn(dim, seed=3)
    for rows in (1, 2, 5, 19):
        for lead in (0, 1, 2, 3):
            for ld in (dim, dim + 1):
                laid = lambda: torch.full((8 + lead + rows * ld + 8,), 7.0, dtype=dtype, device=DEV)  # noqa: E731
                view = lambda buf: buf.as_strided((rows, dim), (ld, 1), 8 + lead)  # noqa: E731
                x, dy = view(laid()), view(laid())
                x.copy_(randn(rows, dim, seed=1, dtype=dtype))
                dy.copy_(randn(rows, dim, seed=2, dtype=dtype))
                ybuf, gbuf = laid(), laid()
                for relu in (0, 1):
                    want = R.dropout_reference(x, b, bool(relu), 0.4, 9, 3, dy=dy)
                    db = c_dropout(x, b, dy, view(ybuf), view(gbuf), relu, _native.Dropout(0.4, 9, 3, None, 0))
                    for got, name in ((view(ybuf), "y"), (view(gbuf), "dx"), (db, "db")):
                        R.assert_within(got, want[name], f"{rows} {lead} {ld} {name}")
                for buf in (ybuf, gbuf):
                    view(buf).fill_(7.0)
                    assert (buf == 7.0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("dim", [8, 47, 64, 100, 301, 602, 2049, 4097])
def test_relu_gradients_where_the_output_rounds_to_zero(dtype, p, dim):
    """x + bias may lie between zero and the type's smallest value: the output is zero, its gradient is not"""
    rows = 37
    least = 2.0 ** (-24 if dtype == F16 else -133)                     # the type's smallest value
    x = torch.zeros(rows, dim, dtype=dtype, device=DEV)
    x[::3] = least
    x[2::6] = -0.0
    x[1::6] = randn(len(range(1, rows, 6)), dim, seed=1, dtype=dtype)
    sizes = torch.tensor([0.25, 0.5, 0.49, 0.51, -0.5, 1.5, 0.0, -0.75, 1.0 / 256])
    b = (sizes[torch.arange(dim) % 9].double() * least).float().to(DEV)
    dy = randn(rows, dim, seed=2, dtype=dtype)
    drop = dict(p=p, seed=5, step=2) if p else {}
    want = R.dropout_reference(x, b, True, dy=dy, **drop)
    zeros = (want["dx"][0] != 0).sum()
    assert zeros > 0.3 * (1 - p) * rows * dim
    per = 8
    wide = -(-dim // per) * per + per
    for xs, gs in ((x, dy), (padded(x, wide), dy), (x, padded(dy, wide)), (padded(x, dim + 1), padded(dy, dim + 2))):
        leaf, bias = xs.detach().requires_grad_(True), b.clone().requires_grad_(True)
        y = norm.dropout(leaf, bias=bias, relu=True, **drop)
        R.assert_within(y, want["y"], "y")
        assert (want["y"][0][torch.signbit(y).cpu().numpy()] > 0).all()     # no other zero has a sign
        only, = torch.autograd.grad(y, leaf, gs, retain_graph=True)
        gx, gb = torch.autograd.grad(y, (leaf, bias), gs)
        R.assert_within(only, want["dx"], "dx alone")
        R.assert_within(gx, want["dx"], "dx")
        R.assert_within(gb, want["db"], "db")
    # the column sums of matrices that lie differently
    for ldy in (dim, wide, dim + 1):
        y, dx = padded(torch.zeros_like(x), ldy), torch.empty_like(dy)
        db = c_dropout(x, b, dy, y, dx, 1, _native.Dropout(p, 5, 2, None, 0) if p else None)
        for got, name in ((y, "y"), (dx, "dx"), (db, "db")):
            R.assert_within(got, want[name], f"ld {ldy} {name}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [8, 47, 64, 130, 602, 2048, 9000])
def test_rows_whose_variance_passes_the_range_of_32_bits(dtype, dim):
    """1 / sqrt(infinity) is zero: such a row is its bias, and its gradient is zero; the other rows do not notice"""
    x = randn(7, dim, seed=1, dtype=dtype)
    w, b = randn(dim, seed=3, shift=1.0), randn(dim, seed=4)
    dy = randn(7, dim, seed=2, dtype=dtype)
    big = torch.where(torch.arange(dim, device=DEV) % 2 == 0, 3e19, -1e20)
    x2 = x.clone()
    x2[1], x2[5] = big.to(dtype), (big * 1e10).to(dtype)
    rows = [0, 2, 3, 4, 6]
    leaves, others = [t.clone().requires_grad_(True) for t in (x2, w, b)], [t.clone().requires_grad_(True) for t in (x[rows], w, b)]
    y, small = norm.layer_norm(*leaves), norm.layer_norm(*others)
    assert torch.equal(y[1].float(), b.to(dtype).float()) and torch.equal(y[5].float(), b.to(dtype).float())
    want = R.norm_reference(x[rows], w, b, dy=dy[rows])
    gx, gw, gb = torch.autograd.grad(y, leaves, dy)
    R.assert_within(y[rows], want["y"], "y")
    R.assert_within(gx[rows], want["dx"], "dx")
    assert (gx[[1, 5]] == 0).all()
    R.assert_within(gw, want["dw"], "dw")                              # h is zero in those rows
    total = dy.double().sum(0).cpu().numpy()
    assert (np.abs(gb.double().cpu().numpy() - total) <= 16 * R.U * dy.double().abs().sum(0).cpu().numpy()).all()
    for p in (0.0, 0.5):
        hidden = norm.layer_norm(x2, w, b, relu=True, p=p, seed=3)
        keep = torch.from_numpy(R.keep_mask(7, dim, p, 3)).to(DEV)
        assert torch.equal(hidden[[1, 5]], torch.where(keep, F.relu(b).expand(7, dim) / (1 - p), 0.0).to(dtype)[[1, 5]])
    assert torch.equal(norm.layer_norm(x, w, b, eps=float("inf")), b.to(dtype).expand(7, dim))


def test_column_sums_of_the_widest_rows():
    """2^30 columns: the two vectors' gradients together have 2^31 entries"""
    lib, s, dim = _native.cuda(), torch.cuda.current_stream().cuda_stream, 2 ** 30
    n = lib.rof_layer_norm_workspace_bytes(1, dim)
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < n + 20 * 2 ** 30:
        pytest.skip("needs 84 GB")
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, dy = (torch.empty((1, dim), dtype=BF16, device=DEV).normal_(generator=gen) for _ in range(2))
    dw, db = (torch.full((dim,), float("nan"), dtype=BF16, device=DEV) for _ in range(2))
    ws, stats = torch.empty((n,), dtype=torch.uint8, device=DEV), torch.tensor([0.25, 0.5], device=DEV)
    for d in (dim, dim - 8):
        dw.fill_(float("nan"))
        db.fill_(float("nan"))
        _native.check(lib.rof_layer_norm_backward(1, dy.data_ptr(), d, x.data_ptr(), d, 1, d, 1, None, None, stats.data_ptr(), 0, None,
                                                  None, d, dw.data_ptr(), db.data_ptr(), ws.data_ptr(), n, s))
        assert torch.equal(db[:d], dy[0, :d]) and torch.isnan(db[d:]).all() and torch.isnan(dw[d:]).all()
        for i in range(0, d, 2 ** 26):
            e = min(i + 2 ** 26, d)
            assert torch.equal(dw[i:e], ((x[0, i:e].float() - 0.25) * 0.5 * dy[0, i:e].float()).to(BF16))
        db.fill_(float("nan"))
        _native.check(lib.rof_dropout_backward(1, dy.data_ptr(), d, None, d, 1, d, 1, 0, None, None, d, db.data_ptr(), ws.data_ptr(), n, s))
        assert torch.equal(db[:d], dy[0, :d])
    del ws
    torch.cuda.empty_cache()


def test_forward_mode_and_traces_are_refused():
    x, v = randn(4, 8, seed=1), randn(8, seed=2)
    for call in (lambda a, b: norm.layer_norm(a, b), lambda a, b: norm.layer_norm(a, None, b, relu=True), lambda a, b: norm.dropout(a, bias=b)):
        with torch.autograd.forward_ad.dual_level():
            for a, b in ((torch.autograd.forward_ad.make_dual(x, x), v), (x, torch.autograd.forward_ad.make_dual(v, v))):
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(a, b)
                with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(a, b)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, (x, v))
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x, v), (x, v))
        assert torch.isfinite(call(x, v)).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [8, 47, 64, 130, 301, 602, 1001])
def test_calm_gradients_with_strides_through_the_c_abi(dtype, dim):
    """mixes of how the four matrices lie, with no gradient next to the ReLU's border"""
    rows, w, b = 41, randn(dim, seed=13, scale=0.3, shift=1.0), randn(dim, seed=14, scale=0.3)
    x0 = randn(rows, dim, seed=11, dtype=dtype)
    dy0 = calm_gradient(randn(rows, dim, seed=12, dtype=dtype), x0, w, b, 1e-5)
    up = -(-dim // 8) * 8
    want = R.norm_reference(x0, w, b, relu=True, p=0.3, seed=9, step=3, row_offset=4, dy=dy0)
    layouts = (up, dim, dim + 1, up + 8)
    for i, lx in enumerate(layouts):
        for ly in (layouts[i], layouts[(i + 1) % 4], layouts[(i + 2) % 4]):
            y, dx = padded(torch.zeros_like(x0), ly), padded(torch.zeros_like(x0), lx)
            dw, db = _c_norm(padded(x0, lx), w, b, padded(dy0, ly), y, dx, 1, _native.Dropout(0.3, 9, 3, None, 4))
            for got, n in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
                R.assert_within(got, want[n], f"{lx} {ly} {n}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, dim", [(1, 7), (129, 47), (65, 100), (300, 128), (40, 602), (5, 1031), (1, 70001), (4000, 33)])
def test_masks_element_by_element(dtype, rows, dim):
    """zero exactly where the definition is, in 16 bits too, forward and back (values whose size the type can hold)"""
    x, dy, b = randn(rows, dim, seed=21, dtype=dtype), randn(rows, dim, seed=22, dtype=dtype), randn(dim, seed=23)
    for bias, relu in ((None, False), (b, False), (None, True), (b, True)):
        want = R.dropout_reference(x, bias, relu, 0.4, 7, 5, 2, dy=dy)
        leaf = x.clone().requires_grad_(True)
        y = norm.dropout(leaf, 0.4, seed=7, step=5, row_offset=2, bias=bias, relu=relu)
        for got, name in ((y, "y"), (torch.autograd.grad(y, leaf, dy)[0], "dx")):
            size = np.abs(want[name][0])
            held = (size == 0) | (size > 4 * R.tiny(dtype))
            assert held.mean() > 0.99 and ((got == 0).cpu().numpy() == (size == 0))[held].all(), (name, relu)


def test_lazily_negated_tensors():
    x, w, b, dy = randn(33, 24, seed=1), randn(24, seed=2), randn(24, seed=3), randn(33, 24, seed=4)
    n = [torch._neg_view(-t) for t in (x, w, b, dy)]

    def both(x, w, b, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y, d = norm.layer_norm(*leaves), norm.dropout(leaves[0], 0.3, seed=1, bias=leaves[2], relu=True)
        return y, d, *torch.autograd.grad(y, leaves, dy), *torch.autograd.grad(d, (leaves[0], leaves[2]), dy)

    for got, want in zip(both(*n), both(x, w, b, dy)):
        assert torch.equal(got, want)


def test_hooks_on_saved_tensors():
    """what is saved may travel (to the CPU and back, into another layout); what comes back as something else is refused: the kernels would
    read its memory"""
    x, w, b, dy = randn(33, 24, seed=1), randn(24, seed=2), randn(24, seed=3), randn(33, 24, seed=4)
    step, calm = torch.tensor([3], device=DEV), calm_gradient(dy, x, w, b, 1e-5)
    kinds = {(33, 24): "rows", (33, 2): "statistics", (24,): "vectors", (1,): "step"}

    def run(op, pack=None, unpack=None):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        if op == "norm":
            f = lambda: norm.layer_norm(*leaves, relu=True, p=0.3, seed=1, step=step)  # noqa: E731
        else:
            leaves.pop(1)
            f = lambda: norm.dropout(leaves[0], 0.3, seed=1, step=step, bias=leaves[1], relu=op == "relu")  # noqa: E731
        if pack is None:
            return torch.autograd.grad(f(), leaves, calm)
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = f()
        return torch.autograd.grad(y, leaves, calm)

    for op, saves in (("norm", {"rows", "statistics", "vectors", "step"}), ("relu", {"rows", "step"}), ("plain", {"step"})):
        want, seen = run(op), []
        if op == "norm":
            ref = R.norm_reference(x, w, b, relu=True, p=0.3, seed=1, step=3, dy=calm)
        else:
            ref = R.dropout_reference(x, b, op == "relu", 0.3, 1, 3, dy=calm)
        for same, pack, unpack in ((True, lambda t: (seen.append(kinds[tuple(t.shape)]), t.cpu())[1], lambda t: t.to(DEV)),
                                   (True, lambda t: t.t().contiguous(), lambda t: t.t()),             # columns one after the other
                                   (False, lambda t: padded(t, t.size(-1) + 3) if t.dim() == 2 else t, lambda t: t)):
            got = run(op, pack, unpack)
            # (rows that lie differently against the 16-byte boundaries are added in another order)
            assert not same or all(torch.equal(a, e) for a, e in zip(got, want)), op
            for g, name in zip(got, ("dx", "dw", "db") if op == "norm" else ("dx", "db")):
                R.assert_within(g, ref[name], f"{op} {name}")
        assert set(seen) == saves
        for kind in saves:
            for bad in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[:0]):
                with pytest.raises(RuntimeError, match="hook on saved tensors|must be"):
                    run(op, lambda t: bad(t) if kinds[tuple(t.shape)] == kind else t, lambda t: t)
        assert all(torch.equal(a, e) for a, e in zip(run(op), want))
    torch.cuda.synchronize()


# ---- in the models --------------------------------------------------------------------------------
def gcn(norm_kind="layer", source="counter", dropout=0.4, activation=F.relu, layers=2):
    g = graphs.config1()
    info = ROF_inputInfo.from_layouts(g.indptr_dst, search.search_graph(g, 3), device=DEV)
    torch.manual_seed(0)
    model = ROF_GCN(40, 16, 7, layers, activation=activation, dropout=dropout, add_self_loops=False, reuse_size=info.reuse_size,
                    norm=norm_kind, dropout_source=source).to(DEV)
    return model, info, randn(g.num_nodes, 40, seed=1)


@pytest.mark.parametrize("norm_kind, source", [(None, "counter"), ("layer", "counter"), ("layer", "torch")])
def test_training_mode_without_gradients_drops_too(norm_kind, source):
    """a pass in training mode is the same with and without gradients (the first pass of a reentrant checkpoint is one without)"""
    model, info, x = gcn(norm_kind, source)

    def run():
        torch.manual_seed(3)
        return model(x, info, seed=11, step=4)

    want = run()
    with torch.no_grad():
        assert torch.equal(run(), want)
    x.requires_grad_(True)
    params = [p for p in model.parameters() if p.requires_grad and p.shape[0] != info.reuse_size]
    torch.manual_seed(3)
    out = torch.utils.checkpoint.checkpoint(lambda t: model(t, info, seed=11, step=4), x, use_reentrant=True)
    assert torch.equal(out, want)
    grads = torch.autograd.grad(run().square().sum(), params)
    for p in params:
        p.grad = None
    out.square().sum().backward()
    for p, g in zip(params, grads):
        assert torch.equal(p.grad, g)
    model.eval()
    with torch.no_grad():
        got = model(x, info)
    assert (got - model(x, info)).abs().max() <= 2e-5 * got.abs().max()


def test_the_plain_stack_keeps_its_pass_without_gradients():
    """upstream's stack under no_grad is the fused inference pass, whatever its mode"""
    model, info, x = gcn(None, "torch")
    with torch.no_grad():
        got = model(x, info)
        assert torch.equal(got, model.eval()(x, info))


def test_hooks_of_a_stack_see_their_modules():
    """with a hook on it a norm or a layer is called as it stands, and the stack's result stays"""
    for norm_kind in ("layer", None):
        model, info, x = gcn(norm_kind)
        for m in model.norms or ():
            m.bias.data.uniform_(-0.5, 0.5)
        for m in model.layers:
            m.bias.data.uniform_(-0.1, 0.1)
        kw = dict(seed=11, step=4)
        want = model(x, info, **kw)
        seen = {}
        handles = [m.register_forward_hook(lambda mod, args, out, k=k: seen.__setitem__(k, (args[0].detach(), out.detach())))
                   for k, m in [(f"layer{i}", m) for i, m in enumerate(model.layers)] + [(f"norm{i}", m) for i, m in enumerate(model.norms or ())]]
        got = model(x, info, **kw)
        assert len(seen) == 3 + (2 if norm_kind else 0)
        for i, layer in enumerate(model.layers):
            given, out = seen[f"layer{i}"]
            assert torch.equal(out, layer(given, info))                # with its bias, without what follows
        for i, m in enumerate(model.norms or ()):
            given, out = seen[f"norm{i}"]
            assert torch.equal(given, seen[f"layer{i}"][1]) and torch.equal(out, norm.layer_norm(given, m.weight, m.bias))
        assert (got - want).abs().max() <= 2e-5 * want.abs().max()
        for h in handles:
            h.remove()
        assert torch.equal(model(x, info, **kw), want)


@pytest.mark.parametrize("make", [lambda: torch.nn.LayerNorm(16), lambda: torch.nn.Identity(), lambda: torch.nn.BatchNorm1d(16),
                                  lambda: norm.LayerNorm(16, relu=True)])
def test_replaced_norms_of_a_stack_are_called(make):
    model, info, x = gcn()
    for i in range(2):
        model.norms[i] = make().to(DEV)
    got = model(x, info, seed=11, step=4)
    h = x
    for i, layer in enumerate(model.layers):
        h = layer(h, info)
        if i < 2:
            mask = torch.from_numpy(R.keep_mask(x.size(0), 16, 0.4, 11, 4 + (i << 40))).to(DEV)
            h = F.relu(model.norms[i](h)) * mask / 0.6
    assert (got - h).abs().max() <= 2e-5 * h.abs().max()


def test_hooked_and_replaced_norms_of_a_gin_stack():
    g = load_golden("c3_n1500_ps3")
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)  # noqa: E731
    plan = AggregationPlan.from_parts(g["N"], t(g["indices_src"]), t(g["indptr_dst"]), t(np.arange(g["N"])))
    torch.manual_seed(0)
    model = ROF_GIN(20, 32, 5, norm="layer", dropout=0.25).to(DEV)
    x, kw = randn(g["N"], 20, seed=1), dict(seed=6, step=1)
    want, seen = model(x, plan, **kw), []
    handle = model.norms[0].register_forward_hook(lambda mod, args, out: seen.append(torch.equal(out, norm.layer_norm(args[0], mod.weight, mod.bias))))
    assert (model(x, plan, **kw) - want).abs().max() <= 2e-5 * want.abs().max() and seen == [True]
    handle.remove()
    handle = torch.nn.modules.module.register_module_forward_hook(lambda mod, args, out: seen.append(mod))
    try:
        model(x, plan, **kw)
    finally:
        handle.remove()
    assert all(m in seen for m in model.norms)
    model.norms[1] = torch.nn.LayerNorm(32).to(DEV)
    assert (model(x, plan, **kw) - want).abs().max() <= 2e-5 * want.abs().max()
    model.norms[0] = norm.LayerNorm(32, p=1.0).to(DEV)                  # its own dropout zeroes everything
    model.norms[0].register_forward_hook(lambda mod, args, out: seen.append(bool((out == 0).all())))
    model(x, plan, **kw)
    assert seen[-1] is True
