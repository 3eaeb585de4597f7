"""Layer norm and dropout without a GPU at calls that the other tests do not make."""
import io
import os
import pickle
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from artifact_b200 import _native, build, norm
from artifact_b200.models import ROF_GCN, ROF_GIN
from conftest import ROOT


@pytest.mark.parametrize("call, takes_v", [(lambda x, v: norm.layer_norm(x), False), (lambda x, v: norm.layer_norm(x, v), True),
                                           (lambda x, v: norm.layer_norm(x, None, v), True), (lambda x, v: norm.dropout(x), False),
                                           (lambda x, v: norm.dropout(x, 0.5, seed=1, bias=v), True)])
@pytest.mark.parametrize("grads", [False, True])
def test_forward_mode_is_refused(call, takes_v, grads):
    """not answered without a tangent"""
    x, v = torch.ones(4, 8, requires_grad=grads), torch.ones(8)
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            call(fwAD.make_dual(x, torch.ones(4, 8)), v)
        with pytest.raises(RuntimeError, match="no forward-mode derivative" if takes_v else "CUDA tensor"):
            call(x, fwAD.make_dual(v, torch.ones(8)))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        call(x, v)


@pytest.mark.parametrize("call", [lambda x: norm.layer_norm(x, relu=True), lambda x: norm.dropout(x, 0.5, seed=1),
                                  lambda x: norm.LayerNorm(8)(x), lambda x: norm.Dropout(0.0)(x)])
def test_traces_are_refused(call):
    """a trace would hold the allocation of the result and nothing that fills it"""
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, torch.ones(4, 8))


def test_no_vector_is_read_behind_the_matrix(tmp_path):
    """rows shorter than a vector: more rows than the last reach behind the matrix's end"""
    exe = str(tmp_path / "matrix_ends")
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(build._nvcc())))
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", build.CSRC, "-isystem", os.path.join(cuda, "include"),
                           os.path.join(ROOT, "tests", "abi", "matrix_ends.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and " wrong 0 held 0" in out.stdout, out.stdout


def test_the_c_abi_builds_without_torch(monkeypatch, capsys):
    """without torch's headers the two libraries that know nothing of torch are built as before"""
    monkeypatch.setattr(build, "_run", lambda cmd, verbose: None)
    monkeypatch.setattr(build, "_stale", lambda target, deps: True)
    found = build.importlib.util.find_spec
    assert build.torch_root() == os.path.dirname(torch.__file__)
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name, *more: None if name == "torch" else found(name, *more))
    monkeypatch.setitem(__import__("sys").modules, "torch", None)         # `import torch` raises
    assert build.build_all(verbose=False) == (build.cuda_lib_path(), build.host_lib_path())
    assert "rof_torch.so is not built" in capsys.readouterr().err


def test_the_torch_binding_is_built_anew_for_another_torch(monkeypatch, tmp_path):
    runs = []
    monkeypatch.setattr(build, "LIB", str(tmp_path))
    monkeypatch.setattr(build, "build_cuda", lambda **kw: "librof_b200.so")
    monkeypatch.setattr(build, "_run", lambda cmd, verbose: (runs.append(cmd), open(build.torch_lib_path(), "w").close()))
    build.build_torch(verbose=False)
    build.build_torch(verbose=False)
    assert len(runs) == 1
    monkeypatch.setattr(build, "_torch_stamp", lambda: "another")
    build.build_torch(verbose=False)
    build.build_torch(verbose=False)
    assert len(runs) == 2


def test_seeds_come_from_the_cpu_whatever_the_default_device():
    torch.manual_seed(5)
    want = [norm.draw_seed() for _ in range(2)]
    torch.manual_seed(5)
    with torch.device("meta"):                                           # (a GPU in a user's program)
        assert [norm.draw_seed() for _ in range(2)] == want


def test_models_saved_before_they_had_norms_load():
    """whole stacks pickled without the attributes that norm and dropout_source brought"""
    for model, made in ((ROF_GCN(8, 4, 2, 1), ("norms", "dropout_source")), (ROF_GIN(8, 4, 2), ("norms", "dropout"))):
        for k in made:
            delattr(model, k)
        buf = io.BytesIO()
        torch.save(model, buf)
        buf.seek(0)
        got = torch.load(buf, weights_only=False)
        assert got.norms is None and (got.dropout_source == "torch" if isinstance(got, ROF_GCN) else got.dropout == 0.0)
    for model in (ROF_GCN(8, 4, 2, 1, norm="layer", dropout_source="counter", dropout=0.3), ROF_GIN(8, 4, 2, norm="layer", dropout=0.3)):
        got = pickle.loads(pickle.dumps(model))
        assert got.dropout == 0.3 and len(got.norms) == len(model.norms) and getattr(got, "dropout_source", "counter") == "counter"


def test_lazily_negated_rows_are_read_negated():
    """a view whose memory holds the negatives (the imaginary part of a conjugate)"""
    rows_of = _native.torch_ops().rows_of
    x = torch.arange(12.0).view(3, 4)
    for v in (torch._neg_view(x), torch._neg_view(x)[:, :3], torch._neg_view(x)[0], torch.randn(4, 1, dtype=torch.complex64).conj().imag):
        r = rows_of(v)
        assert v.is_neg() and not r.is_neg() and torch.equal(r.view_as(v) if v.dim() == 2 else r[0], v.clone())
