"""CPU: csrc/lists.cpp, the short way of lists of tensors to the library -- memory that tensors share until one of them is written, an engine without
the module."""
import pytest
import torch
from test_grads_host import HostEngine, host, t64  # noqa: F401  (fixture)
from optim import grads as G


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
def test_copies_made_on_the_first_write(host, dtype):
    """Every list that a call writes gets memory of its own, whoever shares it so far; lists that are read stay shared."""
    a, p0, m0 = (t64(6, dtype=dtype, seed=i) for i in range(3))
    keep = a.clone()
    b = a._lazy_clone()
    G.clip_grads([b], 0.5)
    assert torch.equal(a, keep) and abs(float(torch.linalg.vector_norm(b)) - 0.5) < 1e-14
    out = a._lazy_clone()
    G.clip_grads([a], 0.5, out=[out])
    assert torch.equal(a, keep) and torch.equal(out, b)
    p, m, g = p0._lazy_clone(), m0._lazy_clone(), a._lazy_clone()
    kp, km = p0.clone(), m0.clone()
    G.sgd_step([p], [g], [m], lr=0.5, momentum=0.5)
    assert torch.equal(p0, kp) and torch.equal(m0, km) and torch.equal(a, keep) and torch.equal(g, keep)
    # (products and sums of three terms, values below 8)
    assert float((m - (0.5 * km + keep)).abs().max()) < 1e-14 and float((p - (kp - 0.5 * (0.5 * km + keep))).abs().max()) < 1e-14
    # parameters, gradients and momentum that share one memory
    p, m, g = keep._lazy_clone(), keep._lazy_clone(), keep._lazy_clone()
    G.sgd_step([p], [g], [m], lr=0.5, momentum=0.5)
    assert torch.equal(g, keep) and torch.equal(keep, a) and float((p - 0.25 * keep).abs().max()) < 1e-14
    assert torch.equal(G.grad_norms([g]), G.grad_norms([keep])) and torch._C._is_cow_tensor(keep._lazy_clone())


def engine(monkeypatch):
    """An engine as its constructor makes it, on a machine whose library has no device behind it."""
    import _native

    class Lib:
        ctm_grad_norms = ctm_grad_clip = ctm_sgd_step = 0
    monkeypatch.setattr(_native, "load_library", lambda: Lib)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(_native.Engine, "_bind_dtype", lambda self, dt: None)
    return _native.Engine(torch.device("cpu"))


def test_an_engine_without_the_module(monkeypatch):
    """The module only reads lists: without it the engine starts, says so, and takes lists its general way."""
    import _native

    def missing():
        raise _native.NativeError("not there")
    assert engine(monkeypatch)._lists is _native.load_lists()
    monkeypatch.setattr(_native, "load_lists", missing)
    with pytest.warns(UserWarning, match="not there"):
        e = engine(monkeypatch)
    assert e._lists is None and e._short("grad_norms", "grad_norms", [t64(3)]) is None


def test_a_module_of_another_torch_is_refused():
    """It reads torch's own structures: compiled against another release it must not load."""
    import os
    import subprocess
    import sys
    from conftest import PKG
    code = "import torch, sys\n%s\nsys.path.insert(0, sys.argv[1])\nimport _native\ntry:\n    _native.load_lists()\nexcept _native.NativeError as e:\n    print('refused:', e)\nelse:\n    print('loaded')"
    for change, want in (("", "loaded"), ("torch.__version__ = '2.9.0+rocm7.0'", "refused: "), ("torch.__version__ = '2.100.0'", "refused: ")):
        r = subprocess.run([sys.executable, "-c", code % change, PKG], capture_output=True, text=True, timeout=110)
        assert r.stdout.startswith(want), (r.stdout, r.stderr[-2000:])
        assert want == "loaded" or "build it with" in r.stdout


def test_the_module_is_built_again_for_another_torch(monkeypatch, tmp_path):
    import importlib.util
    import os
    import subprocess
    from conftest import PKG
    spec = importlib.util.spec_from_file_location("ctm_build", os.path.join(PKG, "csrc", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    runs = []

    def check_call(cmd):
        runs.append(cmd)
        open(b.EXT, "w").close()
    monkeypatch.setattr(subprocess, "check_call", check_call)
    monkeypatch.setattr(b, "EXT", str(tmp_path / "_ctm_lists.so"))
    b.build_ext(verbose=False)
    b.build_ext(verbose=False)
    assert len(runs) == 1
    monkeypatch.setattr(torch, "__version__", "2.9.0")
    b.build_ext(verbose=False)
    b.build_ext(verbose=False)
    assert len(runs) == 2
    b.build_ext(force=True, verbose=False)
    assert len(runs) == 3
