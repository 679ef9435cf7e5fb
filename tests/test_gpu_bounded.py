"""Lists of gradients on the engine: values that are infinite and not a number at once, memory shared until the first write, bounded optimisation over
several epochs, steps that are refused."""
import math
import numpy as np
import pytest
import torch
from optim import grads as G

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("n", [1, 3, 12289, 200003])
@pytest.mark.parametrize("z", [complex(INF, NAN), complex(NAN, INF), complex(-INF, NAN), complex(NAN, -INF), complex(NAN, 0.0), complex(0.0, NAN),
                               complex(NAN, 1e300), complex(5e-324, NAN)])
def test_an_element_that_is_infinite_and_not_a_number(eng, z, n):
    """A NaN in either part: both norms NaN, a scaled list all NaN, whatever the other part is."""
    for at in {0, n // 2, n - 1}:
        a = np.ones(n, complex) * (0.5 - 0.25j)
        a[at] = z
        t = [dev(np.ones(5, complex)), dev(a)]
        assert all(math.isnan(v) for v in G.grad_norms(t).tolist())
        for norm_type in (2, INF):
            p = [torch.ones_like(x) for x in t]
            assert all(math.isnan(v) for v in G.sgd_step(p, t, lr=0.5, max_norm=1.0, norm_type=norm_type).tolist())
            assert all(bool(torch.isnan(torch.view_as_real(x)).all()) for x in p)
            out = [torch.zeros_like(x) for x in t]
            G.clip_grads(t, 1.0, norm_type, out=out)
            assert all(bool(torch.isnan(torch.view_as_real(x)).all()) for x in out)


@pytest.mark.parametrize("n", [1, 200003])
def test_infinite_elements_are_no_nan(eng, n):
    for z in (complex(INF, 0.0), complex(-INF, INF), complex(1e300, -INF)):
        a = np.ones(n, complex)
        a[n - 1] = z
        assert G.grad_norms([dev(a)]).tolist() == [INF, INF]


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
def test_memory_shared_until_the_first_write(eng, dtype):
    a = torch.randn(6, dtype=dtype, generator=torch.Generator().manual_seed(0)).cuda()
    keep = a.clone()
    b = a._lazy_clone()
    G.clip_grads([b], 0.5)
    assert torch.equal(a, keep) and abs(float(torch.linalg.vector_norm(b)) - 0.5) < 1e-14
    p, m, g = keep._lazy_clone(), keep._lazy_clone(), keep._lazy_clone()
    G.sgd_step([p], [g], [m], lr=0.5, momentum=0.5)
    assert torch.equal(g, a) and torch.equal(keep, a) and float((p - 0.25 * keep).abs().max()) < 1e-14


@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_a_refused_first_step(eng, max_norm):
    """A gradient that the call refuses (it is the parameter's own memory): nothing is left behind, the next step is a first one."""
    from _native import NativeError
    from optim.ad_optim_sgd_mod import SGD
    p, g = torch.ones(7, dtype=torch.float64, device="cuda").requires_grad_(), torch.full((7,), 0.125, dtype=torch.float64, device="cuda")
    opt = SGD([p], lr=0.5, momentum=0.5, max_norm=max_norm)
    p.grad = p.detach()
    with pytest.raises(NativeError, match="overlap"):
        opt.step()
    assert len(opt.state_dict()["state"]) == 0
    p.grad = g
    opt.step()
    assert torch.equal(opt.state[p]["momentum_buffer"], g) and torch.equal(p.detach(), 1.0 - 0.5 * g)      # |g| = 0.33: inside the bound


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
def test_bounded_lbfgs_over_several_epochs(eng, tmp_path, dtype):
    """The cases of the host's double (test_bounded_optimisation.py) on the engine."""
    from test_grads_host import run, t64
    from optim import ad_optim_lbfgs_mod as L
    n0 = float(torch.linalg.vector_norm(t64(2, 2, 2, 2, 2, seed=3, dtype=dtype) - 1.0))
    losses, mags, a, _ = run(tmp_path, L, "cuda", dtype, lr=0.5, epochs=60, tolerance_grad=0.0, clip_grad_norm=0.5 * n0)
    assert mags[0][0] > 0.5 * n0 > mags[-1][0] and losses[-1] < 1e-10 * losses[0]
    assert all(y < x or y < 1e-24 for x, y in zip(losses, losses[1:]))
    host = run(tmp_path, L, "cpu", dtype, lr=0.5, epochs=5, tolerance_grad=0.0)[0]
    free = run(tmp_path, L, "cuda", dtype, lr=0.5, epochs=5, tolerance_grad=0.0)[0]
    assert np.allclose(host, free, rtol=1e-12)
    for iters in (1, 4):
        kw = dict(lr=0.75, epochs=8, max_iter_per_epoch=iters, tolerance_change=1e-9, tolerance_grad=1e-7)
        free, wide = run(tmp_path, L, "cuda", dtype, **kw), run(tmp_path, L, "cuda", dtype, clip_grad_norm=1e6, **kw)
        assert free[0] == wide[0] and torch.equal(free[2], wide[2]) and free[1] == wide[1]


@pytest.mark.parametrize("dtype,n,bound", [(dt, n, b) for dt in (torch.float64, torch.complex128) for n in (3, 40, 12289) for b in (1e-3, 1e-10, 1e-300, 5e-324)]
                         + [(torch.float64, 17000003, 1e-10)])
def test_factors_below_the_normal_range(eng, dtype, n, bound):
    """Norms near the largest double under an ordinary bound: c = bound / norm has no 53 bits left, the scaled list has."""
    from test_gpu_grads import check_clip, check_norms, check_step, doubles, host, rand
    import grads_oracle as O
    rng = np.random.default_rng(12)
    a = [rand(n, dtype, rng), rand(5, dtype, rng)]
    a = [x * (1.5e308 / float(np.sqrt(sum((O.real_view(y) ** 2).sum() for y in a)))) for x in a]
    t = [dev(x) for x in a]
    out = [torch.zeros_like(x) for x in t]
    for norm_type in (2, INF):
        norms = check_norms(G.clip_grads(t, bound, norm_type, out=out), a)
        check_clip(host(out), a, bound, norm_type, norms)
    p0, m0 = [rand(x.shape, dtype, rng, bound) for x in a], [rand(x.shape, dtype, rng, bound) for x in a]
    if bound < 1e-200:
        return                                   # (sums of denormal numbers: exact or off by their own grid, nothing of the factor)
    ps, ms = [dev(x) for x in p0], [dev(x) for x in m0]
    G.sgd_step(ps, t, ms, lr=0.5, momentum=0.5, max_norm=bound)
    check_step(host(ps), host(ms), p0, m0, a, O.factor(norms[0], bound), O.tol_n2(doubles(a)) + O.U, 0.5, 0.5, 0.0, False)


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
def test_without_the_module_that_reads_lists(eng, monkeypatch, dtype):
    """The general way reaches the same kernels: the same bits."""
    ts = [torch.randn(n, dtype=dtype, device="cuda") for n in (1, 513, 70001)]

    def all_of_them():
        p, m, x, o = ([t.clone() for t in ts] for _ in range(4))
        r = [G.grad_norms(ts), G.clip_grads(x, 0.5), G.clip_grads(ts, 0.25, INF, out=o), G.sgd_step(p, ts, m, lr=0.5, momentum=0.5, max_norm=2.0)]
        return torch.cat([torch.view_as_real(t).reshape(-1) if t.is_complex() else t for t in r + p + m + x + o])
    short = all_of_them()
    monkeypatch.setattr(eng, "_lists", None)
    assert torch.equal(all_of_them(), short)
