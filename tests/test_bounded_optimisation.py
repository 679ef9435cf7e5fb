"""CPU: bounded gradients in the optimisation driver over several epochs -- L-BFGS whose gradients are scaled now and then, tolerances that mean the
gradient itself, epochs of several iterations; what a step that failed leaves behind."""
import copy
import numpy as np
import pytest
import torch
from test_grads_host import host, run, t64  # noqa: F401  (fixture)
from optim import ad_optim_lbfgs_mod as L


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
@pytest.mark.parametrize("ratio", [0.9, 0.7, 0.5, 0.3, 0.1])
def test_scaling_that_comes_to_an_end_on_the_way(host, tmp_path, dtype, ratio):
    """A convex quadratic whose gradient is scaled at the start and no longer later on: the loss never rises and reaches its minimum.  (Its Hessian is
    the identity: every secant pair of true gradients gives H = 1, so each epoch behind the first moves by 0.5 c g.)"""
    a0 = t64(2, 2, 2, 2, 2, seed=3, dtype=dtype)
    n0 = float(torch.linalg.vector_norm(a0 - 1.0))
    free = run(tmp_path, L, dtype=dtype, lr=0.5, epochs=60, tolerance_grad=0.0)[0]
    losses, mags, a, _ = run(tmp_path, L, dtype=dtype, lr=0.5, epochs=60, tolerance_grad=0.0, clip_grad_norm=ratio * n0)
    assert mags[0][0] > ratio * n0 > mags[-1][0]
    for r in (free, losses):
        assert all(y < x or y < 1e-24 for x, y in zip(r, r[1:])) and r[-1] < 1e-10 * r[0]
    # the loss of each epoch behind the second from the one before: g <- (1 - 0.5 c) g
    for (n, _), (m, _) in list(zip(mags[1:], mags[2:]))[:20]:
        assert abs(m / n - (1.0 - 0.5 * min(1.0, ratio * n0 / n))) < 1e-9


@pytest.mark.parametrize("bound", [1e-3, 1e-5, 5e-6, 1e-9])
def test_a_bound_below_the_tolerances_still_moves(host, tmp_path, bound):
    """The tolerances of the optimiser mean the gradient, not what is left of it: elements of the scaled gradient below tolerance_grad, a squared norm
    below tolerance_change."""
    losses, mags, a, a0 = run(tmp_path, L, lr=0.5, epochs=4, clip_grad_norm=bound, tolerance_grad=1e-5, tolerance_change=1e-30)
    n = mags[0][0]
    assert len(losses) == 4 and all(abs(m[0] / n - 1.0) < 1e-3 for m in mags)
    # four steps of 0.5 c g, |c g| = bound; values below 4: each step rounds each of the 32 elements by 4 x 2^-53 at most
    assert abs(float(torch.linalg.vector_norm(a - a0)) / (4 * 0.5 * bound) - 1.0) < 1e-6 + 4 * 32 ** 0.5 * 4 * 2.0 ** -53 / (2 * bound)
    g = a0 - 1.0
    assert float((a - (a0 - 4 * 0.5 * bound * g / n)).abs().max()) < 1e-5 * bound + 1e-15


def test_the_raw_gradient_ends_the_run(host, tmp_path):
    """max |g| <= tolerance_grad: nothing moves, whether the gradient would be scaled or not."""
    for bound in (0.0, 1e-2, 1e2):
        losses, _, a, a0 = run(tmp_path, L, lr=0.5, epochs=4, clip_grad_norm=bound, tolerance_grad=1e3)
        assert len(losses) == 1 and torch.equal(a, a0)


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
@pytest.mark.parametrize("iters", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("tol", [0.0, 1e-9, 1e-3])
def test_a_bound_above_the_norm_changes_nothing(host, tmp_path, dtype, iters, tol):
    """Bit for bit, down to convergence, with several iterations per epoch."""
    kw = dict(dtype=dtype, lr=0.75, epochs=12, max_iter_per_epoch=iters, tolerance_change=tol, tolerance_grad=1e-7)
    free, wide = run(tmp_path, L, **kw), run(tmp_path, L, clip_grad_norm=1e6, **kw)
    assert free[0] == wide[0] and torch.equal(free[2], wide[2]) and np.allclose(free[1], wide[1], rtol=1e-14)


def test_several_scaled_iterations_per_epoch(host, tmp_path):
    """Iterations of one epoch are those of epochs of one iteration."""
    # (an epoch of 3 iterations of torch's L-BFGS makes 3 evaluations, the last of which ends it: 2 steps)
    one = run(tmp_path, L, lr=0.5, epochs=2, clip_grad_norm=0.5, tolerance_grad=0.0)
    many = run(tmp_path, L, lr=0.5, epochs=1, max_iter_per_epoch=3, clip_grad_norm=0.5, tolerance_grad=0.0)
    assert len(many[0]) == 3 and many[0][:2] == one[0] and torch.equal(one[2], many[2])


def test_history_of_true_gradients_in_the_checkpoint(host, tmp_path):
    """The optimiser's memory holds the gradient itself: a run that resumes without the bound builds on it."""
    run(tmp_path, L, lr=0.5, epochs=3, clip_grad_norm=0.25, tolerance_grad=0.0)
    ck = torch.load(str(tmp_path / "o_checkpoint.p"), weights_only=False)
    st = next(iter(ck["optimizer_state_dict"]["state"].values()))
    for y, s in zip(st["old_dirs"], st["old_stps"]):
        assert float((y - s).abs().max()) <= 8 * 4 * 2.0 ** -53                # (identity Hessian; values below 4, a rounding of each operation)
    assert float(st["prev_flat_grad"].abs().max()) > 0.25


def test_a_checkpoint_brings_its_line_search_along(host, tmp_path):
    """Resumed without override it is the stored search that would run: refused under a bound, as it is at the start."""
    run(tmp_path, L, epochs=2, line_search="strong_wolfe")
    ck = str(tmp_path / "o_checkpoint.p")
    with pytest.raises(RuntimeError, match="clip_grad_norm needs the fixed step"):
        run(tmp_path, L, epochs=1, resume=ck, clip_grad_norm=0.5)
    run(tmp_path, L, epochs=1, resume=ck, override=True, clip_grad_norm=0.5)


def test_an_infinite_gradient_does_not_move_the_others(host, tmp_path):
    """c = 0: nothing is divided by the vanished gradient; 0 x inf is NaN, the other elements stay."""
    class Infinite(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, g):
            g = g.clone()
            g.view(-1)[5] = float("inf")
            return g
    a0 = t64(2, 2, 2, 2, 2, seed=3)
    import os
    import config as cfg
    from ipeps.ipeps_c4v import IPEPS_C4V
    from test_grads_host import Env
    st, opt_args, main_args = IPEPS_C4V(a0.clone()), copy.deepcopy(cfg.opt_args), copy.deepcopy(cfg.main_args)
    opt_args.clip_grad_norm, opt_args.lr = 0.5, 0.5
    main_args.opt_max_iter, main_args.out_prefix = 1, os.path.join(str(tmp_path), "o")
    L.optimize_state(st, Env(), lambda s, e, c: (0.5 * (Infinite.apply(s.site()) ** 2).sum(), e, [], 0.0, 0.0), main_args=main_args, opt_args=opt_args)
    a = st.site().detach().view(-1)
    other = torch.arange(32) != 5
    assert torch.isnan(a[5]) and torch.equal(a[other], a0.view(-1)[other])


# ---- the momentum step that fails -----------------------------------------------------------------------------------------------------------

class Fails:
    """The host's double of the library with calls that are refused as busy."""

    def __init__(self, host, calls):
        self.host, self.calls, self.n = host, set(calls), 0
        self.inner = host.lib.ctm_sgd_step
        host.lib.ctm_sgd_step = self
        host.lib.ctm_last_error = lambda h: b"in use"
        host._bind_dtype = lambda dt: setattr(host._tls, "h", None)
        import threading
        host._tls = threading.local()
        host._tls.h = None

    def __call__(self, *a):
        self.n += 1
        return 7 if self.n in self.calls else self.inner(*a)


def params(n=3):
    ps = [t64(4, 3, seed=i).requires_grad_() for i in range(n)]
    for i, p in enumerate(ps):
        p.grad = t64(4, 3, seed=10 + i)
    return ps


def garbage(monkeypatch):
    """Uninitialised memory holds NaN."""
    empty_like = torch.empty_like
    monkeypatch.setattr(torch, "empty_like", lambda t, **kw: empty_like(t, **kw).fill_(float("nan")))


@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_a_refused_first_step_leaves_nothing_behind(host, monkeypatch, max_norm):
    from _native import NativeError
    from optim.ad_optim_sgd_mod import SGD
    garbage(monkeypatch)
    kw = dict(lr=0.25, momentum=0.5, dampening=0.25, max_norm=max_norm)
    ref, ps = params(), params()
    a, b = SGD(ref, **kw), SGD(ps, **kw)
    a.step()
    a.step()
    Fails(host, [1])
    start = [p.detach().clone() for p in ps]
    with pytest.raises(NativeError, match="busy"):
        b.step()
    assert len(b.state_dict()["state"]) == 0 and b.norms is None and all(torch.equal(x, p) for x, p in zip(start, ps))
    b.step()
    b.step()
    assert all(torch.equal(x, y) and torch.equal(a.state[x]["momentum_buffer"], b.state[y]["momentum_buffer"]) for x, y in zip(ref, ps))


@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("call", [1, 2])
def test_a_refused_step_of_parameters_that_join_later(host, monkeypatch, call, max_norm):
    """Either of the two calls of such a step fails: as before the step, and the same step afterwards as without the failure."""
    from _native import NativeError
    from optim.ad_optim_sgd_mod import SGD
    garbage(monkeypatch)
    kw = dict(lr=0.25, momentum=0.5, dampening=0.25, max_norm=max_norm)

    def one():
        ps = params()
        late, ps[1].grad = ps[1].grad, None
        opt = SGD(ps, **kw)
        opt.step()
        ps[1].grad = late
        return ps, opt
    ref, a = one()
    a.step()
    ps, b = one()
    start, bufs = [p.detach().clone() for p in ps], [b.state[ps[i]]["momentum_buffer"].clone() for i in (0, 2)]
    Fails(host, [call])
    with pytest.raises(NativeError, match="busy"):
        b.step()
    assert all(torch.equal(x, p) for x, p in zip(start, ps)) and "momentum_buffer" not in b.state.get(ps[1], {})
    assert all(torch.equal(x, b.state[ps[i]]["momentum_buffer"]) for x, i in zip(bufs, (0, 2)))
    b.step()
    assert all(torch.equal(x, y) and torch.equal(a.state[x]["momentum_buffer"], b.state[y]["momentum_buffer"]) for x, y in zip(ref, ps))


# ---- checkpoints of torch's own gradient descent --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("momentum", [0.0, 0.5])
def test_state_of_torch_sgd_is_taken(host, momentum):
    """lr, momentum and dampening of torch.optim.SGD and its buffers; it knows no bound.  Without momentum its buffers are None."""
    from optim.ad_optim_sgd_mod import SGD
    ref, ps = params(), params()
    a = torch.optim.SGD(ref, lr=0.25, momentum=momentum, dampening=0.25 if momentum else 0.0)
    a.step()
    with torch.no_grad():
        for x, y in zip(ref, ps):
            y.copy_(x)
    b = SGD(ps, lr=1.0, momentum=0.125, max_norm=1e-3)
    b.load_state_dict(copy.deepcopy(a.state_dict()))          # (torch hands the buffers themselves over: both would write them)
    for _ in range(2):
        a.step()
        b.step()
    # (values below 4, five roundings a step at most, two steps)
    assert all(float((x - y).detach().abs().max()) <= 10 * 4 * 2.0 ** -53 for x, y in zip(ref, ps)) and b.norms is None
    # a momentum that begins later: its first step
    b.param_groups[0].update(momentum=0.5, dampening=0.0)
    if momentum == 0.0:
        before = [p.detach().clone() for p in ps]
        b.step()
        assert all(float((x - 0.25 * p.grad - p.detach()).abs().max()) <= 4 * 4 * 2.0 ** -53 for x, p in zip(before, ps))


@pytest.mark.parametrize("key,value", [("nesterov", True), ("weight_decay", 0.1), ("maximize", True)])
def test_state_of_torch_sgd_with_more_than_this_one_has(key, value):
    """An iteration that this optimiser does not make is refused, not replaced by another."""
    from optim.ad_optim_sgd_mod import SGD
    a, b = torch.optim.SGD(params(), lr=0.25, momentum=0.5, **{key: value}), SGD(params(), lr=0.25, momentum=0.5)
    with pytest.raises(ValueError, match=key):
        b.load_state_dict(a.state_dict())
    assert "nesterov" not in b.param_groups[0]


@pytest.mark.parametrize("override", [False, True])
def test_a_run_resumes_from_a_checkpoint_of_torch_sgd(host, tmp_path, override):
    """The bound, which the checkpoint does not have, is that of the run."""
    import os
    from optim import ad_optim_sgd_mod as S
    a0 = t64(2, 2, 2, 2, 2, seed=3)
    p = a0.clone().requires_grad_()
    opt = torch.optim.SGD([p], lr=0.25, momentum=0.5)
    p.grad = t64(2, 2, 2, 2, 2, seed=4)
    opt.step()
    m = opt.state[p]["momentum_buffer"].clone()
    ck = os.path.join(str(tmp_path), "torch.p")
    torch.save({"epoch": 1, "loss": 0.0, "parameters": {}, "optimizer_state_dict": opt.state_dict()}, ck)
    _, _, a, _ = run(tmp_path, S, epochs=1, resume=ck, override=override, lr=0.125, momentum=0.75, tolerance_grad=0.0, clip_grad_norm=0.5)
    g = a0 - 1.0
    lr, mu = (0.125, 0.75) if override else (0.25, 0.5)
    want = a0 - lr * (mu * m + g * (0.5 / torch.linalg.vector_norm(g)))
    assert float((a - want).abs().max()) < 1e-14


# ---- what the driver logs -------------------------------------------------------------------------------------------------------------------

def test_time_of_the_gradient_is_that_of_the_backward_pass(host, tmp_path, monkeypatch):
    """t_grad of the log line: neither the listing of the gradient (--OPTARGS_opt_log_grad) nor its norms."""
    import logging
    import json
    import time
    now = [0.0]
    monkeypatch.setattr(time, "perf_counter", lambda: now[0])
    tolist = torch.Tensor.tolist

    def slow(t):
        now[0] += 100.0
        return tolist(t)
    monkeypatch.setattr(torch.Tensor, "tolist", slow)
    lines = []

    class Lines(logging.Handler):
        def emit(self, record):
            lines.append(json.loads(record.getMessage()))
    h = Lines()
    L.log.addHandler(h)
    try:
        run(tmp_path, L, epochs=2, opt_log_grad=True, lr=0.5)
    finally:
        L.log.removeHandler(h)
    lines = [l for l in lines if "t_grad" in l]
    assert len(lines) == 2 and all(l["t_grad"] == 0.0 and len(l["grad"]) == 1 for l in lines)


def test_another_optimiser_gets_the_scaled_gradient(host, tmp_path, monkeypatch):
    """`create` of the driver: an optimiser that neither bounds its step itself nor is L-BFGS."""
    from types import SimpleNamespace

    def create(state, **kw):
        ps = list(state.get_parameters())
        for p in ps:
            p.requires_grad_(True)
        return ps, torch.optim.SGD(ps, lr=0.5)

    def optimize_state(*a, **kw):
        L.optimize_state(*a, create=create, **kw)
    losses, mags, a, a0 = run(tmp_path, SimpleNamespace(optimize_state=optimize_state), epochs=1, clip_grad_norm=0.5, opt_log_grad=True)
    g = a0 - 1.0
    n = float(torch.linalg.vector_norm(g))
    assert abs(mags[0][0] / n - 1.0) < 1e-14 and float((a - (a0 - 0.5 * 0.5 / n * g)).abs().max()) < 1e-14


def test_gradients_that_the_engine_does_not_hold(monkeypatch):
    """The log's norms of tensors on another device than the engine's go through torch, as those of host tensors do."""
    import backend

    class Elsewhere:
        device = torch.device("cuda", 1)

        def grad_norms(self, ts):
            raise AssertionError("tensors of another device")

    class OnGpu(torch.Tensor):                   # a host tensor that says it is on a device
        is_cuda = property(lambda t: True)
        device = property(lambda t: torch.device("cuda", 0))
    g = t64(5).as_subclass(OnGpu)
    backend.set_engine(Elsewhere())
    try:
        n2, top = L._grad_norms([g])
    finally:
        backend.set_engine(None)
    assert abs(n2 / float(torch.linalg.vector_norm(t64(5))) - 1) < 1e-14 and top == float(t64(5).abs().max())
