"""CPU: the host side of the optimiser's operators over lists (checks of arguments, orders and views, what is written back), on a double of the
library that computes on host memory; gradient descent and clipping in the optimisation driver."""
import copy
import ctypes as C
import json
import logging
import math
import os
import threading
import numpy as np
import pytest
import torch
import _native
import backend
import config as cfg
import grads_oracle as O
from _native import NativeError
from optim import grads as G

INF = float("inf")


class HostLib:
    """The three C entries on host memory (numpy); `calls` keeps what arrived."""

    def __init__(self):
        self.calls, self.cplx = [], False

    def _arr(self, ptrs, n, i):
        k = n[i] * (2 if self.cplx else 1)
        if k == 0:
            return np.zeros(0)
        return np.ctypeslib.as_array(C.cast(ptrs[i], C.POINTER(C.c_double)), (k,))

    def _norms(self, nt, x, n, ws, code, bound):
        xs = [self._arr(x, n, i) for i in range(nt)]
        n2 = math.sqrt(math.fsum(float(v) ** 2 for a in xs for v in a))
        top = max([0.0] + [float((np.hypot(a[::2], a[1::2]) if self.cplx else np.abs(a)).max()) for a in xs if a.size])
        nrm = n2 if code == 2 else top
        c = 1.0 if bound < 0 or nrm <= bound else bound / nrm
        if ws is not None:
            np.ctypeslib.as_array(C.cast(ws, C.POINTER(C.c_double)), (3,))[:] = (n2, top, c)
        return c

    def ctm_grad_norms(self, h, s, nt, x, n, ws, wsn):
        self.calls.append("norms")
        self._norms(nt, x, n, ws, 2, -1.0)
        return 0

    def ctm_grad_clip(self, h, s, nt, x, y, n, code, bound, ws, wsn):
        self.calls.append("clip")
        c = self._norms(nt, x, n, ws, code, bound)
        for i in range(nt):
            self._arr(y, n, i)[:] = self._arr(x, n, i) * c
        return 0

    def ctm_sgd_step(self, h, s, nt, p, g, m, n, lr, mu, tau, first, code, bound, ws, wsn):
        self.calls.append("step")
        c = self._norms(nt, g, n, ws, code, bound) if bound >= 0 else 1.0
        for i in range(nt):
            d = c * self._arr(g, n, i)
            if m is not None:
                b = self._arr(m, n, i)
                b[:] = d if first else mu * b + (1 - tau) * d
                d = b
            self._arr(p, n, i)[:] -= lr * d
        return 0


class HostEngine(_native.Engine):
    """`short`: with the module that reads plain lists (csrc/lists.cpp), its entries the double's."""

    def __init__(self, short=False):
        self.lib, self.device, self._handles = HostLib(), torch.device("cpu"), {}
        if short:
            self._lists, self._short_calls = _native.load_lists(), 0
            self._handles = {torch.float64: C.c_void_p(8), torch.complex128: C.c_void_p(16)}
            self._keep = {}
            for n in ("grad_norms", "grad_clip", "sgd_step"):
                sig = _native._SIGS["ctm_" + n]

                def entry(h, *a, n=n):
                    self.lib.cplx = h == 16
                    self._short_calls += 1
                    return getattr(self.lib, "ctm_" + n)(h, *[v if v or not isinstance(v, C._Pointer) else None for v in a])
                self._keep[n] = C.CFUNCTYPE(C.c_int, *sig)(entry)
            self._entries = {n: C.cast(f, C.c_void_p).value for n, f in self._keep.items()}

    def __del__(self):
        pass

    def _stream(self):
        return 0

    def _run_lists(self, what, dt, fn):
        self.lib.cplx = dt.is_complex
        self._ck(fn(None, None), what)


@pytest.fixture(params=[False, True], ids=["general", "short"])
def host(request):
    e = HostEngine(request.param)
    backend.set_engine(e)
    yield e
    backend.set_engine(None)


def t64(*shape, seed=0, dtype=torch.float64):
    return torch.randn(*shape, dtype=dtype, generator=torch.Generator().manual_seed(seed))


VIEWS = {"whole": lambda t: t, "transposed": lambda t: t.permute(2, 0, 1), "sliced": lambda t: t[:, 1:3], "stepped": lambda t: t[::2, :, 1],
         "scalar": lambda t: t[1, 2, 0], "empty": lambda t: t[:0]}


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
@pytest.mark.parametrize("view", list(VIEWS))
def test_orders_and_views(host, view, dtype):
    f = VIEWS[view]
    base, other = t64(4, 5, 3, dtype=dtype), t64(7, seed=1, dtype=dtype)
    flat = torch.cat([f(base).reshape(-1), other])
    n = torch.linalg.vector_norm(flat)
    got = G.grad_norms([f(base), other])
    assert torch.allclose(got, torch.stack([n, flat.abs().max()]), rtol=1e-14, atol=0)
    for norm_type, nrm in ((2, n), (INF, flat.abs().max())):
        x, o, out, src = base.clone(), other.clone(), base.clone(), other.clone()
        c = min(1.0, 0.5 / float(nrm))
        v0 = x._version
        assert torch.equal(G.clip_grads([f(x), o], 0.5, norm_type), got)
        want = base.clone()
        f(want).mul_(c)
        assert torch.allclose(x, want, rtol=1e-14, atol=0) and torch.allclose(o, other * c, rtol=1e-14, atol=0)
        assert x._version > v0 and x.stride() == base.stride()
        G.clip_grads([f(base), other], 0.5, norm_type, out=[f(out), src])
        assert torch.equal(out, x) and torch.equal(src, o)
    p, m, g = base.clone(), 2 * base, 3 * base
    G.sgd_step([f(p)], [f(g).contiguous()], [f(m)], lr=0.5, momentum=0.25, dampening=0.5)
    wp, wm = base.clone(), 2 * base
    f(wm).copy_(0.25 * f(2 * base) + 0.5 * f(g))
    f(wp).copy_(f(base) - 0.5 * f(wm))
    assert torch.allclose(p, wp, rtol=1e-14, atol=1e-300) and torch.allclose(m, wm, rtol=1e-14, atol=1e-300) and torch.equal(g, 3 * base)


def test_conjugated_negated_and_broadcast_inputs(host):
    z = t64(3, 4, dtype=torch.complex128)
    e = t64(1, 2).expand(5, 2)
    assert torch.allclose(G.grad_norms([e])[0], torch.linalg.vector_norm(e), rtol=1e-14)
    o = torch.zeros(3, 4, dtype=torch.complex128)
    G.clip_grads([z.conj()], INF, out=[o])
    assert torch.equal(o, z.conj().resolve_conj())
    o = torch.zeros(3, 4, dtype=torch.float64)
    G.clip_grads([z.conj().imag], INF, out=[o])
    assert torch.equal(o, -z.imag)
    p = torch.zeros(3, 4, dtype=torch.complex128)
    G.sgd_step([p], [z.conj()], lr=1.0)
    assert torch.equal(p, -z.conj())


def test_gradients_with_a_pending_conjugation_or_sign(host):
    """What autograd leaves in `.grad`: scaled in place, whatever the flag says about the memory."""
    z = t64(3, 4, dtype=torch.complex128)
    n = float(torch.linalg.vector_norm(z))
    for view in (lambda t: t.conj(), lambda t: t.conj().t(), lambda t: t.conj()[1:, ::2]):
        m = z.clone()
        v = view(m)
        k = float(torch.linalg.vector_norm(v))
        got = G.clip_grads([v], 0.25)
        want = z.clone()
        view(want).mul_(0.25 / k)
        assert abs(float(got[0]) / k - 1) < 1e-14 and torch.allclose(m, want, rtol=1e-14, atol=0) and v.is_conj()
    m = z.clone()
    G.clip_grads([m.conj().imag], 0.0)
    assert torch.equal(m, torch.complex(z.real, torch.zeros_like(z.real)))
    p = torch.zeros_like(z).requires_grad_()
    p.grad = z.clone().conj()
    assert p.grad.is_conj()
    G.clip_grad_norm_([p], 1.0)
    assert torch.allclose(p.grad, z.conj() / n, rtol=1e-14, atol=0)
    G.clip_grad_norm_(p, 0.5)
    assert torch.allclose(p.grad, z.conj() * (0.5 / n), rtol=1e-14, atol=0)
    assert torch.equal(G.grad_norms(z), G.grad_norms([z]))


def test_refusals_before_anything_is_written(host):
    t, u, z = torch.ones(8, dtype=torch.float64), torch.ones(8, dtype=torch.float64), torch.ones(8, dtype=torch.complex128)
    meta = torch.ones(8, dtype=torch.float64, device="meta")
    bad = [lambda: G.grad_norms([t, meta]), lambda: G.grad_norms([t.float()]), lambda: G.grad_norms([t, z]), lambda: G.grad_norms([t, None]),
           lambda: G.grad_norms([3.0]), lambda: G.grad_norms([t.to_sparse()]), lambda: G.clip_grads([t], -1.0), lambda: G.clip_grads([t], float("nan")),
           lambda: G.clip_grads([t], 1.0, norm_type=1), lambda: G.clip_grads([t], 1.0, out=[]), lambda: G.clip_grads([t], 1.0, out=[u[:7]]),
           lambda: G.clip_grads([t[:1].expand(3)], 0.5), lambda: G.clip_grads([z], 0.5, out=[torch.ones_like(z).conj()]),
           lambda: G.sgd_step([z.conj()], [torch.ones_like(z)], lr=0.5), lambda: G.clip_grads([t[0:6:2], t[1:7:2]], 0.5),
           lambda: G.clip_grads([t.as_strided((3, 3), (2, 1))], 0.5), lambda: G.clip_grads([t[::2], t[:4]], 0.5),
           lambda: G.sgd_step([t], [u], lr=-1.0), lambda: G.sgd_step([t], [u], momentum=0.5), lambda: G.sgd_step([t], [u, u]),
           lambda: G.sgd_step([t], [u], [u[:4]], momentum=0.5), lambda: G.sgd_step([t[::2]], [u[::2]], [t[::2]], momentum=0.5),
           lambda: G.sgd_step([t], [z]), lambda: G.sgd_step([t], [u], max_norm=-2.0), lambda: G.sgd_step([t], [u], [u], momentum=float("nan")),
           lambda: G.sgd_step([t], [u], lr=float("nan")), lambda: G.sgd_step([t], [u], max_norm=1.0, norm_type=3)]
    for call in bad:
        with pytest.raises(NativeError):
            call()
    assert not host.lib.calls
    assert torch.equal(t, torch.ones_like(t)) and torch.equal(u, torch.ones_like(u))


def test_which_lists_go_the_short_way():
    """Contiguous tensors of one dtype, in any number; the rest goes the general way with the same results."""
    e, d = HostEngine(True), HostEngine()
    for dt in (torch.float64, torch.complex128):
        ts = [t64(n, dtype=dt, seed=n) for n in (1, 0, 7, 300)]
        assert torch.equal(e.grad_norms(ts), d.grad_norms(ts)) and torch.equal(e.grad_norms(tuple(ts)), d.grad_norms(iter(ts)))
        a, b = [t.clone() for t in ts], [t.clone() for t in ts]
        v = a[2]._version
        assert torch.equal(e.clip_grads(a, 0.5), d.clip_grads(b, 0.5)) and a[2]._version == v + 1
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        o = [torch.zeros_like(t) for t in ts]
        e.clip_grads(ts, 0.5, INF, out=o)
        d.clip_grads(ts, 0.5, INF, out=b)
        assert all(torch.equal(x, y) for x, y in zip(o, b)) and o[2]._version > 0
        p, q, m, k = ([t.clone() for t in ts] for _ in range(4))
        got, want = (f.sgd_step(x, ts, y, lr=0.5, momentum=0.5, dampening=0.25, first=0, max_norm=0.5) for f, x, y in ((e, p, m), (d, q, k)))
        assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(p + m, q + k))
        assert e.sgd_step(p, ts, lr=0.5) is None and d.sgd_step(q, ts, lr=0.5) is None and all(torch.equal(x, y) for x, y in zip(p, q))
        calls = e._short_calls
        odd = [t64(4, 3, dtype=dt).t()]
        assert torch.equal(e.grad_norms(odd), d.grad_norms(odd)) and torch.equal(e.grad_norms([]), d.grad_norms([])) and e._short_calls == calls
    assert e._short_calls == 12
    with torch.inference_mode():
        x = torch.ones(3, dtype=torch.float64)
        e.clip_grads([x], 0.0)
        d.clip_grads([x], 0.0)
    # a status of the library reaches the caller as its error
    e._bind_dtype = lambda dt: None
    e.lib.ctm_last_error = lambda h: b"in use"
    busy = C.CFUNCTYPE(C.c_int, *_native._SIGS["ctm_grad_norms"])(lambda *a: 7)
    e._entries["grad_norms"] = C.cast(busy, C.c_void_p).value
    e._tls = threading.local()
    e._tls.h = None
    with pytest.raises(NativeError, match="busy"):
        e.grad_norms([torch.ones(3, dtype=torch.float64)])


def test_the_workspace_is_what_the_header_asks_for():
    from conftest import REPO
    src = open(os.path.join(REPO, "include", "ctm_hip.h")).read()
    assert "#define CTM_GRAD_WS_DOUBLES(nt) (4 * (1089 + 16 * (nt)))" in src
    for nt in (0, 1, 300):
        assert HostEngine()._grad_ws(nt).numel() == 4 * (1089 + 16 * nt)


def test_tables_and_overlaps_of_lists(tmp_path):
    """csrc/grads_lists.h compiled by itself (lists_check.cpp): what the launches carry, and which calls are refused."""
    import subprocess
    from conftest import PKG, REPO
    exe = str(tmp_path / "lists_check")
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", os.path.join(PKG, "csrc"), os.path.join(REPO, "tests", "lists_check.cpp"),
                    "-o", exe], check=True, timeout=120)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.stdout, r.stderr[-2000:])


def test_optimizer_refusals():
    from optim.ad_optim_sgd_mod import SGD
    p = torch.zeros(3, dtype=torch.float64, requires_grad=True)
    for kw in (dict(lr=-1.0), dict(lr=1.0, momentum=-0.5), dict(lr=1.0, max_norm=-1.0), dict(lr=1.0, norm_type=1), dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            SGD([p], **kw)
    with pytest.raises(ValueError):
        SGD([dict(params=[p]), dict(params=[torch.zeros(2, dtype=torch.float64)])], lr=1.0)


# ---- the driver ----------------------------------------------------------------------------------------------------------------------------

class Env:
    def detach(self):
        return self


def run(tmp_path, module, device="cpu", dtype=torch.float64, epochs=4, target=1.0, resume=None, override=False, **opts):
    """optimize_state on a C4v state with a quadratic loss |a - target|^2 / 2: (losses, logged gradient norms, final tensor, start tensor)."""
    from ipeps.ipeps_c4v import IPEPS_C4V
    a0 = t64(2, 2, 2, 2, 2, seed=3, dtype=dtype)
    st = IPEPS_C4V(a0.clone().to(device))
    opt_args, main_args = copy.deepcopy(cfg.opt_args), copy.deepcopy(cfg.main_args)
    opt_args.tolerance_change = 0.0
    for k, v in opts.items():
        setattr(opt_args, k, v)
    main_args.opt_max_iter, main_args.out_prefix, main_args.opt_resume = epochs, os.path.join(str(tmp_path), "o"), resume
    main_args.opt_resume_override_params = override
    seen, lines = {}, []

    class Lines(logging.Handler):
        def emit(self, record):
            lines.append(json.loads(record.getMessage()))

    def loss_fn(state, env, ctx):
        d = state.site() - target
        return 0.5 * (d * d.conj()).real.sum(), env, [], 0.0, 0.0

    def post(state, env, ctx):
        seen["loss"] = list(ctx["loss_history"]["loss"])
    from optim import ad_optim_lbfgs_mod
    h, level = Lines(), ad_optim_lbfgs_mod.log.level
    ad_optim_lbfgs_mod.log.addHandler(h)
    ad_optim_lbfgs_mod.log.setLevel(logging.INFO)
    try:
        module.optimize_state(st, Env(), loss_fn, post_proc=post, main_args=main_args, opt_args=opt_args)
    finally:
        ad_optim_lbfgs_mod.log.removeHandler(h)
        ad_optim_lbfgs_mod.log.setLevel(level)
    return seen.get("loss", []), [l["grad_mag"] for l in lines if "grad_mag" in l], st.site().detach().cpu(), a0


def descent(a0, target, epochs, lr, mu=0.0, tau=0.0, bound=0.0):
    """The iteration of the driver's gradient descent on that loss (torch's gradient of a real loss of a complex tensor is d loss / d re + i d loss / d im)."""
    a, m, losses, mags = a0.clone(), None, [], []
    for _ in range(epochs):
        g = a - target
        losses.append(0.5 * float((g * g.conj()).real.sum()))
        n = float(torch.linalg.vector_norm(g))
        mags.append([n, float(g.abs().max())])
        if bound > 0.0 and n > bound:
            g = g * (bound / n)
        if mu:
            m = g.clone() if m is None else mu * m + (1 - tau) * g
            g = m
        a = a - lr * g
    return losses, mags, a


def check_descent(tmp_path, device, dtype):
    from optim import ad_optim_sgd_mod as S
    for kw in (dict(lr=0.5), dict(lr=0.25, momentum=0.5, dampening=0.25), dict(lr=0.5, momentum=0.9, clip_grad_norm=0.75)):
        losses, mags, a, a0 = run(tmp_path, S, device, dtype, **kw)
        wl, wm, wa = descent(a0, 1.0, 4, kw["lr"], kw.get("momentum", 0.0), kw.get("dampening", 0.0), kw.get("clip_grad_norm", 0.0))
        # (4 epochs of a few roundings each on values of order one)
        assert np.allclose(losses, wl, rtol=1e-13, atol=0) and np.allclose(mags, wm, rtol=1e-13, atol=0)
        assert float((a - wa).abs().max()) < 1e-13


@pytest.mark.parametrize("dtype", [torch.float64, torch.complex128])
def test_gradient_descent_of_a_state(host, tmp_path, dtype):
    check_descent(tmp_path, "cpu", dtype)


def test_gradient_descent_resumes(host, tmp_path):
    """A run that stops and resumes from its checkpoint walks on with its momentum: the checkpoint is written before each step."""
    from optim import ad_optim_sgd_mod as S
    from optim import ad_optim_lbfgs_mod as L
    kw = dict(lr=0.25, momentum=0.5, tolerance_grad=0.0)
    losses, *_ = run(tmp_path, S, epochs=3, **kw)
    ck = os.path.join(str(tmp_path), "o_checkpoint.p")
    saved = torch.load(ck, weights_only=False)
    buf = saved["optimizer_state_dict"]["state"][0]["momentum_buffer"]
    assert buf.shape == (2, 2, 2, 2, 2) and saved["loss"] == losses[-1]
    a0 = t64(2, 2, 2, 2, 2, seed=3)
    _, _, a, _ = run(tmp_path, S, epochs=1, resume=ck, **kw)
    assert float((a - (a0 - 0.25 * (0.5 * buf + (a0 - 1.0)))).abs().max()) < 1e-14
    torch.save(saved, ck)
    _, _, a, _ = run(tmp_path, S, epochs=1, resume=ck, override=True, lr=0.125, momentum=0.0, tolerance_grad=0.0)
    assert float((a - (a0 - 0.125 * (a0 - 1.0))).abs().max()) < 1e-14
    torch.save(saved, ck)
    with pytest.raises(RuntimeError, match="not a checkpoint of L-BFGS"):
        run(tmp_path, L, epochs=1, resume=ck)
    run(tmp_path, L, epochs=2, lr=0.5)
    with pytest.raises(RuntimeError, match="not a checkpoint of gradient descent"):
        run(tmp_path, S, epochs=1, resume=ck)


def test_line_searches_that_do_not_go_with_it(host, tmp_path):
    from optim import ad_optim_sgd_mod as S
    from optim import ad_optim_lbfgs_mod as L
    for ls in ("strong_wolfe", "backtracking"):
        with pytest.raises(RuntimeError, match="line search"):
            run(tmp_path, S, line_search=ls)
        with pytest.raises(RuntimeError, match="clip_grad_norm needs the fixed step"):
            run(tmp_path, L, line_search=ls, clip_grad_norm=1.0)


def test_bounded_gradients_of_lbfgs(host, tmp_path):
    """L-BFGS sees the scaled gradient, the log the gradient itself; a bound above the norm changes nothing."""
    from optim import ad_optim_lbfgs_mod as L
    free = run(tmp_path, L, lr=0.5, epochs=3)
    wide = run(tmp_path, L, lr=0.5, epochs=3, clip_grad_norm=1e6)
    assert free[0] == wide[0] and torch.equal(free[2], wide[2]) and np.allclose(free[1], wide[1], rtol=1e-14)
    tight = run(tmp_path, L, lr=0.5, epochs=1, clip_grad_norm=1e-3)
    g = tight[3] - 1.0
    n = float(torch.linalg.vector_norm(g))
    c = 1e-3 / n
    t = min(1.0, 1.0 / float((c * g).abs().sum())) * 0.5              # torch's first step of L-BFGS
    assert abs(tight[1][0][0] / n - 1) < 1e-14
    assert float((tight[2] - (tight[3] - t * c * g)).abs().max()) < 1e-14


def test_options_reach_the_driver():
    args = cfg.get_args_parser().parse_args(["--OPTARGS_clip_grad_norm", "0.5", "--OPTARGS_momentum", "0.9"])
    assert args.OPTARGS_clip_grad_norm == 0.5 and args.OPTARGS_momentum == 0.9
    assert cfg.OPTARGS().clip_grad_norm == 0.0
