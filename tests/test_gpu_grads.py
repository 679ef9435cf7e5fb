"""The optimiser's operators over lists of tensors (optim/grads.py, csrc/grads.hip) against extended precision: norms, clipping, momentum step."""
import math
import numpy as np
import pytest
import torch
import grads_oracle as O
from optim import grads as G

pytestmark = pytest.mark.gpu
F64, C128 = torch.float64, torch.complex128
DTYPES = [F64, C128]
INF = float("inf")


def rand(shape, dtype, rng, scale=1.0):
    a = rng.standard_normal(shape)
    if dtype == C128:
        a = a + 1j * rng.standard_normal(shape)
    return a * scale


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(ts):
    return [t.detach().resolve_conj().resolve_neg().cpu().numpy() for t in ts]


def doubles(arrays):
    return sum(O.real_view(a).size for a in arrays)


def check_norms(got, arrays):
    n2, top = O.norms(arrays)
    cplx = any(a.dtype == np.complex128 for a in arrays)
    g2, gt = (float(v) for v in got)
    step = O.LD(2.0 ** -1074)                                         # (results below the normal range lie on this grid)
    assert abs(O.LD(g2) - n2) <= O.tol_n2(doubles(arrays)) * n2 + step, (g2, n2)
    assert abs(O.LD(gt) - top) <= O.tol_top(cplx) * top + (step if cplx else 0), (gt, top)
    return n2, top


def check_clip(outs, arrays, max_norm, norm_type, norms):
    n = norms[0] if norm_type == 2 else norms[1]
    # |c - exact| <= (error of the norm + 1 rounding), one more rounding per product
    tol = (O.tol_n2(doubles(arrays)) if norm_type == 2 else 3 * O.U) + 2 * O.U
    c = O.factor(n, max_norm)
    for o, a in zip(outs, arrays):
        want, have = O.real_view(a).astype(O.LD) * c, O.real_view(o).astype(O.LD)
        assert np.all(np.abs(have - want) <= tol * np.abs(want) + O.LD(2.0 ** -1074))
    return c


def check_step(p1, m1, p0, m0, g, c, ctol, lr, mu, tau, first):
    U = O.U
    for i in range(len(p0)):
        P, Gr = O.real_view(p0[i]).astype(O.LD), O.real_view(g[i]).astype(O.LD)
        d = c * Gr
        ed = (ctol + U) * np.abs(d)                                   # factor and product
        if mu != 0.0:
            if not first:
                M = O.real_view(m0[i]).astype(O.LD)
                a, b = O.LD(mu) * M, O.LD(1.0 - tau) * d
                d = a + b
                ed = U * np.abs(a) + ed * abs(1.0 - tau) + 2 * U * np.abs(b) + U * np.abs(d)
            have = O.real_view(m1[i]).astype(O.LD)
            assert np.all(np.abs(have - d) <= ed * (1 + 8 * U))
        want = P - O.LD(lr) * d
        have = O.real_view(p1[i]).astype(O.LD)
        assert np.all(np.abs(have - want) <= (lr * ed + U * lr * np.abs(d) + U * np.abs(want)) * (1 + 8 * U))


LISTS = {
    "one": [1], "empty_tensor": [0], "two": [2], "odd": [7], "loads": [511, 512, 513, 1023, 1024, 1025], "chunk": [2047, 2048, 2049],
    "chunks": [4095, 4096, 8191, 8193],
    "empties_between": [0, 5, 0, 0, 513, 0], "pieces": [127, 128, 129, 255], "one_group": [16384], "one_group_half": [8192], "one_group_quarter": [4096],
    "group_of_many": [256] * 63 + [255], "group_and_one": [16383, 1], "over_group": [16385], "cell_D4": [512] * 4, "cell_D8": [8192] * 8,
    "short_ones": [3] * 64, "table_full": [5] * 192 + [0] * 7, "table_over": [7] * 257, "several_tables": [(13 * i) % 97 + 1 for i in range(700)] + [30001], "many": [(37 * i) % 411 for i in range(300)], "long": [1 << 19, 3, 277777],
    "one_long": [1500001],
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(LISTS))
def test_norms_of_lists(eng, name, dtype):
    rng = np.random.default_rng(len(name))
    arrays = [rand(n, dtype, rng, 10.0 ** rng.uniform(-4, 2)) for n in LISTS[name]]
    ts = [dev(a) for a in arrays]
    got = G.grad_norms(ts)
    assert got.shape == (2,) and got.dtype == F64 and got.is_cuda
    check_norms(got, arrays)
    assert torch.equal(got, G.grad_norms(ts))                         # (fixed order of the sums)
    for t, a in zip(ts, arrays):
        assert np.array_equal(t.cpu().numpy(), a)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("norm_type,ratio,inplace", [(2, 0.25, True), (2, 0.25, False), (INF, 0.5, True), (INF, 0.125, False), (2, 2.0, True), (INF, 2.0, False)])
def test_clip_of_lists(eng, name, dtype, norm_type, ratio, inplace):
    rng = np.random.default_rng(len(name) + 100)
    arrays = [rand(n, dtype, rng, 10.0 ** rng.uniform(-4, 2)) for n in LISTS[name]]
    ts = [dev(a) for a in arrays]
    n2, top = O.norms(arrays)
    bound = float(ratio * (n2 if norm_type == 2 else top))
    if inplace:
        got = G.clip_grads(ts, bound, norm_type)
        outs = ts
    else:
        outs = [torch.full_like(t, 7.0) for t in ts]
        got = G.clip_grads(ts, bound, norm_type, out=outs)
        for t, a in zip(ts, arrays):
            assert np.array_equal(t.cpu().numpy(), a)
    norms = check_norms(got, arrays)
    check_clip(host(outs), arrays, bound, norm_type, norms)
    if ratio > 1.0:
        for t, a in zip(outs, arrays):
            assert np.array_equal(t.cpu().numpy(), a)                 # inside the bound: the same bits


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("mu,tau,first,max_ratio", [(0.0, 0.0, False, None), (0.0, 0.0, False, 0.3), (0.9, 0.0, False, 0.3), (0.8, 0.25, False, None),
                                                    (0.9, 0.5, True, 0.3), (0.5, 0.1, False, 3.0)])
def test_step_of_lists(eng, name, dtype, mu, tau, first, max_ratio):
    rng = np.random.default_rng(len(name) + 200)
    g = [rand(n, dtype, rng, 10.0 ** rng.uniform(-2, 1)) for n in LISTS[name]]
    p0, m0 = [rand(a.shape, dtype, rng) for a in g], [rand(a.shape, dtype, rng, 0.1) for a in g]
    ps, gs, ms = [dev(a) for a in p0], [dev(a) for a in g], [dev(a) for a in m0]
    norms = O.norms(g)
    bound = None if max_ratio is None else float(max_ratio * norms[0])
    v0 = [t._version for t in ps]
    got = G.sgd_step(ps, gs, ms if mu else None, lr=0.125, momentum=mu, dampening=tau, first=first, max_norm=bound)
    assert all(t._version > v for t, v in zip(ps, v0))                # (autograd and the corner cache see the write)
    if bound is None:
        assert got is None
    else:
        check_norms(got, g)
    c = O.LD(1) if bound is None else O.factor(norms[0], bound)
    check_step(host(ps), host(ms), p0, m0, g, c, 0.0 if c == 1 else O.tol_n2(doubles(g)) + O.U, 0.125, mu, tau, first)
    for t, a in zip(gs, g):
        assert np.array_equal(t.cpu().numpy(), a)
    if not mu:
        for t, a in zip(ms, m0):
            assert np.array_equal(t.cpu().numpy(), a)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1, 8])
def test_lists_longer_than_the_caches(eng, dtype, scale):
    """Whole numbers and factors of 1/2, so that every product and sum is exact: the results equal torch's bit for bit.  0.37 GB and 46 MB, of odd
    lengths at odd places."""
    u = 2 if dtype == C128 else 1
    lens = [35000003 // u // scale, 5, 9000001 // u // scale, 2048, 2300001 // u // scale]
    flat = torch.randint(-3, 4, (sum(lens) + 7, u), device="cuda", generator=torch.Generator("cuda").manual_seed(11)).to(F64)
    flat = torch.view_as_complex(flat) if u == 2 else flat[:, 0]
    cut = lambda t: list(t[1:1 + sum(lens)].split(lens))              # noqa: E731
    squares = sum(int((torch.view_as_real(t) if u == 2 else t).to(torch.int64).pow(2).sum()) for t in cut(flat))
    n2 = math.sqrt(squares)                                           # (sums of whole numbers below 2^53: exact in any order)
    top = 3.0 * math.sqrt(u)
    got = G.grad_norms(cut(flat)).tolist()
    assert got[0] == n2 and abs(got[1] / top - 1) <= O.tol_top(u == 2)
    out = torch.full_like(flat, 9.0)
    assert G.clip_grads(cut(flat), n2 / 2, out=cut(out)).tolist() == got
    assert torch.equal(torch.cat(cut(out)), torch.cat(cut(flat)) * 0.5)
    assert bool((out[:1] == 9.0).all()) and bool((out[1 + sum(lens):] == 9.0).all())
    p, m = flat.flip(0).contiguous(), (flat * 4).contiguous()
    wm = 0.5 * m + 0.75 * (0.5 * flat)
    wp = p - 0.25 * wm
    for t, w in ((wp, p), (wm, m)):
        t[:1], t[1 + sum(lens):] = w[:1], w[1 + sum(lens):]
    assert G.sgd_step(cut(p), cut(flat), cut(m), lr=0.25, momentum=0.5, dampening=0.25, max_norm=n2 / 2).tolist() == got
    assert torch.equal(p, wp) and torch.equal(m, wm)
    q = p.clone()
    G.sgd_step(cut(q), cut(flat), lr=0.25)
    wp = p - 0.25 * flat
    wp[:1], wp[1 + sum(lens):] = p[:1], p[1 + sum(lens):]
    assert torch.equal(q, wp)
    keep = flat.clone()
    G.clip_grads(cut(flat), n2 * 2)                                   # inside the bound
    assert torch.equal(flat, keep)
    G.clip_grads(cut(flat), n2 / 2)                                   # in place
    assert torch.equal(torch.cat(cut(out)), torch.cat(cut(flat)))


def test_offsets_past_32_bits(eng):
    """One tensor of more than 2^31 elements (17 GB): values at its end, at 2^31 elements and at 2^32 bytes."""
    n = (1 << 31) + 4099
    if torch.cuda.mem_get_info()[0] < 3 * 8 * n:
        pytest.skip("not enough free memory")
    x = torch.zeros(n, dtype=F64, device="cuda")
    at = torch.tensor([0, (1 << 29) - 1, 1 << 29, (1 << 30) + 1, (1 << 31) - 1, 1 << 31, n - 2, n - 1], device="cuda")
    x[at] = torch.tensor([1.0, -2.0, 3.0, 4.0, -5.0, 6.0, 7.0, 8.0], dtype=F64, device="cuda")
    n2 = math.sqrt(204.0)
    assert G.grad_norms([x]).tolist() == [n2, 8.0]
    g = x[at].clone()
    assert G.clip_grads([x], 4.0, INF).tolist() == [n2, 8.0]
    assert torch.equal(x[at], g * 0.5) and int(torch.count_nonzero(x)) == 8
    p = torch.zeros_like(x)
    G.sgd_step([p], [x], lr=2.0)
    assert torch.equal(p[at], -g) and int(torch.count_nonzero(p)) == 8
    del x, p
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_a_flat_buffer_and_what_lies_between_them(eng, dtype):
    """Tensors that start at every alignment and odd lengths in between: what lies between them keeps its bits."""
    rng = np.random.default_rng(3)
    lens = [1, 2, 3, 5, 1023, 1024, 1025, 2050, 17, 64, 65, 40001]
    offs, at = [], 1
    for n in lens:
        offs.append(at)
        at += n + 1 + (n % 3)
    flat = rand(at + 5, dtype, rng)
    views = lambda t: [t[o:o + n] for o, n in zip(offs, lens)]        # noqa: E731
    inside = np.zeros(flat.size, bool)
    for o, n in zip(offs, lens):
        inside[o:o + n] = True
    t = dev(flat)
    norms = check_norms(G.grad_norms(views(t)), views(flat))
    bound = float(norms[0]) / 3
    G.clip_grads(views(t), bound)
    check_clip(host(views(t)), views(flat), bound, 2, norms)
    assert np.array_equal(t.cpu().numpy()[~inside], flat[~inside])
    o = dev(np.full_like(flat, 9.0))
    src = dev(flat)
    G.clip_grads(views(src), bound, out=views(o))
    assert torch.equal(torch.cat(views(o)), torch.cat(views(t)))
    assert np.all(o.cpu().numpy()[~inside] == 9.0)
    p0, m0 = rand(flat.shape, dtype, rng), rand(flat.shape, dtype, rng)
    p, m = dev(p0), dev(m0)
    G.sgd_step(views(p), views(src), views(m), lr=0.5, momentum=0.75, max_norm=bound)
    c = O.factor(norms[0], bound)
    check_step(host(views(p)), host(views(m)), views(p0), views(m0), views(flat), c, O.tol_n2(2 * flat.size) + O.U, 0.5, 0.75, 0.0, False)
    assert np.array_equal(p.cpu().numpy()[~inside], p0[~inside]) and np.array_equal(m.cpu().numpy()[~inside], m0[~inside])


@pytest.mark.parametrize("dtype", DTYPES)
def test_orders_and_strides(eng, dtype):
    rng = np.random.default_rng(4)
    base = rand((6, 7, 5), dtype, rng)
    mk = [lambda t: t.permute(2, 0, 1), lambda t: t[:, 1:5], lambda t: t[::2, :, 1], lambda t: t[3, 2, 1], lambda t: t.transpose(0, 2)[1:4],
          lambda t: t[:, :, :0]]
    for f in mk:
        a = f(torch.from_numpy(base)).numpy()
        t = dev(base)
        v = f(t)
        other = dev(base * 2)
        norms = check_norms(G.grad_norms([v, other]), [a, base * 2])
        bound = float(norms[0]) / 2
        G.clip_grads([v, other], bound)
        c = check_clip([v.cpu().numpy(), other.cpu().numpy()], [a, base * 2], bound, 2, norms)
        want = torch.from_numpy(base.copy())
        f(want).mul_(float(c))
        assert np.abs(t.cpu().numpy() - want.numpy()).max() <= 1e-14 * np.abs(base).max()      # (the rest of the base tensor as it was)
        keep = torch.ones(base.shape, dtype=torch.bool)
        f(keep).fill_(False)
        assert np.array_equal(t.cpu().numpy()[keep.numpy()], base[keep.numpy()])
        # raw list kept, output in another order; step of a strided parameter with a gradient in another order
        src, out = dev(base), dev(base)
        G.clip_grads([f(src)], 0.5, out=[f(out)])
        check_clip([f(out).cpu().numpy()], [a], 0.5, 2, O.norms([a]))
        assert np.array_equal(src.cpu().numpy(), base) and np.array_equal(out.cpu().numpy()[keep.numpy()], base[keep.numpy()])
        p, m = dev(base), dev(base * 3)
        G.sgd_step([f(p)], [f(src).contiguous()], [f(m)], lr=0.25, momentum=0.5)
        check_step([f(p).cpu().numpy()], [f(m).cpu().numpy()], [a], [a * 3], [a], O.LD(1), 0.0, 0.25, 0.5, 0.0, False)
        assert np.array_equal(p.cpu().numpy()[keep.numpy()], base[keep.numpy()])
    # broadcast inputs count every element; conjugated and negated views hold their values
    e = dev(base[:1, :1]).expand(3, 4, 5)
    check_norms(G.grad_norms([e]), [np.broadcast_to(base[:1, :1], (3, 4, 5)).copy()])
    if dtype == C128:
        z = dev(base)
        for v, a in ((z.conj(), base.conj()), (z.conj().imag, -base.imag), (z.real, base.real)):
            check_norms(G.grad_norms([v]), [np.ascontiguousarray(a)])
            o = torch.empty(v.shape, dtype=v.dtype, device="cuda")
            G.clip_grads([v], 0.25, out=[o])
            w = v.clone()                                             # (keeps the flag of a conjugate)
            G.clip_grads([w], 0.25)
            check_clip(host([w]), [np.ascontiguousarray(a)], 0.25, 2, O.norms([np.ascontiguousarray(a)]))
            check_clip(host([o]), [np.ascontiguousarray(a)], 0.25, 2, O.norms([np.ascontiguousarray(a)]))


RANGES = {
    "zeros": [0.0, 0.0, -0.0], "tiny": [1e-300, 3e-305, -2e-300], "denormal": [5e-324, 1e-320, 0.0], "huge": [1e300, -3e300, 1e155],
    "huge_and_tiny": [1e200, 1e-200, 1.0], "middle_and_tiny": [1.0, 1e-170, 1e-310], "edge": [2.0 ** 480, 2.0 ** -480, 2.0 ** 479.9],
    "under_edge": [2.0 ** -481, 2.0 ** -480, 0.0], "near_overflow": [1.2e308, 1.2e308, 0.0],
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(RANGES))
@pytest.mark.parametrize("reps", [1, 100001])
def test_values_of_every_size(eng, name, dtype, reps):
    """No square overflows or underflows; a true norm beyond the largest double is infinite."""
    vals = np.array(RANGES[name] * reps)
    a = vals if dtype == F64 else (np.roll(vals, 1) * 0.5 + 1j * vals)
    if name == "near_overflow":
        a = a * (1e-4 if reps > 1 else 0.5)
    ts = [dev(a), dev(np.zeros(5, a.dtype))]
    n2, top = check_norms(G.grad_norms(ts), [a, np.zeros(5, a.dtype)])
    if n2 > 0:
        bound = float(n2) * 0.25
        G.clip_grads(ts, bound)
        # (a clipped denormal is rounded to its grid, and so is the bound)
        if n2 > 1e-300:
            check_clip(host(ts), [a, np.zeros(5, a.dtype)], bound, 2, (n2, top))
    else:
        G.clip_grads(ts, 0.0)
        assert all(np.array_equal(x, y) for x, y in zip(host(ts), [a, np.zeros(5, a.dtype)]))


def test_norm_beyond_the_largest_double(eng):
    a = np.full(1000, 1e308)
    assert G.grad_norms([dev(a)]).tolist() == [INF, 1e308]


@pytest.mark.parametrize("n", [3, 200003])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan(eng, n, dtype):
    rng = np.random.default_rng(5)
    for at in (0, n // 2, n - 1):
        a = rand(n, dtype, rng)
        a[at] = -np.inf
        t = [dev(rand(5, dtype, rng)), dev(a)]
        assert G.grad_norms(t).tolist() == [INF, INF]
        G.clip_grads(t, 1.0)                                          # c = 0
        h = t[1].cpu().numpy()
        assert np.isnan(h[at]) and np.all(np.delete(h, at) == 0) and np.all(t[0].cpu().numpy() == 0)
        a[at] = np.nan
        t = [dev(rand(5, dtype, rng)), dev(a)]
        assert all(math.isnan(v) for v in G.grad_norms(t).tolist())
        p = [dev(np.ones(5, a.dtype)), dev(np.ones(n, a.dtype))]
        got = G.sgd_step(p, t, lr=0.5, max_norm=1.0, norm_type=INF)
        assert all(math.isnan(v) for v in got.tolist())
        assert all(np.isnan(x).all() for x in host(p))
        p = [dev(np.ones(5, a.dtype)), dev(np.ones(n, a.dtype))]
        G.sgd_step(p, t, lr=0.5)                                      # no bound: the arithmetic of each element
        h = p[1].cpu().numpy()
        assert np.isnan(h[at]) and not np.isnan(np.delete(h, at)).any() and not np.isnan(p[0].cpu().numpy()).any()
        a[at - 1] = np.inf
        assert all(math.isnan(v) for v in G.grad_norms([dev(a)]).tolist())


def test_bounds_of_zero_and_infinity(eng):
    a = np.arange(1.0, 6.0)
    t = dev(a)
    G.clip_grads([t], INF)
    assert np.array_equal(t.cpu().numpy(), a)
    G.clip_grads([t], 0.0)
    assert np.array_equal(t.cpu().numpy(), 0 * a)
    G.clip_grads([t], 0.0)                                            # norm 0 <= 0
    assert np.array_equal(t.cpu().numpy(), 0 * a)
    assert G.grad_norms([]).tolist() == [0.0, 0.0] and G.clip_grads([], 1.0).tolist() == [0.0, 0.0]
    assert G.sgd_step([], [], lr=1.0) is None and G.sgd_step([], [], lr=1.0, max_norm=2.0).tolist() == [0.0, 0.0]


def test_the_same_tensor_twice(eng):
    a = np.arange(1.0, 6.0)
    t = dev(a)
    check_norms(G.grad_norms([t, t]), [a, a])
    p = [dev(a), dev(a * 2)]
    G.sgd_step(p, [t, t], lr=0.5)                                     # one gradient for two parameters
    assert np.array_equal(p[0].cpu().numpy(), a - 0.5 * a) and np.array_equal(p[1].cpu().numpy(), 1.5 * a)


def test_refusals(eng):
    import _native
    from _native import NativeError
    t, u, z = dev(np.ones(8)), dev(np.ones(8)), dev(np.ones(8) + 0j)
    h = torch.ones(8, dtype=F64)
    f = torch.ones(8, device="cuda")
    bad = [lambda: G.grad_norms([t, h]), lambda: G.grad_norms([f]), lambda: G.grad_norms([t, z]), lambda: G.grad_norms([t, None]),
           lambda: G.grad_norms([t.to_sparse()]), lambda: G.clip_grads([t], -1.0), lambda: G.clip_grads([t], float("nan")),
           lambda: G.clip_grads([t], 1.0, norm_type=1), lambda: G.clip_grads([t], 1.0, out=[]), lambda: G.clip_grads([t], 1.0, out=[u[:7]]),
           lambda: G.clip_grads([t, t], 0.5), lambda: G.clip_grads([t[:5], t[4:]], 0.5), lambda: G.clip_grads([t, u], 0.5, out=[u, t]),
           lambda: G.clip_grads([t[:4]], 0.5, out=[t[2:6]]), lambda: G.clip_grads([t[:1].expand(3)], 0.5), lambda: G.clip_grads([z], 0.5, out=[torch.ones_like(z).conj()]),
           lambda: G.clip_grads([t[0:6:2], t[1:7:2]], 0.5),
           lambda: G.sgd_step([t], [u], lr=-1.0), lambda: G.sgd_step([t], [u], momentum=0.5), lambda: G.sgd_step([t], [u, u]),
           lambda: G.sgd_step([t], [t]), lambda: G.sgd_step([t], [u], [t], momentum=0.5), lambda: G.sgd_step([t], [u], [u], momentum=0.5),
           lambda: G.sgd_step([t, t], [u, u]), lambda: G.sgd_step([t], [z]), lambda: G.sgd_step([t], [u], max_norm=-2.0),
           lambda: G.sgd_step([t], [u], momentum=float("nan"), bufs=[u])]
    for i, call in enumerate(bad):
        with pytest.raises(NativeError):
            call()
            print("not refused:", i)
    # the C entries by themselves
    import ctypes as C
    e = _native.engine()
    e._bind_dtype(F64)
    ws = torch.empty(4 * 1105, dtype=F64, device="cuda")
    n = (C.c_longlong * 1)(8)
    pt = e._ptrs([t])
    lib, vp = e.lib, C.c_void_p
    assert lib.ctm_grad_norms(e.h, None, -1, pt, n, vp(ws.data_ptr()), ws.numel()) == 1
    assert lib.ctm_grad_norms(e.h, None, 1, None, n, vp(ws.data_ptr()), ws.numel()) == 1
    assert lib.ctm_grad_norms(e.h, None, 1, pt, n, vp(ws.data_ptr()), ws.numel() - 1) == 1
    assert lib.ctm_grad_norms(e.h, None, 1, pt, n, None, ws.numel()) == 1
    assert lib.ctm_grad_norms(e.h, None, 1, pt, (C.c_longlong * 1)(-8), vp(ws.data_ptr()), ws.numel()) == 1
    assert lib.ctm_grad_norms(e.h, None, 1, pt, (C.c_longlong * 1)(1 << 50), vp(ws.data_ptr()), ws.numel()) == 1
    assert lib.ctm_grad_norms(e.h, None, 1, (vp * 1)(t.data_ptr() + 4), n, vp(ws.data_ptr()), ws.numel()) == 1
    assert lib.ctm_grad_clip(e.h, None, 1, pt, pt, n, 1, 1.0, vp(ws.data_ptr()), ws.numel()) == 1
    assert lib.ctm_sgd_step(e.h, None, 1, pt, e._ptrs([u]), None, n, 0.5, 0.9, 0.0, 0, 2, -1.0, None, 0) == 1
    assert lib.ctm_grad_norms(None, None, 1, pt, n, vp(ws.data_ptr()), ws.numel()) == 1
    assert np.array_equal(t.cpu().numpy(), np.ones(8)) and np.array_equal(u.cpu().numpy(), np.ones(8))


def test_another_stream_and_two_at_once(eng):
    """Calls run on the current stream, each with a workspace of its own: two lists clipped at the same time on two streams."""
    rng = np.random.default_rng(6)
    lists = [[rand(n, F64, rng) for n in (300001, 5, 77)], [rand(n, F64, rng, 100.0) for n in (400003, 9)]]
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        ts = [[dev(a) for a in l] for l in lists]
        torch.cuda.synchronize()
        got = []
        for k in (0, 1):
            with torch.cuda.stream(s[k]):
                got.append(G.clip_grads(ts[k], 1.0))
        torch.cuda.synchronize()
        for k in (0, 1):
            check_clip(host(ts[k]), lists[k], 1.0, 2, check_norms(got[k], lists[k]))
    with torch.cuda.stream(s[0]):                                     # in order with the work of its own stream
        x = torch.zeros(3000000, dtype=F64, device="cuda")
        for _ in range(20):
            x.add_(1.0)
        got = G.grad_norms([x])
        x.zero_()
    torch.cuda.synchronize()
    assert got.tolist() == [20.0 * math.sqrt(3000000.0), 20.0] or abs(got[0].item() / (20.0 * math.sqrt(3e6)) - 1) < 1e-14


@pytest.mark.parametrize("lens", [[32], [512] * 4, [100003, 7, 4096, 1]])
def test_captured_and_replayed(eng, lens):
    """Graphs of the whole sequence: each replay reads the values of its time, with eager calls between the replays."""
    rng = np.random.default_rng(7)
    mk = lambda k=1.0: [rand(n, C128, rng, k) for n in lens]          # noqa: E731
    p0, m0, g0 = mk(), mk(), mk()
    side = torch.cuda.Stream()
    ps, ms, gs, outs = [dev(a) for a in p0], [dev(a) for a in m0], [dev(a) for a in g0], [dev(0 * a) for a in g0]
    torch.cuda.synchronize()

    def body():
        a = G.grad_norms(gs)
        b = G.clip_grads(gs, 0.5, INF, out=outs)
        c = G.sgd_step(ps, outs, ms, lr=0.25, momentum=0.5, max_norm=0.75)
        return a, b, c
    with torch.cuda.stream(side):
        body()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            res = body()
        graphs.append((gr, res))
    for k in range(6):
        p, m, g = host(ps), host(ms), mk(10.0 ** (k - 2))
        for t, a in zip(gs, g):
            t.copy_(dev(a))
        gr, res = graphs[k % 2]
        gr.replay()
        torch.cuda.synchronize()
        na, nb, nc = (r.clone() for r in res)
        norms = check_norms(na, g)
        assert torch.equal(na, nb)
        check_clip(host(outs), g, 0.5, INF, norms)
        o = host(outs)
        no = check_norms(nc, o)
        check_step(host(ps), host(ms), p, m, o, O.factor(no[0], 0.75), O.tol_n2(doubles(o)) + O.U, 0.25, 0.5, 0.0, False)
        # eager work between the replays, on other data
        assert torch.equal(G.grad_norms([dev(a) for a in g]), na)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mu,tau,max_norm", [(0.0, 0.0, None), (0.9, 0.0, 0.5), (0.6, 0.25, None)])
def test_optimizer_follows_torch(eng, dtype, mu, tau, max_norm):
    """A run of them together, as an optimisation uses them: backward, norms, bounded momentum step; against torch's own SGD after torch's clipping."""
    from optim.ad_optim_sgd_mod import SGD
    rng = np.random.default_rng(8)
    init = [rand(s, dtype, rng) for s in ((2, 3, 3, 3, 3), (2, 2, 4, 2, 4), (5,))]
    mine, ref = [dev(a).requires_grad_() for a in init], [torch.from_numpy(a.copy()).requires_grad_() for a in init]
    opt = SGD(mine, lr=0.05, momentum=mu, dampening=tau, max_norm=max_norm)
    topt = torch.optim.SGD(ref, lr=0.05, momentum=mu, dampening=tau)

    def loss(ps, opt):
        opt.zero_grad()
        l = sum(0.5 * (p.abs() ** 2).sum() + 0.02 * (p.abs() ** 4).sum() for p in ps)
        l.backward()
        return l
    for _ in range(6):
        opt.step(lambda: loss(mine, opt))
        loss(ref, topt)
        if max_norm is not None:
            n = torch.sqrt(sum((p.grad.abs() ** 2).sum() for p in ref))
            assert abs(opt.norms[0].item() / n.item() - 1) < 1e-12
            for p in ref:
                p.grad.mul_(min(1.0, max_norm / n.item()))
        topt.step()
        for a, b in zip(mine, ref):
            # six steps, each with at most 8 roundings and twice the bound of the norm (< 130 half steps in all), of an iteration that enlarges a
            # difference at most tenfold (lr times the largest curvature, 0.05 x 6, is far inside its stable range): 6 x 130 x 10 U < 1e-12
            assert (a.detach().cpu() - b.detach()).abs().max() <= 1e-12 * b.abs().max()
    sd = opt.state_dict()
    opt2 = SGD(mine, lr=0.05, momentum=mu, dampening=tau, max_norm=max_norm)
    opt2.load_state_dict(sd)
    assert (mu == 0.0) == (len(opt2.state) == 0)


def test_a_parameter_that_joins_later(eng):
    """Parameters on their first step next to others: the factor is that of all gradients."""
    from optim.ad_optim_sgd_mod import SGD
    rng = np.random.default_rng(9)
    a, b = dev(rand(7, F64, rng)).requires_grad_(), dev(rand(9, F64, rng)).requires_grad_()
    opt = SGD([a, b], lr=0.5, momentum=0.5, dampening=0.25, max_norm=1.0)
    a.grad = dev(rand(7, F64, rng))
    opt.step()
    a.grad, b.grad = dev(rand(7, F64, rng, 3.0)), dev(rand(9, F64, rng, 3.0))
    p0, m0, g = host([a, b]), host([opt.state[a]["momentum_buffer"]]), host([a.grad, b.grad])
    opt.step()
    n = O.norms(g)
    check_norms(opt.norms, g)
    c = O.factor(n[0], 1.0)
    tol = O.tol_n2(16) + 2 * O.U
    ms = host([opt.state[t]["momentum_buffer"] for t in (a, b)])
    check_step(host([a]), ms[:1], p0[:1], m0, g[:1], c, tol, 0.5, 0.5, 0.25, False)
    check_step(host([b]), ms[1:], p0[1:], [None], g[1:], c, tol, 0.5, 0.5, 0.25, True)
    assert np.array_equal(host([a.grad])[0], g[0])


def test_clip_grad_norm_of_parameters(eng):
    rng = np.random.default_rng(10)
    ps = [dev(rand((3, 4), F64, rng)).requires_grad_() for _ in range(3)]
    g = [rand((3, 4), F64, rng), None, rand((3, 4), F64, rng)]
    for p, a in zip(ps, g):
        p.grad = None if a is None else dev(a)
    got = G.clip_grad_norm_(ps, 0.5)
    norms = check_norms(got, [g[0], g[2]])
    check_clip(host([ps[0].grad, ps[2].grad]), [g[0], g[2]], 0.5, 2, norms)
    assert ps[1].grad is None


def test_a_written_tensor_is_noticed_by_autograd(eng):
    x = dev(np.ones(4)).requires_grad_()
    y = (x * x).sum()
    G.sgd_step([x], [dev(np.ones(4))], lr=0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()




@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_descent_of_a_state_on_the_engine(eng, tmp_path, dtype):
    from test_grads_host import check_descent
    check_descent(tmp_path, "cuda", dtype)


def test_bounded_gradients_of_lbfgs_on_the_engine(eng, tmp_path):
    from test_grads_host import run
    from optim import ad_optim_lbfgs_mod as L
    free = run(tmp_path, L, "cuda", lr=0.5, epochs=3)
    wide = run(tmp_path, L, "cuda", lr=0.5, epochs=3, clip_grad_norm=1e6)
    assert free[0] == wide[0] and torch.equal(free[2], wide[2]) and free[1] == wide[1]
    tight = run(tmp_path, L, "cuda", lr=0.5, epochs=1, clip_grad_norm=1e-3)
    g = tight[3] - 1.0
    n = float(torch.linalg.vector_norm(g))
    c = 1e-3 / n
    t = min(1.0, 1.0 / float((c * g).abs().sum())) * 0.5              # torch's first step of L-BFGS
    assert abs(tight[1][0][0] / n - 1) < 1e-13 and float((tight[2] - (tight[3] - t * c * g)).abs().max()) < 1e-13


@pytest.mark.parametrize("script,extra", [("optim_j1j2_c4v.py", ["--optimizer", "sgd", "--OPTARGS_momentum", "0.5"]),
                                          ("optim_j1j2.py", ["--optimizer", "sgd", "--tiling", "BIPARTITE"]),
                                          ("optim_j1j2_c4v.py", ["--GLOBALARGS_dtype", "complex128"])])
def test_optimisation_commands(tmp_path, script, extra):
    """The commands with gradient descent and with bounded gradients: they run their epochs, log the norms of the gradients and leave state and
    checkpoint behind; a momentum step is no longer than lr times the bound over 1 - momentum."""
    import json, os, subprocess, sys
    from conftest import PKG
    env = dict(os.environ, PYTHONPATH=PKG + os.pathsep + os.environ.get("PYTHONPATH", ""))
    pre = str(tmp_path / "o")
    lr, bound = 0.05, 0.01
    args = [sys.executable, os.path.join(PKG, "examples", "j1j2", script), "--bond_dim", "2", "--chi", "8", "--opt_max_iter", "3", "--seed", "123",
            "--CTMARGS_ctm_max_iter", "6", "--GLOBALARGS_device", "cuda:0", "--out_prefix", pre, "--OPTARGS_lr", str(lr), "--OPTARGS_clip_grad_norm", str(bound)]
    r = subprocess.run(args + extra, capture_output=True, text=True, env=env, timeout=110)
    assert r.returncode == 0, r.stderr[-3000:]
    lines = [json.loads(l[l.index("{"):]) for l in open(pre + ".log") if "grad_mag" in l]
    assert len(lines) == 3 and all(l["grad_mag"][0] >= l["grad_mag"][1] > 0 for l in lines)
    assert os.path.exists(pre + "_state.json")
    ck = torch.load(pre + "_checkpoint.p", weights_only=False, map_location="cpu")
    group = ck["optimizer_state_dict"]["param_groups"][0]
    if "sgd" in extra:
        assert group["lr"] == lr and group["max_norm"] == bound
        if "--OPTARGS_momentum" in extra:
            m = torch.cat([s["momentum_buffer"].reshape(-1) for s in ck["optimizer_state_dict"]["state"].values()])
            assert float(torch.linalg.vector_norm(m)) <= bound / (1 - 0.5) * (1 + 1e-12)
    else:
        assert "history_size" in group
