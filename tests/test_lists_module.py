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
