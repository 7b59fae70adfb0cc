"""Adam's constants: 1 - beta and 1 - beta^t are those of the betas as they are passed (64 bits), not of betas rounded to fp32 first -- 1 - 0.999 would
come out 1.3e-5 of itself too small, and with it every new term of the second moment."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32 = torch.float32


@pytest.fixture(scope="module")
def O():  # noqa: E743
    from fdgan_hip import lib, optim
    lib.load()
    return optim


def adam64(p, g, m, v, t, lr, betas, eps, max_norm):
    b1, b2 = betas
    g = g.double()
    n = float(g.square().sum().sqrt())
    if max_norm is not None:
        g = g * min(1.0, max_norm / (n + 1e-6))
    m = b1 * m.double() + (1 - b1) * g
    v = b2 * v.double() + (1 - b2) * g * g
    d = lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
    return p.double() - d, m, v, d


# one workgroup, two launches, past the caches; a last group that is not whole
@pytest.mark.parametrize("n", [1, 2, 3, 4, 7, 1023, 1025, 4097, 8191, 8192, 8193, 16389, 70001, 790416, 9000001])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.5, 0.999), (0.95, 0.9999), (0.0, 0.99)])
@pytest.mark.parametrize("max_norm", [None, 1e9, 0.25, 0.0])
def test_one_step(O, n, betas, max_norm):
    gen = torch.Generator().manual_seed(n)
    p, g, m = (torch.randn(n, generator=gen) * s for s in (0.1, 0.3, 0.01))
    v = torch.rand(n, generator=gen) * 10.0 ** -torch.randint(3, 9, (n,), generator=gen).float()       # g * g above v and below it
    for t in (1, 7, 1000, 100000):
        d = [a.to(DEV) for a in (p, g, m, v)]
        O.adam_step_(*d, t, 1e-3, betas, 1e-8, max_norm)
        pw, mw, vw, dw = adam64(p, g, m, v, t, 1e-3, betas, 1e-8, max_norm)
        # m: each beta constant, product and sum a rounding of its term (3u), the factor 6u more; v: the new term 4u and the factor twice.  The
        # step: half of v's and all of m's errors, the bias corrections' roundings, and its own quotients, root, sum and products: 24u
        e_m = 10 * U * (betas[0] * m.double().abs() + (mw - betas[0] * m.double()).abs()) + 1e-45
        e_v = 18 * U * vw + 1e-45
        off = lambda got, ref: (got.cpu().double() - ref).abs()  # noqa: E731
        assert (off(d[2], mw) <= e_m).all() and (off(d[3], vw) <= e_v).all()
        den = (vw / (1 - betas[1] ** t)).sqrt() + 1e-8
        assert (off(d[0], pw) <= U * pw.abs() + 24 * U * dw.abs() + 1e-3 * (e_m / (1 - betas[0] ** t)) / den + 1e-40).all()


def test_a_bound_that_is_not_reached_changes_no_bit(O):
    for n in (5, 8191, 70003):
        gen = torch.Generator().manual_seed(n)
        a = [(torch.randn(n, generator=gen) * s).to(DEV) for s in (0.1, 0.3, 0.01)] + [torch.rand(n, generator=gen).to(DEV) * 1e-4]
        b = [t.clone() for t in a]
        for t in range(1, 4):
            O.adam_step_(*a, t, 1e-3, (0.9, 0.999), 1e-8)
            O.adam_step_(*b, t, 1e-3, (0.9, 0.999), 1e-8, 1e9)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_against_torch(O):
    """torch.optim.Adam on the CPU, several steps: both round each step's quotient of 1e-3 a few times."""
    gen = torch.Generator().manual_seed(1)
    p = torch.randn(1000, generator=gen)
    ref = torch.nn.Parameter(p.clone())
    opt = torch.optim.Adam([ref], lr=1e-3, betas=(0.5, 0.999), eps=1e-8)
    d = [p.to(DEV)] + [torch.zeros(1000, device=DEV) for _ in range(3)]
    for t in range(1, 9):
        g = torch.randn(1000, generator=gen) * 10.0 ** (t % 3 - 1)
        ref.grad = g.clone()
        opt.step()
        d[1].copy_(g)
        O.adam_step_(*d, t, 1e-3, (0.5, 0.999), 1e-8)
        v = opt.state[ref]["exp_avg_sq"].double()
        assert ((d[3].cpu().double() - v).abs() <= 2 * t * 8 * U * v).all()      # either side: up to 4 roundings a step
        assert float((d[0].cpu() - ref.detach()).abs().max()) <= t * (2 * U * 4.0 + 64 * U * 1e-3 * 10)


def test_an_optimizer_without_a_bound_needs_the_library_alone(O, monkeypatch):
    """FlatAdam(max_norm=None) is one entry of the library: it steps where the torch module is not there."""
    from fdgan_hip import lib as L

    def gone():
        raise L.FdganLibraryError("libfdgan_torch.so not found")
    ps = [torch.nn.Parameter(torch.randn(5, 3, device=DEV)), torch.nn.Parameter(torch.randn(7, device=DEV))]
    twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = O.FlatAdam(ps, lr=1e-2), O.FlatAdam(twin, lr=1e-2, max_norm=1e9)
    for opt in (a, b):
        opt.grad.copy_(torch.linspace(-1, 1, opt.grad.numel(), device=DEV))
    b.step()
    monkeypatch.setattr(L, "torch_ops", gone)
    version = ps[0]._version
    a.step()
    assert a.grad_norm is None and ps[0]._version > version
    assert torch.equal(a.flat, b.flat) and torch.equal(a.m, b.m) and torch.equal(a.v, b.v)
    assert b.grad_norm is not None
    b.max_norm = None                                      # the bound is taken off: no norm of an earlier step stays behind
    b.step()
    assert b.grad_norm is None
