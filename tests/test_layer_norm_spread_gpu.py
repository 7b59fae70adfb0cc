"""Layer norm of rows whose values are all equal.  There x - mean is 0 whatever the size of the value, so y is the bias, the row adds nothing to the
weight's gradient, and dx is the centred gradient over sqrt(eps): each to the last bit or to a few steps, not up to the value's own rounding
times 1 / sqrt(eps) = 316."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}
VALUES = [4096.3, 60000.3, 250000.7, -1000000.3, 0.1, 1e9, -3.3e-3, 7.0]      # fp16 holds those below 65504, rounded to it
# a width in every variant: 1 to 1024 lanes with 1 to 4 vectors, 12 elements a lane, split rows
COLS = [3, 7, 12, 23, 36, 45, 72, 95, 144, 190, 333, 700, 1001, 1500, 2100, 3001, 4096, 5000, 6143, 7001, 9001, 13001, 20001, 31001, 40001, 100003]


@pytest.fixture(scope="module")
def N():
    from fdgan_hip import lib, norm
    lib.load()
    return norm


def rows(c, dtype):
    v = torch.tensor([v for v in VALUES if dtype != F16 or abs(v) < 65504]).to(dtype)
    return v[:, None].expand(len(v), c).contiguous()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("c", COLS)
def test_the_result_is_the_bias(N, c, dtype):
    g = torch.Generator().manual_seed(c)
    w, b = torch.randn(c, generator=g), torch.randn(c, generator=g)
    x = rows(c, dtype)
    y = N.layer_norm(x.to(DEV), c, w.to(DEV), b.to(DEV)).cpu()
    assert torch.equal(y, b.to(dtype).expand_as(y))
    if dtype == F32:                                              # a few steps of spread on a large mean
        k = torch.randint(0, 64, (5, c), generator=g).double()
        d = (k - k.mean(1, keepdim=True)) * 2.0 ** -8             # 60000's own step: x is exact
        s = 1.0 / (d.square().mean(1, keepdim=True) + 1e-5).sqrt()
        h = d * s
        got = N.layer_norm((60000.0 + k * 2.0 ** -8).float().to(DEV), c, None, None).cpu().double()
        # what the mean is off by: differences below 0.5 (0.25 and some steps that the first mean is off), summed in a tree of K(c); in split rows
        # (above 16384) the pieces' means and the row's are rounded to 60000's half step as well, 2^-9 each
        off = (64 + c / 64) * U * 0.5 + (2.0 ** -8 if c > 16384 else 0.0)
        assert ((got - h).abs() <= s * off + h.abs() * (s * off + (64 + c / 64) * U)).all()


def backward(N, x, dy, w, b):
    lv = [t.detach().to(DEV).requires_grad_(True) for t in (x, w, b)]
    return torch.autograd.grad(N.layer_norm(lv[0], x.shape[1], lv[1], lv[2]), lv, dy.to(DEV))


def check_gradients(c, dy, w, dx, dw, dt):
    assert not dw.cpu().any()
    s = 1.0 / 1e-5 ** 0.5
    g = dy.double() * w.double()
    want = s * (g - g.mean(1, keepdim=True))
    # the product, the mean (a sum of c terms in a tree: K(c) u), the difference, rstd and the product with it; then the type's own rounding
    bound = s * ((64 + c / 64) * U * g.abs().mean(1, keepdim=True) + 4 * U * g.abs()) + 8 * U * want.abs()
    rel = torch.finfo(dt).eps / 2
    assert ((dx.cpu().double() - want).abs() <= bound * (1 + rel) + rel * want.abs() + 1e-40).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("c", COLS)
def test_the_gradients(N, c, dtype):
    g = torch.Generator().manual_seed(c)
    w, b = torch.randn(c, generator=g), torch.randn(c, generator=g)
    x = rows(c, dtype)
    if dtype == F16:
        w = w * 2.0 ** -6                                         # 316 times a gradient has to stay below 65504
    x = x.repeat(7, 1)
    dy = torch.randn(x.shape, generator=g).to(dtype)
    dx, dw, db = backward(N, x, dy, w, b)
    check_gradients(c, dy, w, dx, dw, dtype)


def entry(N, x, dy, w, mean=None, rstd=None):
    """The C entries as a planned network calls them (weight gradients added to a sink); the statistics given, or the forward pass's own."""
    from fdgan_hip import lib as L
    lib = L.load()
    r, c = x.shape
    dt = {F32: L.FD_F32, F16: L.FD_F16, BF16: L.FD_BF16}
    view = lambda t: L.FdTensor(t.data_ptr(), r, 1, 1, c, (C.c_int64 * 4)(c, c, c, 1), dt[t.dtype], 0)  # noqa: E731
    xd, dyd, wd = x.to(DEV), dy.to(DEV), w.to(DEV)
    y, dx = torch.empty_like(xd), torch.empty_like(dyd)
    dw, db = torch.full((2, c), 3.0, device=DEV)
    fl = max(lib.fdgan_layer_norm_workspace(r, c, k) for k in (0, 1))
    ws = torch.empty(max(fl, 1), device=DEV)
    st = torch.cuda.current_stream().cuda_stream
    if mean is None:
        mean, rstd = torch.empty(2, r, device=DEV)
        L.check(lib.fdgan_layer_norm_fwd(view(xd), wd.data_ptr(), None, L.FD_F32, 1e-5, view(y), mean.data_ptr(), rstd.data_ptr(), ws.data_ptr(), fl, st))
    L.check(lib.fdgan_layer_norm_bwd(view(xd), view(dyd), wd.data_ptr(), L.FD_F32, mean.data_ptr(), rstd.data_ptr(), view(dx), dw.data_ptr(), db.data_ptr(), 1,
                                     ws.data_ptr(), fl, st))
    return dx, dw - 3.0


@pytest.mark.parametrize("c", [5, 72, 144, 1000, 2500, 13001])
def test_the_gradients_of_the_planned_form(N, c):
    """fp16 activations with bf16 gradients."""
    x = rows(c, F16).repeat(9, 1)
    g = torch.Generator().manual_seed(c)
    w = torch.randn(c, generator=g)
    dy = torch.randn(x.shape, generator=g).to(BF16)
    dx, dw = entry(N, x, dy, w)
    check_gradients(c, dy, w, dx, dw, BF16)


@pytest.mark.parametrize("c", COLS)
def test_values_whose_product_with_rstd_leaves_fp32(N, c):
    """2e36 / sqrt(1e-5) is beyond fp32: neither the elements that are there nor the empty places of the last vectors may form it."""
    for dtype in (F32, BF16):
        x = torch.full((11, c), 2e36).to(dtype)
        g = torch.Generator().manual_seed(c)
        w = torch.randn(c, generator=g)
        dy = torch.randn(x.shape, generator=g).to(dtype)
        mean, rstd = x[:, 0].float().to(DEV), torch.full((11,), 1e-5, dtype=torch.float64).rsqrt().float().to(DEV)
        dx, dw = entry(N, x, dy, w, mean, rstd)
        check_gradients(c, dy, w, dx, dw, dtype)
