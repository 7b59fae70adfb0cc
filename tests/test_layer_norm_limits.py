"""Layer norm at the limits of what one call takes: refused on the host beyond them, right up to them."""
import ctypes as C

import pytest
import torch

DEV = "cuda:0"


def view(rows, c, dtype, ptr):
    from fdgan_hip import lib as L
    return L.FdTensor(ptr, rows, 1, 1, c, (C.c_int64 * 4)(c, c, c, 1), dtype, 0)


def test_more_pieces_than_a_launch_holds_are_refused():
    from fdgan_hip import lib as L
    lib = L.load()
    room = 1 << 62
    for rows, c, dt in ((1 << 24, 16385, L.FD_F32), (1 << 22, 16385, L.FD_F32), (1 << 30, 1 << 20, L.FD_F16), (1 << 40, 1 << 29, L.FD_F32)):
        x, y, dx = (view(rows, c, dt, 1 << k) for k in (40, 50, 60))
        assert lib.fdgan_layer_norm_fwd(x, None, None, 1, 1e-5, y, None, None, 4096, room, None) == L.FD_EINVAL
        assert b"too many" in lib.fdgan_last_error()
        assert lib.fdgan_layer_norm_bwd(x, y, None, 1, 4096, 4096, dx, 4096, 4096, 0, 4096, room, None) == L.FD_EINVAL
        assert b"too many" in lib.fdgan_last_error()
    for backward in (0, 1):
        assert lib.fdgan_layer_norm_workspace(1 << 40, 1 << 29, backward) < 0 and lib.fdgan_layer_norm_workspace(1 << 30, 1 << 20, backward) < 0
        assert lib.fdgan_layer_norm_workspace(1 << 30, 1000, backward) >= 0            # held rows: any number
    assert lib.fdgan_layer_norm_workspace(1 << 23, 20000, 0) >= 0                      # 16-bit rows of that length are held, fp32 ones are not


@pytest.mark.gpu
@pytest.mark.parametrize("c", [(1 << 24) + 24, (1 << 26) + 8])
def test_weight_gradients_of_the_widest_rows(c):
    """Two columns sums of each of 2^24 and more values: more than one turn of the joining pass."""
    from fdgan_hip import norm
    g = torch.Generator(device=DEV).manual_seed(c)
    x, dy = (torch.randn(2, c, generator=g, device=DEV, dtype=torch.float16) for _ in range(2))
    w, b = torch.ones(c, device=DEV, requires_grad=True), torch.zeros(c, device=DEV, requires_grad=True)
    dw, db = torch.autograd.grad(norm.layer_norm(x, c, w, b), (w, b), dy)
    assert torch.equal(db, dy[0].float() + dy[1].float())
    m = x.double().mean(1, keepdim=True)
    h = (x.double() - m) / (x.double().var(1, correction=0, keepdim=True) + 1e-5).sqrt()
    want = (dy.double() * h).sum(0)
    # the mean of 2^26 values of size 1, in a tree over pieces: 40 steps of 2^-24 of their mean size; rstd and the products a few steps each
    bound = 2.0 ** -24 * (dy.double().abs() * (40.0 + 48.0 * h.abs())).sum(0)
    assert ((dw.double() - want).abs() <= bound).all()
