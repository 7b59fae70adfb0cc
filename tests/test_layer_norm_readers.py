"""A planned layer norm whose source has other readers: every reader's part reaches the source's gradient, whichever comes first in the plan; a source that a later
op overwrites is refused (the reverse walk reads it again)."""
import pytest
import torch

DEV = "cuda:0"


def plan_of(dev, order, c, c0, pitch, n=2, h=6, w=5):
    """source `a` -> layer norm -> `y`, and copies of a -> `b` (whole groups of eight channels) where `order` says so."""
    from fdgan_hip import engine as E
    from fdgan_hip.netplan import NetPlan
    from fdgan_hip.norm import LayerNorm
    P = NetPlan(torch.device(dev))
    a, y, b, z = E.new_act(n, h, w, pitch, dev, zero=True), *(E.new_act(n, h, w, (c + 7) // 8 * 8, dev, zero=True) for _ in range(3))
    ln = LayerNorm(c).to(dev)
    src, wide = E.View(a, c0, c), E.View(a, c0, (c + 7) // 8 * 8)
    for op in order:
        if op == "norm":
            P.layer_norm(src, E.View(y, 0, c), ln)
        elif op == "read":
            P.copy(wide, E.View(b))
        elif op == "read elsewhere":
            P.copy(E.View(z), E.View(b))
        elif op == "overwrite":
            P.copy(E.View(z), wide)
    return P, ln, a, y, b


def test_who_stores_and_what_is_refused():
    from fdgan_hip.backward import layer_norm_sources
    for order, want in ((["norm"], [True]), (["norm", "read"], [False]), (["read", "norm"], [False]), (["norm", "read elsewhere"], [True]),
                        (["norm", "norm"], [False, False]), (["overwrite", "read", "norm"], [False]), (["read", "overwrite", "norm"], [True]),
                        (["read elsewhere"], [])):
        P = plan_of("cpu", order, 16, 0, 16)[0]
        assert list(layer_norm_sources(P.records).values()) == want, order
    for order in (["norm", "overwrite"], ["norm", "read", "overwrite"]):
        with pytest.raises(NotImplementedError, match="overwrites"):
            layer_norm_sources(plan_of("cpu", order, 16, 0, 16)[0].records)


def gradient64(a, ln, dy):
    x = a.double().requires_grad_(True)
    w, b = (p.detach().cpu().double().requires_grad_(True) for p in (ln.weight, ln.bias))
    torch.nn.functional.layer_norm(x, (a.shape[-1],), w, b, 1e-5).backward(dy.double())
    return x.grad, w.grad, b.grad


@pytest.mark.gpu
@pytest.mark.parametrize("order", [["norm"], ["norm", "read"], ["read", "norm"]], ids="-".join)
@pytest.mark.parametrize("c,c0,pitch", [(16, 0, 16), (20, 0, 24), (20, 8, 40)])
def test_every_reader_adds_its_part(order, c, c0, pitch):
    from fdgan_hip import engine as E
    from fdgan_hip.backward import PlanBackward
    from fdgan_hip.optim import FlatAdam
    P, ln, a, y, b = plan_of(DEV, order, c, c0, pitch)
    FlatAdam(ln.parameters())                              # from the third walk on a recorded tape
    P.finish()
    B = PlanBackward(P)
    cc = b.shape[-1]
    for k in range(5):
        g = torch.Generator().manual_seed(k)
        rnd = lambda t, ch, dt: torch.randn(t.shape[:3] + (ch,), generator=g).to(dt)  # noqa: E731
        va, dy, db = rnd(a, c, torch.float16), rnd(y, c, torch.bfloat16), rnd(b, cc, torch.bfloat16)
        a[..., c0:c0 + c] = va.to(DEV)
        P.main.launch()                                    # (no conv in this plan: no filter image to refresh)
        B.zero_()
        gs = B.G(E.View(a)).buf
        B.G(E.View(y)).buf[..., :c] = dy.to(DEV)
        if "read" in order:
            B.G(E.View(b)).buf.copy_(db)
        ln.weight.grad.zero_(), ln.bias.grad.zero_()
        B.run({})
        torch.cuda.synchronize()
        dx, dw, dbias = gradient64(va, ln, dy)
        dx = torch.nn.functional.pad(dx, (0, cc - c))
        want = dx + (db.double() if "read" in order else 0.0)
        got = gs.cpu().double()
        # dx rounded to bf16, the sum once more; fp32 sums of 20 terms in between are below a hundredth of that
        assert ((got[..., c0:c0 + cc] - want).abs() <= 1.01 * 2.0 ** -8 * (dx.abs() + want.abs()) + 1e-5).all(), k
        assert not got[..., :c0].any() and not got[..., c0 + cc:].any()
        assert torch.allclose(ln.weight.grad.cpu().double(), dw, rtol=1e-5, atol=1e-4) and torch.allclose(ln.bias.grad.cpu().double(), dbias, rtol=1e-5, atol=1e-4)
    assert any(t is not None for t in B.tapes.values())


@pytest.mark.gpu
def test_a_network_head_that_reads_the_source(c=16):
    """A conv outside the plan (a network's last one) on the same source: its part comes first in the walk and stays."""
    from fdgan_hip import engine as E
    from fdgan_hip.backward import PlanBackward
    P, ln, a, y, _ = plan_of(DEV, ["norm"], c, 0, c)
    g = torch.Generator().manual_seed(7)
    filt = torch.nn.Parameter((0.1 * torch.randn(8, c, 3, 3, generator=g)).to(DEV))
    w = P.weight(filt, 8, c, 3)
    P.finish()
    va, dy, dh = (torch.randn(2, 6, 5, k, generator=g) for k in (c, c, 8))
    va, dy, dh = va.half(), dy.bfloat16(), dh.bfloat16()
    a.copy_(va)
    P.launch()
    B = PlanBackward(P)
    head = dict(x=E.View(a), w=w, k=3, pad=1, stride=1, bias=None, pro=None)
    seed = dh.to(DEV).contiguous()
    for _ in range(3):
        B.zero_()
        B.G(E.View(y)).buf.copy_(dy)
        B.run({}, head=(head, E.View(seed)))
        torch.cuda.synchronize()
        got = B.G(E.View(a)).buf.cpu().double()
        dx = gradient64(va, ln, dy)[0]
        part = torch.nn.functional.conv_transpose2d(dh.double().permute(0, 3, 1, 2), filt.detach().cpu().bfloat16().double(), padding=1).permute(0, 2, 3, 1)
        want = dx + part
        # bf16 filters and gradients as they are; the head's part is rounded to bf16, dx too, and the sum again
        assert ((got - want).abs() <= 1.01 * 2.0 ** -8 * (dx.abs() + part.abs() + want.abs()) + 1e-4).all()
