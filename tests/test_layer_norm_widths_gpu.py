"""Layer norm where its rows are no whole vectors inside a padded buffer (the discriminator with few filters), and the split backward pass with many rows a
workgroup."""
import pytest
import torch

from test_layer_norm_critic_gpu import plain_d, rel
from test_layer_norm_gpu import BF16, DEV, F16, F32, NAMES, compare, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nf", [3, 5, 10, 13, 22])
def test_discriminator_with_few_filters(nf):
    """2 nf and 4 nf channels in buffers of whole groups of eight: forward and all gradients against the network in plain torch, with operands rounded
    where the kernels round them; bounds of the test at 36 filters."""
    import models.dehaze1113 as net
    from fdgan_hip import lib
    from hiputil import emulate_kernel_operands
    lib.load()
    torch.manual_seed(nf)
    ref = plain_d(9, nf)
    with torch.no_grad():
        for n, p in ref.named_parameters():
            if ".ln." in n:
                p.add_(0.2 * torch.randn_like(p))
    d = net.D(9, nf, norm="layer")
    d.load_state_dict(ref.state_dict())
    d = d.to(DEV)
    g = torch.Generator().manual_seed(2)
    x = torch.rand(2, 9, 48, 40, generator=g) * 2 - 1
    cot = torch.rand(2, 1, 22, 18, generator=g) * 2 - 1
    with torch.no_grad():
        y, want = d(x.to(DEV)).cpu(), ref(x.clone())
    assert float((y - want).abs().max()) < 2e-2 and rel(y, want) < 1e-2
    emulate_kernel_operands(ref)
    xo, xg = x.clone().requires_grad_(True), x.to(DEV).requires_grad_(True)
    (ref(xo) * cot).sum().backward()
    for _ in range(2):
        d.zero_grad()
        xg.grad = None
        (d(xg) * cot.to(DEV)).sum().backward()
        got = {"x": rel(xg.grad.cpu(), xo.grad)}
        for (n, p), q in zip(d.named_parameters(), ref.parameters()):
            got[n] = rel(p.grad.cpu(), q.grad)
        assert len(got) == 10 and max(got.values()) < 5e-2, got


@pytest.mark.parametrize("r,c,dtype", [(3001, 6500, F32), (2309, 13000, F16), (2307, 16385, BF16)], ids=lambda v: NAMES.get(v, str(v)) if isinstance(v, torch.dtype) else str(v))
def test_split_backward_with_many_rows_a_workgroup(r, c, dtype):
    """rows x pieces above 9216: more than eight rows a workgroup, the last one fewer."""
    from fdgan_hip import norm
    x, dy, w, b = make(r, c, dtype, F32)
    compare(run(norm, x.to(DEV), dy.to(DEV), w.to(DEV), b.to(DEV)), reference(x, dy, w, b, 1e-5), dtype, F32)
