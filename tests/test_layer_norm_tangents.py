"""Forward-mode derivatives are refused: a tangent must not be dropped on the way."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD


def refuses(dev):
    from fdgan_hip import norm
    x, w, b = torch.randn(4, 8, device=dev), torch.randn(8, device=dev), torch.randn(8, device=dev)
    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(x), w, b), (x, dual(w), b), (x, w, dual(b)), (dual(x), None, None)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                norm.layer_norm(args[0], 8, args[1], args[2])
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                norm.layer_norm(args[0], 8, args[1], args[2])
        with pytest.raises(RuntimeError, match="forward-mode"):
            norm.layer_norm(dual(x.clone().requires_grad_(True)), 8, w, b)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: norm.layer_norm(t, 8, w, b), (x,), (torch.ones_like(x),))
    return norm, x, w, b


def test_refused_on_the_cpu():
    refuses("cpu")


@pytest.mark.gpu
def test_refused_on_the_gpu():
    norm, x, w, b = refuses("cuda:0")
    assert norm.layer_norm(x, 8, w, b).shape == x.shape            # the same tensors without tangents
