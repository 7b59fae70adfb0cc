"""Adam's betas: what divides by 1 - beta^t is refused before a launch."""
import pytest
import torch

BAD = [(1.0, 0.999), (0.9, 1.0), (-0.1, 0.9), (0.9, -1e-9), (float("nan"), 0.9), (0.9, float("nan")), (2.0, 0.9)]


@pytest.mark.parametrize("betas", BAD)
def test_the_entries_refuse(betas):
    from fdgan_hip import lib as L
    lib = L.load()
    assert lib.fdgan_adam_step(4096, 4096, 4096, 4096, 8, 1e-3, *betas, 1e-8, 1, None) == L.FD_EINVAL
    assert lib.fdgan_last_error().startswith(b"adam_step: betas")
    assert lib.fdgan_adam_step_clipped(4096, 4096, 4096, 4096, 8, 1e-3, *betas, 1e-8, 1, 1.0, 4096, 9, 4096, None) == L.FD_EINVAL
    assert lib.fdgan_last_error().startswith(b"adam_step_clipped: betas")


@pytest.mark.gpu
@pytest.mark.parametrize("betas", BAD)
def test_the_python_entry_refuses(betas):
    from fdgan_hip import optim
    t = [torch.zeros(8, device="cuda:0") for _ in range(4)]
    for max_norm in (None, 1.0):
        with pytest.raises(ValueError, match="betas"):
            optim.adam_step_(*t, 1, 1e-3, betas, 1e-8, max_norm)


@pytest.mark.parametrize("betas", BAD)
def test_the_optimizer_refuses(betas):
    from fdgan_hip import optim
    with pytest.raises(ValueError, match="betas"):
        optim.FlatAdam([torch.nn.Parameter(torch.ones(4))], betas=betas)
