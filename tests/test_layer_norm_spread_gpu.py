"""Layer norm of rows whose values are all equal.  There x - mean is 0 whatever the size of the value, so y is the bias, the row adds nothing to the
weight's gradient, and dx is the centred gradient over sqrt(eps): each to the last bit or to a few steps, not up to the value's own rounding
times 1 / sqrt(eps) = 316."""
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
