"""The verification of drafted tokens on the GPU over the whole range of logits and temperatures that it accepts."""
import pytest
import torch

from test_gpu_verify_drafts import check, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature,top", [(1.0, 1e10), (1.0, -1e10), (1.0, 2.7e9), (0.7, 6e9), (1e-3, 1e7), (1e-4, 1.5e6), (1e-4, 1048577.0), (1.2e-4, 81920.0), (1e4, 1e14), (1e4, -3e38), (1.0, 3e38), (1e4, 1e10), (1.0, 1e7), (0.5, -3e6)])
@pytest.mark.parametrize("with_draft", [False, True])
def test_neighbours_of_large_logits(pkg, temperature, top, with_draft):
    """Logits far from 0, where neighbouring numbers lie up to some thousand temperatures apart: what the distance leaves weighs what it should, and the rest nothing."""
    g, S, K, V = gen(5), 6, 2, 700
    steps = torch.randint(0, 5, (S, K + 1, V), device="cuda", generator=g)
    x = torch.full((S, K + 1, V), top, device="cuda")
    below = torch.tensor(float("-inf"), device="cuda")
    for i in range(1, 5):  # 0 to 4 numbers below the largest
        x = torch.where(steps >= i, torch.nextafter(x, below), x)
    x[:, :, 3] = top
    x[:3, :, 100:] = 0.5 * top if top > 0 else 1.1 * top  # (finite: 1.1 * 3e38 is)
    y = x[:, :K].flip(2).contiguous() if with_draft else None
    drafts = torch.randint(0, V, (S, K), device="cuda", generator=g).int()
    drafts[::2, 0] = 3
    for seed in range(3):
        check(pkg, x, drafts, torch.rand(S, K + 1, device="cuda", generator=g), y, temperature)
    check(pkg, x[:, :1], drafts[:, :0], torch.rand(S, 1, device="cuda", generator=g), None, temperature)
    only = torch.full((2, 1, 50), float("-inf"), device="cuda")  # the largest and its neighbour alone
    only[:, :, 7] = top
    only[:, :, 8] = torch.nextafter(only[:, :, 7], below)
    check(pkg, only, drafts[:2, :0], torch.tensor([[0.2], [0.999]], device="cuda"), None, temperature)


@pytest.mark.parametrize("temperature", [1e-50, -1e-50, 1e-46, 5e-324, 1e-45, 9e-5, 1.1e4, 1e300])
def test_temperatures_that_are_refused(pkg, temperature):
    """Also those that FP32 rounds to 0: they are not 0, and most likely tokens are not what was asked for."""
    x, u = torch.zeros(1, 2, 8, device="cuda"), torch.zeros(1, 2, device="cuda")
    with pytest.raises(pkg.native.B200Error, match="temperature"):
        pkg.verify_drafts(x, torch.zeros(1, 1, device="cuda", dtype=torch.int32), u, temperature=temperature)
