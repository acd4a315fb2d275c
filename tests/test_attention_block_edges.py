"""qk_norm_rotate and diff_attention on the CPU: the oracle at the border of what the operators take."""
import pytest
import torch

from custom_d_fine_amd import kernels
from . import attention_block_ref as ref


def _heads(seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(*s, generator=g) for s in ((2, 5, 4, 2, 16), (2, 7, 2, 2, 16), (2, 7, 2, 32)))
    return [q, k, v, 0.2 * torch.randn(4, 4, 16, generator=g), 1 + 0.2 * torch.randn(32, generator=g)]


@pytest.mark.parametrize("eps", [0.0, 1e-60])
def test_oracle_rows_that_see_nothing_without_epsilon(oracle_backend, eps):
    args = [t.requires_grad_(True) for t in _heads()]
    mask = torch.zeros(5, 7, dtype=torch.bool)
    mask[2] = True
    y = kernels.diff_attention(*args[:4], 0.3, args[4], eps, attn_mask=mask, kv_lengths=torch.tensor([7, 0]))
    none = torch.zeros(2, 5, dtype=torch.bool)
    none[0, 2] = none[1] = True
    assert (y[none] == 0).all() and torch.isfinite(y).all()
    want = ref.diff_attention(*[t.detach().double() for t in args[:4]], 0.3, args[4].detach().double(), eps, ref.visible(2, 5, 7, mask, torch.tensor([7, 0])), 0.25)
    assert ref.rel(y[~none], want[~none]) < 512 * 2 ** -24
    for t in torch.autograd.grad(y.sum(), args):
        assert torch.isfinite(t).all()
