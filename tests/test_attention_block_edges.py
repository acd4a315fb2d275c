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


def test_oracle_what_is_hidden_may_hold_anything(oracle_backend):
    """Keys that no query sees and queries that see no key: no value, no gradient."""
    mask = torch.rand(5, 7, generator=torch.Generator().manual_seed(3)) < 0.3
    mask[2] = mask[:, 4] = True
    lens = torch.tensor([6, 5])
    dy = torch.randn(2, 5, 4, 32, generator=torch.Generator().manual_seed(4))

    def run(args, dy):
        args = [t.detach().clone().requires_grad_(True) for t in args]
        y = kernels.diff_attention(*args[:4], 0.3, args[4], attn_mask=mask, kv_lengths=lens)
        return (y.detach(),) + torch.autograd.grad(y, args, dy)

    args = _heads()
    clean = run(args, dy)
    for t, what in ((args[1], float("nan")), (args[2], float("inf"))):
        t[0, 6:] = t[1, 5:] = t[:, 4] = what
    args[0][:, 2] = dy[:, 2] = float("nan")
    for a, b in zip(clean, run(args, dy)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_position_outside_the_table_is_nan_there_only(oracle_backend, interleaved):
    g = torch.Generator().manual_seed(1)
    q, angle = torch.randn(1, 6, 2, 32, generator=g), torch.rand(8, 8, generator=g)
    p = torch.tensor([0, 7, 8, -1, 3, 2 ** 40])
    y, _ = kernels.qk_norm_rotate(q, None, None, None, angle.cos(), angle.sin(), p, interleaved=interleaved)
    bad = torch.tensor([False, False, True, True, False, True])
    assert torch.isnan(y[0, bad][..., :16]).all() and torch.isfinite(y[0, ~bad]).all() and torch.isfinite(y[0, bad][..., 16:]).all()
    z, _ = kernels.qk_norm_rotate(q[:, ~bad], None, None, None, angle.cos(), angle.sin(), p[~bad], interleaved=interleaved)
    assert torch.equal(y[:, ~bad], z)


@pytest.mark.parametrize("N,M", [(5, 0), (0, 7)])
def test_oracle_without_keys_or_queries(oracle_backend, N, M):
    args = [torch.randn(*s, requires_grad=True) for s in ((2, N, 4, 2, 16), (2, M, 2, 2, 16), (2, M, 2, 32), (4, 16), (32,))]
    y = kernels.diff_attention(*args[:4], 0.3, args[4])
    assert y.shape == (2, N, 4, 32) and (y == 0).all()
    for t in torch.autograd.grad(y.sum(), args):
        assert (t == 0).all()
