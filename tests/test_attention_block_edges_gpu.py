"""Calls of qk_norm_rotate and diff_attention at the border of what they take: no epsilon under rows that see nothing, derivatives and traces that go past the
autograd functions, channels that the rotation leaves alone."""
import pytest
import torch

from . import attention_block_ref as ref
from .test_diff_attention_gpu import EPS, INIT, _inputs, _off, _tol

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


# one run of the keys, runs that are joined, many rows
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,M,H,Hk,d,dv", [(2, 70, 140, 6, 3, 32, 64), (3, 3, 3000, 8, 2, 64, 128), (16, 130, 130, 8, 8, 16, 32)])
@pytest.mark.parametrize("eps", [0.0, 1e-60])                        # (1e-60: 0 in 32 bits)
def test_rows_that_see_nothing_without_epsilon(cuda, dtype, eps, B, N, M, H, Hk, d, dv):
    from custom_d_fine_amd import kernels
    q, k, v, lam, w, dy, g = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
    mask = torch.rand(N, M, generator=g) < 0.3
    mask[::3] = True
    mask = mask.to(cuda)
    lens = torch.full((B,), M, device=cuda)
    lens[-1] = 0
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam, w)]
    y = kernels.diff_attention(*leaves[:4], INIT, norm_weight=leaves[4], norm_eps=eps, attn_mask=mask, kv_lengths=lens)
    grads = torch.autograd.grad(y, leaves, dy)
    seen = ref.visible(B, N, M, mask, lens, device=cuda)
    none = ~seen.any(2)
    assert (y[none] == 0).all() and (grads[0][none] == 0).all()
    assert all(torch.isfinite(t).all() for t in grads)
    full = [t.double() for t in (q, k, v, lam)]
    want = ref.diff_attention(*full, INIT, w.double(), eps, seen, d ** -0.5)
    spread = ref.diff_attention_spread(*full, INIT, w.double(), EPS, seen, d ** -0.5, dy.double())["out"]
    assert _off(y[~none], want[~none], spread) <= _tol("out", dtype, M, d)
    with torch.no_grad():                                            # no key at all
        y = kernels.diff_attention(q, k, v, lam, INIT, w, eps, attn_mask=torch.ones(N, M, dtype=torch.bool, device=cuda))
        z = kernels.diff_attention(q, k[:, :0], v[:, :0], lam, INIT, w, eps)
    assert (y == 0).all() and (z == 0).all()


def _norm_inputs(cuda):
    g = torch.Generator().manual_seed(4)
    q, k = torch.randn(2, 5, 4, 16, generator=g).to(cuda), torch.randn(2, 5, 2, 16, generator=g).to(cuda)
    wq, wk = (1 + 0.2 * torch.randn(16, generator=g)).to(cuda), (1 + 0.2 * torch.randn(16, generator=g)).to(cuda)
    angle = torch.rand(5, 4, generator=g)
    return [q, k, wq, wk, angle.cos().to(cuda), angle.sin().to(cuda)]


def test_forward_mode_derivatives_are_refused(cuda):
    """An operand with a tangent is refused, with and without gradients; without one a call inside a dual level is as it is outside."""
    import torch.autograd.forward_ad as fw

    from custom_d_fine_amd import kernels
    heads = list(_inputs(cuda, 1, 9, 9, 6, 6, 16, 32, torch.float32)[:5])
    attend = lambda q, k, v, lam, w: kernels.diff_attention(q, k, v, lam, INIT, norm_weight=w)  # noqa: E731
    for call, args in ((attend, heads), (lambda *a: kernels.qk_norm_rotate(*a)[0], _norm_inputs(cuda))):
        base = call(*args)
        with fw.dual_level():
            assert torch.equal(call(*args), base)
            for at in range(len(args)):
                dual = [fw.make_dual(t, torch.ones_like(t)) if j == at else t for j, t in enumerate(args)]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*dual)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*dual)
        assert torch.equal(call(*args), base)


def test_traces_are_refused(cuda):
    from custom_d_fine_amd import kernels
    q, k, v, lam, w, _, _ = _inputs(cuda, 1, 9, 9, 6, 6, 16, 32, torch.float32)
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(lambda x: kernels.diff_attention(x, k, v, lam, INIT, w), (q,), check_trace=False)
    args = _norm_inputs(cuda)
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(lambda x: kernels.qk_norm_rotate(x, *args[1:])[0], (args[0],), check_trace=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_channels_that_pass_know_nothing_of_their_neighbours(cuda, dtype, what):
    """Channels from 8 on are not rotated: what channel 12 holds, its weight or its gradient, stays out of channel 13, in either order of the pairs."""
    from custom_d_fine_amd import kernels
    q, _, w, _, cos, sin = _norm_inputs(cuda)
    q = q.to(dtype)
    others = [c for c in range(16) if c != 12]
    for interleaved in (True, False):
        base = kernels.qk_norm_rotate(q, None, w, None, cos, sin, interleaved=interleaved)[0]
        bad = w.clone()
        bad[12] = what
        y = kernels.qk_norm_rotate(q, None, bad, None, cos, sin, interleaved=interleaved)[0]
        assert torch.equal(y[..., others], base[..., others]) and not torch.isfinite(y[..., 12]).any()
        wl = w.clone().requires_grad_(True)
        dy = torch.ones_like(base)
        dy[..., 12] = what
        (dw,) = torch.autograd.grad(kernels.qk_norm_rotate(q, None, wl, None, cos, sin, interleaved=interleaved)[0], wl, dy)
        assert torch.isfinite(dw[others]).all() and not torch.isfinite(dw[12])
    x = q.clone()
    x[..., 12] = float("inf")                                         # a norm of 1 / infinity: the head's other channels are 0
    y = kernels.qk_norm_rotate(x, None, None, None, cos, sin, interleaved=True)[0]
    assert (y[..., others] == 0).all()
