"""csrc/qknorm.hip through kernels.qk_norm_rotate against a 64-bit restatement.

Tolerances, in the 2-norm.  32-bit arithmetic: every result is a product of about 8 roundings (sum of squares over D <= 256 terms in a tree of at most
8 + 5 levels, rsqrt 2, four products, one sum), each at most 2^-24: 32 * 2^-24.  bf16 results add one rounding, 2^-8.  Weight gradients are 32-bit sums
over n rows in a tree / serial runs of at most n / 16 + 64 terms: their error grows like the root of the run at random signs, at most
(32 + 4 sqrt(n)) * 2^-24, against sums whose terms have random signs too."""
import pytest
import torch

from . import attention_block_ref as ref

pytestmark = pytest.mark.gpu


def _case(cuda, B, L, Hq, Hk, D, R, dtype, interleaved, T=None, seed=0):
    g = torch.Generator().manual_seed(seed + B + L + D)
    q = torch.randn(B, L, Hq, D, generator=g).to(dtype).to(cuda)
    k = torch.randn(B, L, Hk, D, generator=g).to(dtype).to(cuda)
    wq, wk = (1 + 0.3 * torch.randn(D, generator=g)).to(cuda), (1 + 0.3 * torch.randn(D, generator=g)).to(cuda)
    T = T or L + 3
    angle = torch.rand(T, R // 2, generator=g, dtype=torch.float64) * 20 - 10
    return q, k, wq, wk, angle.cos().float().to(cuda), angle.sin().float().to(cuda), g


def _tol(dtype, n=0):
    t = (32 + 4 * n ** 0.5) * 2 ** -24
    return t + (2 ** -8 if dtype == torch.bfloat16 else 0)


def _check(cuda, q, k, wq, wk, cos, sin, positions, eps, interleaved, g):
    from custom_d_fine_amd import kernels
    dtype = q.dtype
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, wq, wk)]
    yq, yk = kernels.qk_norm_rotate(*leaves, cos, sin, positions, eps, interleaved)
    rows = torch.arange(q.shape[1], device=cuda) if positions is None else positions.long()
    dl = [t.detach().double().requires_grad_(True) if t is not None else None for t in (q, k, wq, wk)]
    rq = ref.norm_rotate(dl[0], dl[2], cos, sin, rows, eps, interleaved)
    rk = ref.norm_rotate(dl[1], dl[3], cos, sin, rows, eps, interleaved)
    assert yq.dtype == dtype and yq.shape == q.shape and yq.is_contiguous()
    assert ref.rel(yq, rq) <= _tol(dtype) and ref.rel(yk, rk) <= _tol(dtype)
    gq = torch.randn(q.shape, generator=g).to(dtype).to(cuda)
    gk = torch.randn(k.shape, generator=g).to(dtype).to(cuda)
    got = torch.autograd.grad([yq, yk], [t for t in leaves if t is not None], [gq, gk])
    want = torch.autograd.grad([rq, rk], [t for t in dl if t is not None], [gq.double(), gk.double()])
    for name, a, b in zip(("dq", "dk", "dwq", "dwk"), got, want):
        n = q.shape[0] * q.shape[1] * max(q.shape[2], k.shape[2])
        tol = _tol(dtype) if name in ("dq", "dk") else _tol(a.dtype, n)
        assert a.dtype == b.dtype or a.dtype in (torch.float32, torch.bfloat16)
        assert ref.rel(a, b) <= tol, name
    with torch.no_grad():                                        # the call without gradients gives the same bits
        zq, zk = kernels.qk_norm_rotate(q, k, wq, wk, cos, sin, positions, eps, interleaved)
    assert torch.equal(zq, yq) and torch.equal(zk, yk)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,L,Hq,Hk,D,R", [(1, 1, 1, 1, 8, 8), (2, 7, 4, 2, 16, 8), (3, 5, 3, 1, 24, 24), (1, 65, 8, 8, 32, 32), (2, 33, 6, 3, 40, 16),
                                           (2, 100, 5, 5, 64, 64), (1, 31, 2, 1, 80, 80), (4, 9, 40, 8, 96, 48), (1, 17, 7, 3, 128, 128),
                                           (1, 12, 3, 2, 200, 104), (2, 3, 2, 2, 256, 256)])
def test_against_64_bits(cuda, dtype, interleaved, B, L, Hq, Hk, D, R):
    q, k, wq, wk, cos, sin, g = _case(cuda, B, L, Hq, Hk, D, R, dtype, interleaved)
    _check(cuda, q, k, wq, wk, cos, sin, None, 1e-6, interleaved, g)


@pytest.mark.parametrize("per_sequence,kind", [(True, torch.int64), (True, torch.int32), (False, torch.int64)])
def test_positions(cuda, per_sequence, kind):
    q, k, wq, wk, cos, sin, g = _case(cuda, 3, 20, 4, 2, 48, 32, torch.bfloat16, True, T=1000)
    p = torch.randint(0, 1000, (3, 20) if per_sequence else (20,), generator=g).to(kind).to(cuda)
    _check(cuda, q, k, wq, wk, cos, sin, p, 1e-5, True, g)


def test_many_tokens_and_weights_of_either_type(cuda):
    q, k, wq, wk, cos, sin, g = _case(cuda, 3, 5001, 6, 3, 32, 32, torch.bfloat16, False)
    _check(cuda, q, k, wq.bfloat16(), None, cos, sin, None, 1e-6, False, g)
    _check(cuda, q, k, None, wk, cos, sin, None, 1e-6, False, g)


def test_strides_and_alignment(cuda):
    """Slices of a packed projection, [B, H, L, D] order, a view that starts off a 16-byte border, expanded gradients."""
    from custom_d_fine_amd import kernels
    B, L, H, D = 2, 37, 4, 32
    g = torch.Generator().manual_seed(5)
    packed = torch.randn(B, L, 3 * H * D, generator=g).bfloat16().to(cuda)
    angle = torch.rand(L, D // 2, generator=g) * 6
    cos, sin = angle.cos().to(cuda), angle.sin().to(cuda)
    q, k = packed[..., :H * D].view(B, L, H, D), packed[..., H * D:2 * H * D].view(B, L, H, D)
    base = kernels.qk_norm_rotate(q.contiguous(), k.contiguous(), None, None, cos, sin)
    flat = torch.empty(B * L * H * D + 8, device=cuda, dtype=torch.bfloat16)
    off = flat[3:3 + q.numel()].view(q.shape).copy_(q)
    for qq in (q, q.transpose(1, 2).contiguous().transpose(1, 2), off, torch.stack([q, q], -1)[..., 0]):
        y = kernels.qk_norm_rotate(qq, k, None, None, cos, sin)
        assert torch.equal(y[0], base[0]) and torch.equal(y[1], base[1])
    ql = q.detach().requires_grad_(True)
    kernels.qk_norm_rotate(ql, None, None, None, cos, sin)[0].sum().backward()
    qd = q.double().requires_grad_(True)
    ref.norm_rotate(qd, None, cos, sin, torch.arange(L, device=cuda), 1e-6, False).sum().backward()
    assert ref.rel(ql.grad, qd.grad) <= _tol(torch.bfloat16)


def test_no_rotation_no_keys_and_empty(cuda):
    from custom_d_fine_amd import kernels
    g = torch.Generator().manual_seed(9)
    q = torch.randn(2, 5, 3, 24, generator=g).to(cuda)
    y, none = kernels.qk_norm_rotate(q, None)
    assert none is None and ref.rel(y, ref.norm_rotate(q.double(), None, None, None, None, 1e-6, False)) <= _tol(torch.float32)
    w = torch.ones(24, device=cuda, requires_grad=True)
    e = torch.empty(2, 0, 3, 24, device=cuda, requires_grad=True)
    z, _ = kernels.qk_norm_rotate(e, None, w)
    assert z.shape == e.shape
    z.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and e.grad.shape == e.shape


def test_position_outside_the_table_is_nan_there_only(cuda):
    from custom_d_fine_amd import kernels
    q, k, wq, wk, cos, sin, g = _case(cuda, 1, 6, 2, 1, 32, 16, torch.float32, False, T=8)
    p = torch.tensor([0, 7, 8, -1, 3, 2 ** 40], device=cuda)
    y, _ = kernels.qk_norm_rotate(q, k, wq, wk, cos, sin, p)
    bad = torch.tensor([False, False, True, True, False, True], device=cuda)
    assert torch.isnan(y[0, bad][..., :16]).all() and torch.isfinite(y[0, ~bad]).all() and torch.isfinite(y[0, bad][..., 16:]).all()


def test_zero_rows_and_large_values(cuda):
    from custom_d_fine_amd import kernels
    q = torch.zeros(1, 3, 1, 16, device=cuda)
    q[0, 1] = 1e15
    y, _ = kernels.qk_norm_rotate(q.requires_grad_(True), None)
    assert torch.equal(y[0, 0], torch.zeros_like(y[0, 0])) and torch.allclose(y[0, 1], torch.ones_like(y[0, 1]))
    (dq,) = torch.autograd.grad(y.sum(), q)
    assert torch.isfinite(dq).all()


def test_captured_replay_equals_eager(cuda):
    from custom_d_fine_amd import kernels
    q, k, wq, wk, cos, sin, g = _case(cuda, 2, 50, 4, 2, 64, 64, torch.bfloat16, False)
    go = torch.randn(q.shape, generator=g).bfloat16().to(cuda)
    ql, kl, wl = q.clone().requires_grad_(True), k.clone().requires_grad_(True), wq.clone().requires_grad_(True)

    def step():
        yq, yk = kernels.qk_norm_rotate(ql, kl, wl, wk, cos, sin)
        return (yq, yk) + torch.autograd.grad([yq, yk], [ql, kl, wl], [go, torch.ones_like(yk)])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            ql.copy_(torch.randn(q.shape, generator=g).to(cuda))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
