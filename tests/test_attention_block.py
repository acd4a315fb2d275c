"""qk_norm_rotate and diff_attention on the CPU: what they refuse, and their oracle against the 64-bit restatement and differences."""
import pytest
import torch

from custom_d_fine_amd import kernels
from . import attention_block_ref as ref


def _qk():
    return torch.randn(2, 5, 4, 16), torch.randn(2, 5, 2, 16), torch.randn(9, 4), torch.randn(9, 4)


@pytest.mark.parametrize("change,kind", [
    (dict(q=torch.randn(2, 5, 4, 12)), ValueError), (dict(q=torch.randn(2, 5, 64)), ValueError), (dict(q=torch.randn(2, 5, 4, 264)), ValueError),
    (dict(q=torch.randn(2, 5, 4, 16).half()), TypeError), (dict(k=torch.randn(2, 5, 2, 16).bfloat16()), TypeError), (dict(k=torch.randn(2, 6, 2, 16)), ValueError),
    (dict(q_weight=torch.ones(8)), ValueError), (dict(q_weight=torch.ones(16).double()), TypeError), (dict(k=None, k_weight=torch.ones(16)), ValueError),
    (dict(sin=None), ValueError), (dict(cos=torch.randn(9, 3), sin=torch.randn(9, 3)), ValueError), (dict(cos=torch.randn(9, 12), sin=torch.randn(9, 12)), ValueError),
    (dict(cos=torch.randn(4, 4), sin=torch.randn(4, 4)), ValueError), (dict(cos=torch.randn(9, 4).bfloat16()), TypeError),
    (dict(cos=torch.randn(9, 4, requires_grad=True)), ValueError), (dict(positions=torch.zeros(2, 4, dtype=torch.int64)), ValueError),
    (dict(positions=torch.zeros(2, 5)), TypeError), (dict(cos=None, sin=None, positions=torch.zeros(5, dtype=torch.int64)), ValueError), (dict(eps=-1.0), ValueError)])
def test_qk_norm_rotate_refuses(oracle_backend, change, kind):
    q, k, cos, sin = _qk()
    with pytest.raises(kind, match="qk_norm_rotate"):
        kernels.qk_norm_rotate(**{**dict(q=q, k=k, cos=cos, sin=sin), **change})


def _diff():
    return dict(q=torch.randn(2, 5, 4, 2, 16), k=torch.randn(2, 7, 2, 2, 16), v=torch.randn(2, 7, 2, 32), lambda_vectors=torch.randn(4, 4, 16) * 0.1, lambda_init=0.3)


@pytest.mark.parametrize("change,kind", [
    (dict(q=torch.randn(2, 5, 4, 16)), ValueError), (dict(q=torch.randn(2, 5, 3, 2, 16)), ValueError), (dict(q=torch.randn(2, 5, 4, 2, 20)), ValueError),
    (dict(k=torch.randn(3, 7, 2, 2, 16)), ValueError), (dict(k=torch.randn(2, 7, 2, 2, 16).bfloat16()), TypeError), (dict(v=torch.randn(2, 6, 2, 32)), ValueError),
    (dict(v=torch.randn(2, 7, 2, 136)), ValueError), (dict(v=torch.randn(2, 7, 2, 12)), ValueError), (dict(lambda_vectors=torch.randn(4, 2, 16)), ValueError),
    (dict(lambda_vectors=torch.randn(4, 4, 16).double()), TypeError), (dict(norm_weight=torch.ones(16)), ValueError),
    (dict(attn_mask=torch.zeros(5, 7)), TypeError), (dict(attn_mask=torch.zeros(7, 5, dtype=torch.bool)), ValueError),
    (dict(kv_lengths=torch.tensor([1.0, 2.0])), TypeError), (dict(kv_lengths=torch.tensor([1, 2, 3])), ValueError), (dict(query_start=3), ValueError),
    (dict(query_start=torch.tensor([1, 2])), ValueError), (dict(causal=True, query_start=2 ** 40), ValueError), (dict(scale=0.0), ValueError),
    (dict(scale=-1.0), ValueError), (dict(scale=1e-31), ValueError), (dict(scale=float("nan")), ValueError), (dict(norm_eps=-1.0), ValueError)])
def test_diff_attention_refuses(oracle_backend, change, kind):
    with pytest.raises(kind, match="diff_attention"):
        kernels.diff_attention(**{**_diff(), **change})


def test_wide_heads_are_refused(oracle_backend):
    with pytest.raises(ValueError, match="multiples of 8"):
        kernels.diff_attention(torch.randn(1, 2, 1, 2, 72), torch.randn(1, 2, 1, 2, 72), torch.randn(1, 2, 1, 8), torch.randn(4, 72), 0.1)


def test_no_cpu_kernels():
    q, k, cos, sin = _qk()
    with pytest.raises(RuntimeError, match="HIP kernel"):
        kernels.qk_norm_rotate(q, k, cos=cos, sin=sin)
    with pytest.raises(RuntimeError, match="HIP kernel"):
        kernels.diff_attention(**_diff())


def test_c_entries_refuse_without_a_gpu():
    """Bad arguments come back as a status before anything touches a device."""
    from custom_d_fine_amd import hip
    pack = hip._DA_SHAPE
    shape = [2, 5, 7, 4, 2, 16, 32, 1, 4, 1, 1, 0, 0, 0] + [8] * 14
    call = lambda s, scale=0.25, q=None: hip._lib.dfine_diff_attn_fwd(q, q, q, q, None, None, None, None, q, None, None, None, None, s and pack(*s), scale, 0.1, 1e-5, None)  # noqa: E731
    assert call(shape) == -1                                                            # null pointers
    assert call(None) == -1
    for at, bad in ((3, 3), (5, 12), (5, 72), (6, 130), (7, 2), (8, 3), (14, 4)):
        s = list(shape)
        s[at] = bad
        assert call(s, q=1 << 20) == -1 and hip._lib.dfine_diff_attn_bwd_ws_bytes(pack(*s)) == -1 and hip._lib.dfine_diff_attn_fwd_ws_bytes(pack(*s)) == -1
    assert call(shape, scale=0.0, q=1 << 20) == -1 and call(shape, q=(1 << 20) + 2) == -1
    assert call([0] + shape[1:]) == 0
    assert hip._lib.dfine_diff_attn_bwd_ws_bytes(pack(*shape)) > 0 and hip._lib.dfine_diff_attn_mask_words(1, 65, 130) == 65 * 3 + 130 * 2 + 2 * 3 + 1
    assert hip._lib.dfine_diff_attn_mask(None, 1, 5, 5, 0, 5, None, None) == -1
    qkn = [2, 5, 4, 2, 16, 8, 9, 1, 0, 0, 0, 0, 0] + [0] * 12
    for at, bad in ((4, 12), (4, 264), (5, 12), (5, 24), (6, 4), (7, 3), (0, -1)):
        s = list(qkn)
        s[at] = bad
        assert hip._lib.dfine_qk_norm_rotate_fwd(1 << 20, 1 << 20, None, None, 1 << 20, 1 << 20, None, 1 << 20, 1 << 20, hip._QKN_SHAPE(*s), 1e-6, None) == -1
    assert hip._lib.dfine_qk_norm_rotate_fwd(None, None, None, None, 1 << 20, 1 << 20, None, None, None, hip._QKN_SHAPE(*qkn), 1e-6, None) == -1
    none = hip._QKN_SHAPE(*([2, 5, 0, 0] + qkn[4:]))
    assert hip._lib.dfine_qk_norm_rotate_fwd(None, None, None, None, 1 << 20, 1 << 20, None, None, None, none, 1e-6, None) == 0


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_norm_rotate(oracle_backend, interleaved):
    q, k, cos, sin = _qk()
    angle = torch.rand(9, 4)
    cos, sin, w = angle.cos(), angle.sin(), torch.rand(16)
    p = torch.tensor([8, 0, 3, 3, 1])
    y, z = kernels.qk_norm_rotate(q, k, w, None, cos, sin, p, interleaved=interleaved)
    assert ref.rel(y, ref.norm_rotate(q.double(), w.double(), cos, sin, p, 1e-6, interleaved)) < 64 * 2 ** -24
    assert ref.rel(z, ref.norm_rotate(k.double(), None, cos, sin, p, 1e-6, interleaved)) < 64 * 2 ** -24


def test_oracle_diff_attention_and_its_gradients(oracle_backend):
    """The oracle against the 64-bit restatement; the restatement's gradients against differences."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 5, 4, 2, 16), (2, 7, 2, 2, 16), (2, 7, 2, 32)))
    lam, w = 0.2 * torch.randn(4, 4, 16, generator=g, dtype=torch.float64), 1 + 0.2 * torch.randn(32, generator=g, dtype=torch.float64)
    mask = torch.rand(5, 7, generator=g) < 0.4
    mask[2] = True
    mask[:, 4] = True
    lens, start = torch.tensor([7, 3]), torch.tensor([1, 2])
    seen = ref.visible(2, 5, 7, mask, lens, True, start)
    y = kernels.diff_attention(q.float(), k.float(), v.float(), lam.float(), 0.3, w.float(), attn_mask=mask, kv_lengths=lens, causal=True, query_start=start)
    assert y.shape == (2, 5, 4, 32)
    f = lambda *a: ref.diff_attention(a[0], a[1], a[2], a[3], 0.3, a[4], 1e-5, seen, 0.25)  # noqa: E731
    assert ref.rel(y, f(q, k, v, lam, w)) < 512 * 2 ** -24
    assert torch.autograd.gradcheck(f, [t.clone().requires_grad_(True) for t in (q, k, v, lam, w)], eps=1e-6, atol=1e-5, rtol=1e-4)
