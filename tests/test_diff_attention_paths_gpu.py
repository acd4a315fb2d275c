"""kernels.diff_attention on the kernels that grids of real size take: the forward pass for many rows (128 rows per workgroup, at least 256 workgroups), masks of
more than 64 tiles of keys or queries, runs of the keys joined for the widest heads; against the 64-bit restatement with test_diff_attention_gpu's tolerances."""
import pytest
import torch

from . import attention_block_ref as ref
from .test_diff_attention_gpu import DTYPES, EPS, INIT, _check, _inputs, _run

pytestmark = pytest.mark.gpu

# three sizes of heads, with and without shared key heads and channels that fill them; each makes 256 workgroups of 128 rows or more
MANY = [(16, 130, 130, 8, 8, 16, 32), (12, 165, 203, 16, 4, 8, 24), (16, 130, 131, 8, 8, 32, 64), (16, 131, 131, 16, 8, 24, 48), (16, 130, 130, 8, 8, 64, 128),
        (12, 161, 161, 16, 4, 40, 80)]


def _names(fn):
    """Names of the kernels that fn launches."""
    fn()
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        fn()
        torch.cuda.synchronize()
    return " ".join(e.key for e in prof.key_averages())


@pytest.mark.parametrize("dtype", DTYPES)
def test_which_forward_kernel(cuda, dtype):
    """The shapes of this file reach the kernels that they are here for."""
    from custom_d_fine_amd import kernels
    for shape, want in [(s, "diff_attn_fwd_kernel") for s in MANY] + [((3, 3, 3000, 8, 2, 64, 128), "diff_attn_join_kernel"), ((2, 40, 300, 8, 2, 64, 128), "diff_attn_fwd_split_kernel")]:
        q, k, v, lam, w, _, _ = _inputs(cuda, *shape, dtype)
        names = _names(lambda: kernels.diff_attention(q, k, v, lam, INIT, w))
        assert want in names and (want != "diff_attn_fwd_kernel" or "split" not in names), (shape, names)


def _kind(kind, cuda, B, N, M, g):
    kw = {}
    if kind == "groups":
        i, j = torch.arange(N) // 20, torch.arange(M) // 20
        kw["attn_mask"] = (i[:, None] != j[None, :]).to(cuda)
    if kind in ("rows", "together"):                                   # scattered, with rows that see nothing
        m = torch.rand(N, M, generator=g) < 0.4
        m[::7] = True
        m[70:] |= torch.arange(M) < 64
        kw["attn_mask"] = m.to(cuda)
    if kind == "batched":
        m = torch.rand(B, N, M, generator=g) < 0.6
        m[0, 3] = True
        m[1] = True
        kw["attn_mask"] = m.to(cuda)
    if kind == "all":
        kw["attn_mask"] = torch.ones(N, M, dtype=torch.bool, device=cuda)
    if kind in ("lengths", "together"):
        kw["kv_lengths"] = torch.tensor([M - 5, 1, 0, M, 64, 65] * B, device=cuda)[:B]
    if kind == "causal":
        kw.update(causal=True, query_start=M - N)
    if kind in ("starts", "together"):
        kw.update(causal=True, query_start=torch.tensor([0, -10, 40, M, -N] * B, device=cuda)[:B])
    return kw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["none", "groups", "rows", "batched", "all", "lengths", "causal", "starts", "together"])
@pytest.mark.parametrize("B,N,M,H,Hk,d,dv", MANY)
def test_many_rows(cuda, dtype, kind, B, N, M, H, Hk, d, dv):
    q, k, v, lam, w, dy, g = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
    kw = _kind(kind, cuda, B, N, M, g)
    got = _check(cuda, q, k, v, lam, w, dy, **kw)
    seen = ref.visible(B, N, M, kw.get("attn_mask"), kw.get("kv_lengths"), kw.get("causal", False), kw.get("query_start", 0), cuda)
    none, dead = ~seen.any(2), ~seen.any(1)
    assert (got[0][none] == 0).all() and (got[1][none] == 0).all()
    assert (got[2][dead] == 0).all() and (got[3][dead] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,M,H,Hk,d,dv", [MANY[0], MANY[3], MANY[5]])
def test_many_rows_without_norm_shared_and_negative_vectors(cuda, dtype, B, N, M, H, Hk, d, dv):
    q, k, v, lam, _, dy, _ = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype, shared=True)
    _check(cuda, q, k, v, lam, None, dy, scale=0.05)
    q, k, v, lam, w, dy, _ = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
    lam[2:, ::2] = (0.8 / d) ** 0.5
    _check(cuda, q, k, v, lam, w, dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,M,H,Hk,d,dv", [MANY[0], MANY[3], MANY[4]])
def test_many_rows_hidden_values_and_a_visible_nan(cuda, dtype, B, N, M, H, Hk, d, dv):
    q, k, v, lam, w, dy, g = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
    mask = torch.rand(N, M, generator=g) < 0.3
    mask[:, 10:30] = mask[5] = mask[33:40] = True
    mask = mask.to(cuda)
    lens = torch.tensor([100, 121, 0, M] * B, device=cuda)[:B]
    clean, _ = _run(q, k, v, lam, w, dy, attn_mask=mask, kv_lengths=lens)
    q2, k2, v2, dy2 = q.clone(), k.clone(), v.clone(), dy.clone()
    for b, n in enumerate(lens.tolist()):
        k2[b, n:], v2[b, n:] = float("nan"), float("inf")
    k2[:, 10:30], v2[:, 10:30] = float("inf"), float("nan")
    q2[:, 5], q2[:, 33:40] = float("nan"), float("-inf")
    dy2[:, 5] = float("nan")
    dirty, _ = _run(q2, k2, v2, lam, w, dy2, attn_mask=mask, kv_lengths=lens)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    start = 40 - N                                                     # keys from 40 on lie behind the last causal position
    clean, _ = _run(q, k, v, lam, w, dy, causal=True, query_start=start)
    k2, v2 = k.clone(), v.clone()
    k2[:, 40:], v2[:, 40:] = float("nan"), float("nan")
    dirty, _ = _run(q, k2, v2, lam, w, dy, causal=True, query_start=start)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    k2 = k.clone()
    k2[0, 3, 2, 0, 1] = float("nan")
    y = _run(q, k2, v, lam, w, dy)[0][0]
    heads = torch.arange(H, device=cuda) // (H // Hk) == 2
    assert torch.isnan(y[0][:, heads]).all() and torch.isfinite(y[0][:, ~heads]).all() and torch.isfinite(y[1:]).all()


def test_many_rows_strides(cuda):
    """Slices of one projection, maps first in memory, values off a 16-byte border: the same bits."""
    from custom_d_fine_amd import kernels
    B, N, H, d, dv = 16, 130, 8, 32, 64
    g = torch.Generator().manual_seed(3)
    packed = torch.randn(B, N, H * (4 * d + dv), generator=g).bfloat16().to(cuda)
    q, k, v = packed[..., :2 * H * d].view(B, N, H, 2, d), packed[..., 2 * H * d:4 * H * d].view(B, N, H, 2, d), packed[..., 4 * H * d:].view(B, N, H, dv)
    lam, w = torch.randn(4, d, generator=g).mul(0.1).to(cuda), torch.ones(dv, device=cuda)
    base = kernels.diff_attention(q.contiguous(), k.contiguous(), v.contiguous(), lam, INIT, w)
    flat = torch.empty(v.numel() + 8, device=cuda, dtype=torch.bfloat16)
    off = flat[1:1 + v.numel()].view(v.shape).copy_(v)
    for a, b, c in ((q, k, v), (q.permute(0, 3, 2, 1, 4).contiguous().permute(0, 3, 2, 1, 4), k, v), (q, k.permute(0, 2, 1, 3, 4).contiguous().permute(0, 2, 1, 3, 4), off)):
        assert torch.equal(kernels.diff_attention(a, b, c, lam, INIT, w), base)


def test_many_rows_two_streams_and_replay(cuda):
    """Few rows on one stream and many on another, with their backward passes; the calls for many rows captured and replayed on new data."""
    shapes = [(2, 4, 3000, 8, 2, 64, 128), MANY[2]]
    sets = [_inputs(cuda, *s, torch.bfloat16, seed=j) for j, s in enumerate(shapes)]
    base = [_run(*s[:6])[0] for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(5):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[j].append(_run(*sets[j][:6])[0])
    torch.cuda.synchronize()
    for j in range(2):
        for one in got[j]:
            for a, b in zip(one, base[j]):
                assert torch.equal(a, b)
    from custom_d_fine_amd import kernels
    q, k, v, lam, w, dy, g = sets[1]
    mask = (torch.rand(130, 131, generator=g) < 0.3).to(cuda)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, lam, w)]

    def step():
        y = kernels.diff_attention(*leaves[:4], INIT, norm_weight=leaves[4], norm_eps=EPS, attn_mask=mask)
        return (y,) + torch.autograd.grad(y, leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            leaves[i].copy_(torch.randn(leaves[i].shape, generator=g).to(cuda))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def _long_mask(kind, N, M, g):
    """Scattered pairs; blocks that leave out whole stretches of more than 64 tiles, free ones and mixed ones in between."""
    if kind == "scattered":
        m = torch.rand(N, M, generator=g) < 0.5
        m[::5] = True
        return m
    m = torch.ones(N, M, dtype=torch.bool)
    if M >= N:
        m[:, 4160:4231] = m[:, M - 70:] = False                        # keys far apart
        m[N // 2:, 64:192] = False
    else:
        m[4160:4231] = m[N - 70:] = False                              # queries far apart
        m[64:192, M // 2:] = False
    m[N // 3, :] = True
    return m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["scattered", "blocks"])
@pytest.mark.parametrize("B,N,M,H,Hk,d,dv", [
    (2, 3, 5003, 8, 2, 64, 128), (1, 40, 9001, 4, 4, 64, 128), (2, 17, 9100, 6, 2, 16, 32),           # few rows: runs of the keys, joined
    (1, 1030, 4400, 32, 32, 16, 32), (1, 1029, 5001, 64, 16, 32, 64),                                 # many rows
    (1, 5001, 70, 4, 2, 32, 64), (2, 8301, 130, 2, 2, 64, 128), (1, 4300, 65, 8, 8, 16, 32)])         # many queries: the walk along them for dK and dV
def test_masks_of_more_than_64_tiles(cuda, dtype, kind, B, N, M, H, Hk, d, dv):
    q, k, v, lam, w, dy, g = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
    mask = _long_mask(kind, N, M, g).to(cuda)
    got = _check(cuda, q, k, v, lam, w, dy, attn_mask=mask)
    none, dead = mask.all(1), mask.all(0)
    assert (got[0][:, none] == 0).all() and (got[1][:, none] == 0).all()
    assert (got[2][:, dead] == 0).all() and (got[3][:, dead] == 0).all()
    lens = torch.tensor([M - 3, 4200 if M > 4200 else M // 2], device=cuda)[:B]
    _check(cuda, q, k, v, lam, w, dy, attn_mask=mask[None].expand(B, N, M), kv_lengths=lens, causal=True, query_start=M - N + 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,M,H,Hk,d,dv", [(3, 1, 2900, 8, 2, 64, 128), (16, 1, 1900, 16, 4, 64, 128), (1, 5, 40001, 4, 1, 64, 128), (2, 33, 1025, 6, 3, 40, 128)])
def test_joined_runs_of_wide_heads(cuda, dtype, B, N, M, H, Hk, d, dv):
    q, k, v, lam, w, dy, g = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
    n = torch.randint(0, M + 1, (B,), generator=g).to(torch.int32)
    n[0] = M
    _check(cuda, q, k, v, lam, w, dy, kv_lengths=n.to(cuda))
    _check(cuda, q, k, v, lam, w, dy, causal=True, query_start=(n - N).to(cuda))


# how many independent roundings to bf16 are in a result: probabilities / dS, dU, W and the result itself
ACCURACY = {"out": 2, "dq": 3, "dk": 3, "dv": 3, "dlam": 2, "dweight": 2}


@pytest.mark.parametrize("B,N,H,Hk,d,dv,kind", [(4, 492, 4, 4, 32, 64, "groups"), (1, 2048, 8, 2, 64, 128, "causal"), (1, 6000, 4, 1, 64, 128, "causal")])
def test_errors_are_those_of_the_roundings(cuda, B, N, H, Hk, d, dv, kind):
    """bf16, self-attention over values with means, relative to the results themselves.  What one rounding is off by is measured on the 64-bit results: E, the
    2-norm of their own rounding over theirs.  k roundings of independent errors make sqrt(k) E where every term of the later sums carries them and nothing
    averages out; 1.2 times that is allowed (dq: 0.0035).  A U rounded to bf16 adds an error that does not average out and grows with the length: dq of the same
    formulas with that rounding put in (a simulation in 64 bits) is 0.0038 off at 492 tokens and 0.0040 at 6000 causal ones, without it 0.0030 and 0.0029."""
    g = torch.Generator(device=cuda).manual_seed(N)
    mk = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    q, k = mk(B, N, H, 2, d).bfloat16(), mk(B, N, Hk, 2, d).bfloat16()
    v = mk(B, N, Hk, dv).bfloat16() + 0.5 * mk(Hk, dv).bfloat16()
    lam, w = (0.1 * mk(4, H, d)).bfloat16(), (1 + 0.2 * mk(dv)).bfloat16()
    dy = (mk(B, N, H, dv) + 0.5 * mk(H, dv)).bfloat16()
    kw = dict(causal=True)
    if kind == "groups":
        dn = N * 2 // 5
        group = torch.arange(N, device=cuda) // (dn // 6)
        group = torch.where(torch.arange(N, device=cuda) < dn, group, -1)
        kw = dict(attn_mask=~((group[:, None] == group[None]) | (group[None] == -1)))
    got, _ = _run(q, k, v, lam, w, dy, **kw)
    seen = ref.visible(B, N, N, kw.get("attn_mask"), None, kw.get("causal", False), 0, cuda)
    dl = [t.double().requires_grad_(True) for t in (q, k, v, lam, w)]
    y = ref.diff_attention(*dl[:4], INIT, dl[4], EPS, seen, d ** -0.5)
    want = (y,) + torch.autograd.grad(y, dl, dy.double())
    bad = []
    for name, a, b in zip(("out", "dq", "dk", "dv", "dlam", "dweight"), got, want):
        err, tol = ref.rel(a, b), 1.2 * ACCURACY[name] ** 0.5 * ref.rel(b.bfloat16(), b)
        print(name, "%.5f of %.5f" % (err, tol))
        if err > tol:
            bad.append(name)
    assert not bad
