"""csrc/diffattn.hip through kernels.diff_attention against a 64-bit restatement.

Tolerances, in the 2-norm.  A rounding to bf16 is off by at most 2^-8 of the value; the probabilities (forward), A_1 V, dU and dS (backward) and the
result are rounded once each.  out: 2 roundings; dV: P, A_1 V, dU, result = 4; dq, dk: also dS = 5; parameters: A_1 V, P, result = 3.  What such a
rounding is 2^-8 of are the TERMS of the sums that follow it, and their errors add up as terms of random signs do: the larger of the result's 2-norm and of
attention_block_ref.diff_attention_spread's.  (A row that sees ONE key shows why: dS = 0 there, and dl of a normed head is eps-small, while dP and D are not.)
fp32: sums of n = M (N for dk, dv) terms in 32 bits, at most (n + 8 d + 64) 2^-24 with scores up to 8 * sqrt(d) * scale in the exponent, of the same."""
import pytest
import torch

from . import attention_block_ref as ref

pytestmark = pytest.mark.gpu

INIT, EPS = 0.35, 1e-5
ROUNDINGS = {"out": 2, "dq": 5, "dk": 5, "dv": 4, "dlam": 3, "dweight": 3}


def _tol(name, dtype, n, d):
    if dtype == torch.bfloat16:
        return ROUNDINGS[name] * 2 ** -8
    return (n + 8 * d + 64) * 2 ** -24


def _off(a, b, spread):
    return (a.detach().double() - b.detach()).norm().item() / max(b.norm().item(), spread, 1e-300)


def _inputs(cuda, B, N, M, H, Hk, d, dv, dtype, shared=False, seed=1):
    g = torch.Generator().manual_seed(seed + 7 * N + M + d)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k = mk(B, N, H, 2, d).to(dtype).to(cuda), mk(B, M, Hk, 2, d).to(dtype).to(cuda)
    v = (mk(B, M, Hk, dv) + 0.5 * mk(Hk, dv)).to(dtype).to(cuda)
    lam = (0.15 * mk(*((4, d) if shared else (4, H, d)))).to(dtype).to(cuda)
    w = (1 + 0.2 * mk(dv)).to(dtype).to(cuda)
    dy = (mk(B, N, H, dv) + 0.5 * mk(H, dv)).to(dtype).to(cuda)
    return q, k, v, lam, w, dy, g


def _run(q, k, v, lam, w, dy, init=INIT, **kw):
    from custom_d_fine_amd import kernels
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam) + (() if w is None else (w,))]
    y = kernels.diff_attention(*leaves[:4], init, norm_weight=None if w is None else leaves[4], norm_eps=EPS, **kw)
    return (y,) + torch.autograd.grad(y, leaves, dy), leaves


def _check(cuda, q, k, v, lam, w, dy, init=INIT, **kw):
    from custom_d_fine_amd import kernels
    B, N, H, _, d = q.shape
    M = k.shape[1]
    got, _ = _run(q, k, v, lam, w, dy, init, **kw)
    seen = ref.visible(B, N, M, kw.get("attn_mask"), kw.get("kv_lengths"), kw.get("causal", False), kw.get("query_start", 0), cuda)
    dl = [t.detach().double().requires_grad_(True) for t in (q, k, v, lam) + (() if w is None else (w,))]
    y = ref.diff_attention(*dl[:4], init, None if w is None else dl[4], EPS, seen, kw.get("scale") or d ** -0.5)
    want = (y,) + torch.autograd.grad(y, dl, dy.double())
    spread = ref.diff_attention_spread(*[t.detach() for t in dl[:4]], init, None if w is None else dl[4].detach(), EPS, seen, kw.get("scale") or d ** -0.5, dy.double())
    for name, a, b in zip(("out", "dq", "dk", "dv", "dlam", "dweight"), got, want):
        assert a.dtype == q.dtype or name in ("dlam", "dweight")
        assert a.shape == b.shape and torch.isfinite(a).all(), name
        err, tol = _off(a, b, spread[name]), _tol(name, q.dtype, max(M, N), d)
        print(name, "%.2e of %.2e" % (err, tol))
        assert err <= tol, name
    with torch.no_grad():
        z = kernels.diff_attention(q, k, v, lam, init, norm_weight=w, norm_eps=EPS, **kw)
    assert _off(z, y, spread["out"]) <= _tol("out", q.dtype, M, d)
    return got


DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,M,H,Hk,d,dv", [(1, 1, 1, 6, 6, 8, 8), (2, 33, 33, 6, 6, 16, 32), (2, 77, 77, 6, 2, 8, 24), (1, 129, 65, 8, 4, 24, 48),
                                             (2, 130, 200, 6, 1, 32, 64), (1, 300, 300, 8, 8, 32, 64), (2, 64, 96, 6, 6, 40, 80), (1, 100, 257, 8, 2, 64, 128),
                                             (1, 70, 70, 6, 3, 48, 16), (1, 50, 131, 6, 6, 16, 128)])
def test_sizes(cuda, dtype, B, N, M, H, Hk, d, dv):
    q, k, v, lam, w, dy, _ = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
    _check(cuda, q, k, v, lam, w, dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["groups", "rows", "batched", "columns", "all", "lengths", "causal", "causal behind", "causal starts", "together"])
@pytest.mark.parametrize("B,N,M,H,Hk,d,dv", [(2, 150, 150, 6, 6, 16, 32), (3, 97, 203, 6, 2, 32, 64), (2, 131, 131, 8, 2, 64, 128)])
def test_masks(cuda, dtype, kind, B, N, M, H, Hk, d, dv):
    q, k, v, lam, w, dy, g = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
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
        kw["attn_mask"] = m.to(cuda)
    if kind == "columns":                                              # padding as a mask: expanded rows
        m = torch.zeros(B, 1, M, dtype=torch.bool)
        m[0, :, M // 2:] = True
        kw["attn_mask"] = m.expand(B, N, M).to(cuda)
    if kind == "all":
        kw["attn_mask"] = torch.ones(N, M, dtype=torch.bool, device=cuda)
    if kind in ("lengths", "together"):
        kw["kv_lengths"] = torch.tensor([M - 5, 1, 0][:B], device=cuda)
    if kind == "causal":
        kw.update(causal=True)
    if kind == "causal behind":
        kw.update(causal=True, query_start=M - N - 3)
    if kind in ("causal starts", "together"):
        kw.update(causal=True, query_start=torch.tensor([0, -10, 40][:B], device=cuda))
    got = _check(cuda, q, k, v, lam, w, dy, **kw)
    seen = ref.visible(B, N, M, kw.get("attn_mask"), kw.get("kv_lengths"), kw.get("causal", False), kw.get("query_start", 0), cuda)
    none = ~seen.any(2)
    assert (got[0][none] == 0).all() and (got[1][none] == 0).all()
    dead = ~seen.any(1)
    assert (got[2][dead] == 0).all() and (got[3][dead] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_norm_shared_vectors_and_scale(cuda, dtype):
    q, k, v, lam, _, dy, _ = _inputs(cuda, 2, 80, 90, 6, 3, 32, 64, dtype, shared=True)
    _check(cuda, q, k, v, lam, None, dy)
    _check(cuda, q, k, v, lam, None, dy, scale=0.05)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,M,H,Hk,d,dv", [(3, 1, 1000, 8, 2, 64, 128), (2, 1, 1, 6, 6, 32, 64), (2, 5, 3001, 6, 1, 24, 48), (1, 40, 2500, 8, 2, 16, 32),
                                             (16, 1, 700, 16, 4, 64, 128)])
def test_few_queries_over_long_caches(cuda, dtype, B, N, M, H, Hk, d, dv):
    q, k, v, lam, w, dy, g = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
    n = torch.randint(0, M + 1, (B,), generator=g).to(torch.int32)
    n[0] = M
    _check(cuda, q, k, v, lam, w, dy, kv_lengths=n.to(cuda))
    _check(cuda, q, k, v, lam, w, dy, causal=True, query_start=(n - N).to(cuda))


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_hidden_may_hold_anything(cuda, dtype):
    """NaN and infinities behind kv_lengths, in keys that the mask hides from every query, in queries that see nothing."""
    B, N, M, H, Hk, d, dv = 2, 70, 140, 6, 3, 32, 64
    q, k, v, lam, w, dy, g = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
    mask = torch.rand(N, M, generator=g) < 0.3
    mask[:, 10:30] = True
    mask[5] = True
    mask[33:40] = True
    mask = mask.to(cuda)
    lens = torch.tensor([100, 131], device=cuda)
    clean, _ = _run(q, k, v, lam, w, dy, attn_mask=mask, kv_lengths=lens)
    q, k, v, dy = q.clone(), k.clone(), v.clone(), dy.clone()
    for b, n in enumerate((100, 131)):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    k[:, 10:30], v[:, 10:30] = float("inf"), float("nan")
    q[:, 5], q[:, 33:40] = float("nan"), float("-inf")
    dy[:, 5] = float("nan")
    dirty, _ = _run(q, k, v, lam, w, dy, attn_mask=mask, kv_lengths=lens)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)


@pytest.mark.parametrize("N", [1, 40])
def test_a_cache_behind_the_last_causal_position_may_hold_anything(cuda, N):
    B, M, H, Hk, d, dv = 2, 500, 6, 2, 32, 64
    q, k, v, lam, w, dy, g = _inputs(cuda, B, N, M, H, Hk, d, dv, torch.bfloat16)
    start = torch.tensor([101, 333], device=cuda)
    clean, _ = _run(q, k, v, lam, w, dy, causal=True, query_start=start)
    for b, n in enumerate((101 + N, 333 + N)):
        k[b, n:], v[b, n:] = float("nan"), float("nan")
    dirty, _ = _run(q, k, v, lam, w, dy, causal=True, query_start=start)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)


def test_a_visible_nan_reaches_the_result(cuda):
    q, k, v, lam, w, dy, _ = _inputs(cuda, 1, 40, 40, 6, 6, 32, 64, torch.bfloat16)
    k[0, 3, 2, 0, 1] = float("nan")
    y, *_ = _run(q, k, v, lam, w, dy)[0]
    assert torch.isnan(y[:, :, 2]).all() and torch.isfinite(y[:, :, [0, 1, 3, 4, 5]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(cuda, dtype):
    """Scores of hundreds: the running maximum keeps the exponentials in range; the answer is close to a choice of single keys."""
    q, k, v, lam, w, dy, _ = _inputs(cuda, 1, 90, 300, 6, 6, 32, 64, dtype)
    from custom_d_fine_amd import kernels
    q = q * 40
    y = kernels.diff_attention(q, k, v, lam, INIT, norm_weight=w, norm_eps=EPS)
    seen = ref.visible(1, 90, 300, device=cuda)
    want = ref.diff_attention(q.double(), k.double(), v.double(), lam.double(), INIT, w.double(), EPS, seen, 32 ** -0.5)
    # 32 bits: a score of s is off by at most (32 + 2) 2^-24 |s| in the exponent, |s| < 40 * 6 * 6: 2e-3 at the most
    assert ref.rel(y, want) <= (2.5 * 2 * 2 ** -8 if dtype == torch.bfloat16 else 0) + 34 * 2 ** -24 * 40 * 36 * 2.5      # (|A_0 V|, |l A_1 V| against |U|: 2.5)


def test_strides_and_alignment(cuda):
    from custom_d_fine_amd import kernels
    B, N, H, d, dv = 2, 75, 6, 16, 32
    g = torch.Generator().manual_seed(3)
    packed = torch.randn(B, N, H * (4 * d + dv), generator=g).bfloat16().to(cuda)
    q = packed[..., :2 * H * d].view(B, N, H, 2, d)
    k = packed[..., 2 * H * d:4 * H * d].view(B, N, H, 2, d)
    v = packed[..., 4 * H * d:].view(B, N, H, dv)
    lam, w = torch.randn(4, d, generator=g).mul(0.1).to(cuda), torch.ones(dv, device=cuda)
    base = kernels.diff_attention(q.contiguous(), k.contiguous(), v.contiguous(), lam, INIT, w)
    maps_first = q.permute(0, 3, 2, 1, 4).contiguous().permute(0, 3, 2, 1, 4)       # [B, 2, H, N, d] storage
    flat = torch.empty(v.numel() + 8, device=cuda, dtype=torch.bfloat16)
    off = flat[1:1 + v.numel()].view(v.shape).copy_(v)
    for a, b, c in ((q, k, v), (maps_first, k, v), (q, k.permute(0, 2, 1, 3, 4).contiguous().permute(0, 2, 1, 3, 4), off)):
        assert torch.equal(kernels.diff_attention(a, b, c, lam, INIT, w), base)
    ql, kl, vl = (t.detach().requires_grad_(True) for t in (q, k, v))
    y = kernels.diff_attention(ql, kl, vl, lam, INIT, w)
    y.sum().backward()                                                              # an expanded gradient
    dl = [t.detach().double().requires_grad_(True) for t in (q, k, v)]
    ref.diff_attention(*dl, lam.double(), INIT, w.double(), EPS, ref.visible(B, N, N, device=cuda), d ** -0.5).sum().backward()
    for name, a, b in zip(("dq", "dk", "dv"), (ql, kl, vl), dl):
        assert ref.rel(a.grad, b.grad) <= 2.5 * _tol(name, torch.bfloat16, N, d), name


def test_empty_and_zero_keys(cuda):
    from custom_d_fine_amd import kernels
    lam, w = torch.zeros(4, 16, device=cuda, requires_grad=True), torch.ones(32, device=cuda, requires_grad=True)
    q, k, v = (torch.randn(s, device=cuda, requires_grad=True) for s in ((2, 5, 6, 2, 16), (2, 0, 6, 2, 16), (2, 0, 6, 32)))
    y = kernels.diff_attention(q, k, v, lam, INIT, w, attn_mask=torch.zeros(5, 0, dtype=torch.bool, device=cuda))
    assert torch.equal(y, torch.zeros_like(y))
    for g_ in torch.autograd.grad(y.sum(), (q, k, v, lam, w)):
        assert (g_ == 0).all()
    q0 = torch.randn(2, 0, 6, 2, 16, device=cuda, requires_grad=True)
    k1, v1 = torch.randn(2, 9, 6, 2, 16, device=cuda, requires_grad=True), torch.randn(2, 9, 6, 32, device=cuda, requires_grad=True)
    y = kernels.diff_attention(q0, k1, v1, lam, INIT, w)
    assert y.shape == (2, 0, 6, 32)
    for g_ in torch.autograd.grad(y.sum(), (q0, k1, v1, lam, w)):
        assert (g_ == 0).all()


def test_same_bits_every_time_and_only_what_is_asked(cuda):
    q, k, v, lam, w, dy, _ = _inputs(cuda, 2, 200, 333, 8, 2, 32, 64, torch.bfloat16)
    one, two = _run(q, k, v, lam, w, dy)[0], _run(q, k, v, lam, w, dy)[0]
    for a, b in zip(one, two):
        assert torch.equal(a, b)
    from custom_d_fine_amd import kernels
    for at, index in ((0, 1), (1, 2), (2, 3), (3, 4), (4, 5)):
        leaves = [t.detach().requires_grad_(j == at) for j, t in enumerate((q, k, v, lam, w))]
        y = kernels.diff_attention(*leaves[:4], INIT, norm_weight=leaves[4], norm_eps=EPS)
        (got,) = torch.autograd.grad(y, [leaves[at]], dy)
        assert torch.equal(got, one[index])


def test_gradient_against_differences(cuda):
    """fp32: a directional difference of the kernel's own forward.  h = 2^-7, second-order error h^2 ~ 6e-5 of third derivatives of order one, rounding of
    the sums 2^-24 sqrt(n) / h ~ 1e-3 of a term: 1e-2 of the derivative's scale covers both."""
    from custom_d_fine_amd import kernels
    q, k, v, lam, w, dy, g = _inputs(cuda, 1, 24, 40, 6, 2, 16, 32, torch.float32)
    grads = _run(q, k, v, lam, w, dy, causal=True, query_start=16)[0][1:]
    args, h = [q, k, v, lam, w], 2.0 ** -7

    def f(vals):
        return (kernels.diff_attention(*vals[:4], INIT, norm_weight=vals[4], norm_eps=EPS, causal=True, query_start=16).double() * dy.double()).sum().item()

    for at, grad in enumerate(grads):
        step = torch.randn(args[at].shape, generator=g).to(cuda)
        up, down = ([a + s * h * step if j == at else a for j, a in enumerate(args)] for s in (1, -1))
        diff, want = (f(up) - f(down)) / (2 * h), (grad.double() * step.double()).sum().item()
        assert abs(diff - want) <= 1e-2 * grad.double().norm().item() * step.double().norm().item() / step.numel() ** 0.5 * 4, at


def test_other_stream_and_captured_replay(cuda):
    """Forward and backward captured once and replayed on new data, eager work between the replays, against the eager result; two graphs alive."""
    from custom_d_fine_amd import kernels
    q, k, v, lam, w, dy, g = _inputs(cuda, 2, 90, 90, 6, 3, 32, 64, torch.bfloat16)
    mask = (torch.rand(90, 90, generator=g) < 0.3).to(cuda)
    graphs = []
    for n in range(2):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v, lam, w)]

        def step(leaves=leaves):
            y = kernels.diff_attention(*leaves[:4], INIT, norm_weight=leaves[4], norm_eps=EPS, attn_mask=mask)
            return (y,) + torch.autograd.grad(y, leaves, dy)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            warm = step()
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(warm, step()):
            assert torch.equal(a, b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, leaves, step, out))
    for i in range(3):
        for graph, leaves, step, out in graphs:
            with torch.no_grad():
                leaves[i % 3].copy_(torch.randn(leaves[i % 3].shape, generator=g).to(cuda))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, _, step, out in graphs:
            for a, b in zip(out, step()):
                assert torch.equal(a, b)


def test_attention_block_of_a_token_stream(cuda):
    """Projection -> norms + rotation -> differential attention -> projection, training step under bf16 autocast, as a layer of this framework would run it,
    against the same chain in 64 bits.  Roundings: projection, norm, out, output projection on top of diff_attention's own counts (2 and 6), each of terms at most
    1 + l < 2.5 times the difference of the maps."""
    from custom_d_fine_amd import kernels
    B, L, E, H, d, dv = 2, 196, 128, 2, 32, 64
    g = torch.Generator().manual_seed(8)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = mk(B, L, E).to(cuda)
    params = [(mk(3 * E, E) / E ** 0.5).to(cuda), (0.1 * mk(3 * E)).to(cuda), (mk(E, E) / E ** 0.5).to(cuda), (0.1 * mk(E)).to(cuda),
              (1 + 0.1 * mk(d)).to(cuda), (1 + 0.1 * mk(d)).to(cuda), (0.1 * mk(4, H, d)).to(cuda), (1 + 0.1 * mk(dv)).to(cuda)]
    y0, x0 = torch.meshgrid(torch.arange(14.0), torch.arange(14.0), indexing="ij")
    freq = 100.0 ** (-torch.arange(d // 4) / (d // 4))
    angle = torch.cat([y0.reshape(-1, 1) * freq, x0.reshape(-1, 1) * freq], 1)        # rows by their y and x: a 14 x 14 map
    cos, sin = angle.cos().to(cuda), angle.sin().to(cuda)
    mask = (torch.rand(L, L, generator=g) < 0.2).to(cuda)
    dy = mk(B, L, E).to(cuda)

    def chain(x, in_w, in_b, out_w, out_b, wq, wk, lam, wn, exact):
        if exact:
            p = x @ in_w.t() + in_b
        else:
            p = kernels.linear(x, in_w, in_b)
        q, k, v = p[..., :E].view(B, L, 2 * H, d), p[..., E:2 * E].view(B, L, 2 * H, d), p[..., 2 * E:].view(B, L, H, dv)
        if exact:
            rows = torch.arange(L, device=cuda)
            q, k = ref.norm_rotate(q, wq, cos, sin, rows, 1e-6, False), ref.norm_rotate(k, wk, cos, sin, rows, 1e-6, False)
            o = ref.diff_attention(q.view(B, L, H, 2, d), k.view(B, L, H, 2, d), v, lam, INIT, wn, EPS, ref.visible(B, L, L, mask, device=cuda), d ** -0.5)
            return o.reshape(B, L, E) @ out_w.t() + out_b
        q, k = kernels.qk_norm_rotate(q, k, wq, wk, cos, sin)
        o = kernels.diff_attention(q.view(B, L, H, 2, d), k.view(B, L, H, 2, d), v, lam, INIT, wn, EPS, attn_mask=mask)
        return kernels.linear(o.view(B, L, E), out_w, out_b)

    leaves = [t.clone().requires_grad_(True) for t in [x] + params]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = chain(*leaves, exact=False)
    got = torch.autograd.grad(y, leaves, dy.bfloat16())
    dl = [(t.bfloat16() if i in (0, 1, 3) else t).double().requires_grad_(True) for i, t in enumerate([x] + params)]      # operands of the projections
    z = chain(*dl, exact=True)
    want = torch.autograd.grad(z, dl, dy.bfloat16().double())
    assert ref.rel(y, z) <= 2.5 * 6 * 2 ** -8
    for i, (a, b) in enumerate(zip(got, want)):
        assert ref.rel(a, b) <= 2.5 * 12 * 2 ** -8, i


def test_decoding_steps_captured(cuda):
    """One token at a time: norms + rotation at the token's position, the cache written, attention over the filled part.  The step is captured once and replayed
    for every token, eager work between the replays; each equals the eager step, and the last the whole sequence at once within the roundings of both."""
    from custom_d_fine_amd import kernels
    B, M, H, Hk, d, dv, steps = 3, 1500, 4, 2, 32, 64, 6
    g = torch.Generator().manual_seed(21)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    toks = [[t.bfloat16().to(cuda) for t in (mk(B, 1, 2 * H, d), mk(B, 1, 2 * Hk, d), mk(B, 1, Hk, dv))] for _ in range(steps)]
    wq, wk, wn, lam = (1 + 0.1 * mk(d)).to(cuda), (1 + 0.1 * mk(d)).to(cuda), (1 + 0.1 * mk(dv)).to(cuda), (0.1 * mk(4, H, d)).to(cuda)
    angle = torch.arange(M)[:, None] * 100.0 ** (-torch.arange(d // 2) / (d // 2))
    cos, sin = angle.cos().to(cuda), angle.sin().to(cuda)
    first = torch.tensor([3, 1200, 700], device=cuda)
    batch = torch.arange(B, device=cuda)

    def state():
        gg = torch.Generator().manual_seed(22)
        k0, v0 = torch.randn(B, M, Hk, 2, d, generator=gg).bfloat16().to(cuda), torch.randn(B, M, Hk, dv, generator=gg).bfloat16().to(cuda)
        return {"k": k0, "v": v0, "len": first.clone(), "in": [t.clone() for t in toks[0]]}

    def step(s):
        q, k = kernels.qk_norm_rotate(s["in"][0], s["in"][1], wq, wk, cos, sin, s["len"][:, None])
        s["k"][batch, s["len"]] = k.view(B, Hk, 2, d)
        s["v"][batch, s["len"]] = s["in"][2][:, 0]
        s["len"] += 1
        return kernels.diff_attention(q.view(B, 1, H, 2, d), s["k"], s["v"], lam, INIT, wn, EPS, kv_lengths=s["len"])

    with torch.no_grad():
        side, cap, eager = torch.cuda.Stream(), state(), state()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(cap)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cap)
        fresh = state()
        for a, b in zip((cap["k"], cap["v"], cap["len"]), (fresh["k"], fresh["v"], fresh["len"])):
            a.copy_(b)
        for t in toks:
            for s in (cap, eager):
                for a, b in zip(s["in"], t):
                    a.copy_(b)
            want = step(eager)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        # the tokens at once, behind each sequence's own prefix
        q, k = kernels.qk_norm_rotate(torch.cat([t[0] for t in toks], 1), torch.cat([t[1] for t in toks], 1), wq, wk, cos, sin,
                                      first[:, None] + torch.arange(steps, device=cuda))
        whole = kernels.diff_attention(q.view(B, steps, H, 2, d), eager["k"], eager["v"], lam, INIT, wn, EPS, causal=True, query_start=first)
        assert torch.equal(eager["k"][1, 1200:1200 + steps], k.view(B, steps, Hk, 2, d)[1])
        assert ref.rel(whole[:, -1:], want) <= 2 * 2.5 * _tol("out", torch.bfloat16, M, d)


def test_saved_tensors_that_moved_and_a_second_backward(cuda):
    """What the graph saved comes back from the host with other strides; a graph that is kept gives its gradients again; operands that are recomputed."""
    from torch.utils.checkpoint import checkpoint

    from custom_d_fine_amd import kernels
    B, N, H, d, dv = 2, 90, 4, 32, 64
    g = torch.Generator().manual_seed(5)
    packed = torch.randn(B, N, H * (4 * d + dv), generator=g).bfloat16().to(cuda)
    lam, w = (0.1 * torch.randn(4, H, d, generator=g)).to(cuda), torch.ones(dv, device=cuda)
    mask = (torch.rand(N, N, generator=g) < 0.3).to(cuda)
    dy = torch.randn(B, N, H, dv, generator=g).bfloat16().to(cuda)

    def f(p, l, n):
        q, k = kernels.qk_norm_rotate(p[..., :2 * H * d].view(B, N, 2 * H, d), p[..., 2 * H * d:4 * H * d].view(B, N, 2 * H, d))
        return kernels.diff_attention(q.view(B, N, H, 2, d), k.view(B, N, H, 2, d), p[..., 4 * H * d:].view(B, N, H, dv), l, INIT, n, EPS, attn_mask=mask)

    leaves = [t.clone().requires_grad_(True) for t in (packed, lam, w)]
    y = f(*leaves)
    base = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        z = f(*leaves)
    moved = torch.autograd.grad(z, leaves, dy)
    redone = torch.autograd.grad(checkpoint(f, *leaves, use_reentrant=False), leaves, dy)
    for one in (again, moved, redone):
        for a, b in zip(one, base):
            assert torch.equal(a, b)


def test_offsets_past_32_bits(cuda):
    """A cache of 4.3 GB whose second sequence and last tokens lie past 2^31 elements: sequence stride 2^30 + 512, token stride 2^24 and 64 tokens."""
    from custom_d_fine_amd import kernels
    Hk, d, dv = 1, 64, 128
    flat = torch.empty(2 ** 31 + 2 ** 20, device=cuda, dtype=torch.bfloat16)            # only the rows below are ever written
    for B, M, sb, st in ((2, 130, 2 ** 31, 128), (2, 64, 2 ** 30 + 512, 2 ** 24)):
        q, k, v, lam, w, dy, _ = _inputs(cuda, B, 3, M, 6, Hk, d, dv, torch.bfloat16)
        far = flat.as_strided((B, M, Hk, 2, d), (sb, st, 2 * d, d, 1))
        assert (B - 1) * sb + (M - 1) * st + 2 * d <= flat.numel() and (B - 1) * sb + (M - 1) * st >= 2 ** 31 - 2 ** 24
        far.copy_(k)
        one, two = _run(q, far, v, lam, w, dy)[0], _run(q, k, v, lam, w, dy)[0]
        for a, b in zip(one, two):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk,d,dv", [(6, 2, 16, 32), (6, 6, 32, 64), (4, 2, 64, 128)])
def test_negative_and_zero_lambda(cuda, dtype, H, Hk, d, dv):
    """l < 0 for every second head (exp(d x^2) = 2.2 taken away from 1 + init); then l = 1 - 1 + 0 exactly: nothing comes through the second map."""
    q, k, v, lam, w, dy, _ = _inputs(cuda, 2, 70, 101, H, Hk, d, dv, dtype)
    lam[2:, ::2] = (0.8 / d) ** 0.5
    _check(cuda, q, k, v, lam, w, dy)
    _check(cuda, q, k, v, lam, None, dy)
    lam = torch.zeros_like(lam)
    _check(cuda, q, k, v, lam, w, dy, 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,M,H,Hk,d,dv", [(2, 3, 70, 40, 1, 16, 32), (1, 130, 130, 66, 2, 8, 16), (3, 1, 300, 64, 1, 64, 128)])
def test_many_heads_of_one_key_head(cuda, dtype, B, N, M, H, Hk, d, dv):
    """More heads to a key head than a wave has rows, and numbers of them that no power of two divides."""
    q, k, v, lam, w, dy, _ = _inputs(cuda, B, N, M, H, Hk, d, dv, dtype)
    _check(cuda, q, k, v, lam, w, dy, causal=True, query_start=M - N)


def test_masks_as_they_come(cuda):
    """An expanded mask, a transposed one, one batch's own, and lengths in 64 bits that do not fit 32."""
    from custom_d_fine_amd import kernels
    B, N, M = 3, 70, 90
    q, k, v, lam, w, _, g = _inputs(cuda, B, N, M, 6, 2, 32, 64, torch.bfloat16)
    mask = (torch.rand(N, M, generator=g) < 0.4).to(cuda)

    def run(m, n=B, lengths=None, **kw):
        return kernels.diff_attention(q[:n], k[:n], v[:n], lam, INIT, w, attn_mask=m, kv_lengths=lengths, **kw)

    base = run(mask)
    assert torch.equal(run(mask.expand(B, N, M)), base)
    assert torch.equal(run(mask.t().contiguous().t()), base)
    assert torch.equal(run(mask[None].repeat(B, 1, 1).transpose(0, 1).contiguous().transpose(0, 1)), base)
    assert torch.equal(run(mask[None], 1), base[:1])
    far = torch.tensor([2 ** 40, 2 ** 32 + 5, -2 ** 40], device=cuda)
    assert torch.equal(run(None, lengths=far), run(None, lengths=torch.tensor([M, M, 0], device=cuda, dtype=torch.int32)))
    assert torch.equal(run(None, causal=True, query_start=far), run(None, causal=True, query_start=torch.tensor([M, M, -M - N], device=cuda, dtype=torch.int32)))


def test_two_streams_at_once(cuda):
    """Calls on two streams that may run side by side, few rows (runs of the keys) and many, with their backward passes: nothing of one call is another's."""
    sets = [_inputs(cuda, 2, n, m, 8, 2, 32, 64, torch.bfloat16, seed=n) for n, m in ((4, 3000), (300, 300))]
    base = [_run(*s[:6])[0] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[j].append(_run(*sets[j][:6])[0])
    torch.cuda.synchronize()
    for j in range(2):
        for one in got[j]:
            for a, b in zip(one, base[j]):
                assert torch.equal(a, b)


def test_small_scales(cuda):
    """scale = 1e-20: both maps are flat, and the row statistics over scale still fit 32 bits."""
    q, k, v, lam, w, dy, _ = _inputs(cuda, 2, 50, 60, 6, 2, 16, 32, torch.float32)
    got, _ = _run(q, k, v, lam, w, dy, scale=1e-20)
    dl = [t.detach().double().requires_grad_(True) for t in (v, lam, w)]
    G = 3
    x = torch.exp((dl[1][0] * dl[1][1]).sum(-1)) - torch.exp((dl[1][2] * dl[1][3]).sum(-1)) + INIT
    u = ((1 - x)[None, :, None] * dl[0].mean(1).repeat_interleave(G, 1))[:, None].expand(2, 50, 6, 32)
    y = (1 - INIT) * dl[2] * u / (u.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    want = (y,) + torch.autograd.grad(y, dl, dy.double())
    for name, a, b in zip(("out", "dv", "dweight"), (got[0], got[3], got[5]), (want[0], want[1], want[3])):
        assert ref.rel(a, b) <= (60 + 8 * 16 + 64) * 2 ** -24, name
    assert torch.isfinite(torch.stack([g.double().abs().max() for g in got])).all()


def test_no_second_derivative(cuda):
    from custom_d_fine_amd import kernels
    q, k, v, lam, w, dy, _ = _inputs(cuda, 1, 8, 8, 6, 6, 16, 32, torch.float32)
    q.requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(kernels.diff_attention(q, k, v, lam, INIT, w), q, dy, create_graph=True)
    x = torch.randn(1, 4, 2, 16, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(kernels.qk_norm_rotate(x, None)[0].sum(), x, create_graph=True)
