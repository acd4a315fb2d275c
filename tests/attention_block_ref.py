"""64-bit restatements of qk_norm_rotate and diff_attention for their tests, written from the formulas; gradients by autograd."""
import math

import torch


def norm_rotate(x, w, cos, sin, rows, eps, interleaved):
    x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        x = x * w
    if cos is None:
        return x
    r = 2 * cos.shape[1]
    c, s = cos.double()[rows], sin.double()[rows]
    if c.dim() == 2:
        c, s = c[None], s[None]
    c, s = c[:, :, None], s[:, :, None]
    if interleaved:
        z = x[..., :r].unflatten(-1, (r // 2, 2))
        y = torch.stack([z[..., 0] * c - z[..., 1] * s, z[..., 0] * s + z[..., 1] * c], -1).flatten(-2)
    else:
        a, b = x[..., :r].chunk(2, -1)
        y = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([y, x[..., r:]], -1)


def visible(B, N, M, mask=None, lengths=None, causal=False, start=0, device="cpu"):
    seen = torch.ones(B, N, M, dtype=torch.bool, device=device)
    if mask is not None:
        seen = seen & ~mask
    j, i = torch.arange(M, device=device), torch.arange(N, device=device)[:, None]
    if lengths is not None:
        seen = seen & (j < lengths.long().view(B, 1, 1))
    if causal:
        seen = seen & (j <= i + (start.long().view(B, 1, 1) if torch.is_tensor(start) else start))
    return seen


def diff_attention(q, k, v, lam, init, weight, eps, seen, scale):
    """All operands 64-bit; seen [B, N, M]."""
    B, N, H, _, d = q.shape
    G = H // k.shape[2]
    hidden = ~seen.any(1)                                             # keys no query sees may hold anything
    k = torch.where(hidden[:, :, None, None, None], 0.0, k).repeat_interleave(G, 2)
    v = torch.where(hidden[:, :, None, None], 0.0, v).repeat_interleave(G, 2)
    q = torch.where(seen.any(2)[:, :, None, None, None], q, 0.0)
    x = lam if lam.dim() == 3 else lam[:, None].expand(4, H, d)
    l = torch.exp((x[0] * x[1]).sum(-1)) - torch.exp((x[2] * x[3]).sum(-1)) + init
    u = []
    for t in range(2):
        s = torch.matmul(q[:, :, :, t].transpose(1, 2), k[:, :, :, t].permute(0, 2, 3, 1)) * scale
        s = s.masked_fill(~seen[:, None], -math.inf)
        a = torch.softmax(s, -1)
        a = torch.where(seen.any(2)[:, None, :, None], a, 0.0)
        u.append(torch.matmul(a, v.transpose(1, 2)))
    y = (u[0] - l[:, None, None] * u[1]).transpose(1, 2)
    if weight is not None:
        y = (1 - init) * weight * y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    return y


def diff_attention_spread(q, k, v, lam, init, weight, eps, seen, scale, dy):
    """2-norms of what the results and gradients are made of, terms added with random signs: sqrt(sum of squares) in the place of every sum.  Where the
    terms cancel (a row that sees one key has dS = 0; U is short where the maps agree) rounding errors stay in proportion to these and not to the result."""
    B, N, H, _, d = q.shape
    G = H // k.shape[2]
    hidden = ~seen.any(1)
    k = torch.where(hidden[:, :, None, None, None], 0.0, k).repeat_interleave(G, 2)
    v = torch.where(hidden[:, :, None, None], 0.0, v).repeat_interleave(G, 2).transpose(1, 2)
    q = torch.where(seen.any(2)[:, :, None, None, None], q, 0.0)
    x = lam if lam.dim() == 3 else lam[:, None].expand(4, H, d)
    e = [torch.exp((x[0] * x[1]).sum(-1)), torch.exp((x[2] * x[3]).sum(-1))]
    l = e[0] - e[1] + init
    a = []
    for t in range(2):
        s = torch.matmul(q[:, :, :, t].transpose(1, 2), k[:, :, :, t].permute(0, 2, 3, 1)) * scale
        a.append(torch.where(seen.any(2)[:, None, :, None], torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1), 0.0))
    o = [torch.matmul(t, v) for t in a]
    u = o[0] - l[:, None, None] * o[1]
    dy = torch.where(seen.any(2)[:, None, :, None], dy.transpose(1, 2), 0.0)
    both = a[0] ** 2 + (l[:, None, None] * a[1]) ** 2
    u2 = torch.matmul(both, v ** 2) + u ** 2
    r = 1.0
    t = dy
    if weight is not None:
        r = 1 / (u.pow(2).mean(-1, keepdim=True) + eps).sqrt()
        t = (1 - init) * weight * dy
    du2 = (r * t) ** 2                                                # (the norm's backward takes away from this)
    norm = lambda z: z.sum().sqrt().item()  # noqa: E731
    got = {"out": norm(u2 * ((1 - init) * weight * r) ** 2 if weight is not None else u2), "dv": norm(torch.matmul(both.transpose(2, 3), du2))}
    dq = dk = 0.0
    for t, f in ((0, torch.ones_like(l)), (1, l)):
        s2 = (f[:, None, None] * a[t] * scale) ** 2 * (torch.matmul(du2, (v ** 2).transpose(2, 3)) + (du2 * (o[t] ** 2 + u2)).sum(-1, keepdim=True))
        dq = dq + torch.matmul(s2, (k[:, :, :, t] ** 2).transpose(1, 2)).sum()
        dk = dk + torch.matmul(s2.transpose(2, 3), (q[:, :, :, t] ** 2).transpose(1, 2)).sum()
    got["dq"], got["dk"] = dq.sqrt().item(), dk.sqrt().item()
    dl2 = (du2 * (o[1] ** 2 + u2)).sum((0, 2, 3))[:, None]
    got["dlam"] = norm(dl2 * (e[0][:, None] ** 2 * (x[0] ** 2 + x[1] ** 2) + e[1][:, None] ** 2 * (x[2] ** 2 + x[3] ** 2)))
    got["dweight"] = norm(((1 - init) * r * dy) ** 2 * u2)
    return got


def rel(got, ref):
    """2-norm of the difference over the 2-norm of the reference (the difference itself where that is zero)."""
    got, ref = got.detach().double(), ref.detach().double()
    n = ref.norm().item()
    return (got - ref).norm().item() / (n if n else 1.0)
