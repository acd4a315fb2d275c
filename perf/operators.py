"""Timed cases of the attention-block operators: `kernels.diff_attention` (differential attention: the difference of two softmax
maps, learned weights, norm of each head's result) and `kernels.qk_norm_rotate` (norms of queries and keys for each head with the
position rotation in the same pass).

`own` chooses between the framework's kernels and the plain form of the same mathematics in elementary torch operations; `exact`
restates the results in 64 bits, gradients by their formulas.
"""
import math

import torch

own = False

BF16, FP32 = "bfloat16", "float32"


# ------------------------------------------------------------------------------------------------------------------ cases
def _attn(name, batch, queries, keys, heads, kv_heads, dim, vdim, dtype, mask, train):
    return {"name": name, "op": "attention", "batch": batch, "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "vdim": vdim, "dtype": dtype, "mask": mask, "train": train}


def _norm(name, batch, length, heads, kv_heads, dim, rot, dtype, table, paired, placed, train):
    return {"name": name, "op": "norm_rotate", "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "dtype": dtype, "table": table, "paired": paired, "placed": placed, "train": train}


def listed():
    return [
        # decoder self-attention of one training step: hidden 256, batch 32, 192 denoising + 300 matching queries, their group mask
        _attn("decoder queries train", 32, 492, 492, 4, 4, 32, 64, BF16, "groups", True),
        # the encoder layer over the 30 x 30 map of a 960 x 960 image, hidden 384, inference
        _attn("encoder map forward", 8, 900, 900, 8, 8, 24, 48, BF16, "none", False),
        # the decoder layer of one image at inference: the time of a launch
        _attn("one image forward", 1, 300, 300, 4, 4, 32, 64, BF16, "none", False),
        # training in 32 bits on images padded to one size: every image has its own number of tokens
        _attn("padded batch train fp32", 16, 396, 396, 4, 4, 32, 64, FP32, "lengths", True),
        # training on one long sequence, every key head shared by four heads
        _attn("long sequence train", 1, 8192, 8192, 16, 4, 64, 128, BF16, "causal", True),
        # one new token for each of 16 sequences, over caches filled to different lengths
        _attn("one token, long caches", 16, 1, 32768, 16, 4, 64, 128, BF16, "lengths", False),
        # a few new tokens at once behind a long prefix, odd sizes
        _attn("few tokens behind a prefix", 4, 17, 10001, 8, 2, 64, 128, BF16, "causal", False),
        # queries and keys of the decoder's self-attention in a training step
        _norm("decoder heads train", 32, 492, 8, 8, 32, 32, BF16, 512, False, False, True),
        # a batch of long sequences in training, shared key heads, wide heads
        _norm("long sequences train", 4, 8192, 32, 8, 128, 128, BF16, 8192, False, False, True),
        # one new token for each of 16 sequences at far positions
        _norm("one token", 16, 1, 32, 8, 64, 64, BF16, 131072, True, True, False),
        # a 30 x 30 map in 32 bits: heads of 24 channels, 16 of them rotated
        _norm("encoder map fp32", 16, 900, 16, 16, 24, 16, FP32, 900, False, False, False),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    if rng.random() < 0.6:
        dtype = BF16 if rng.random() < 0.75 else FP32
        dim = rng.choice([8, 16, 24, 32, 40, 48, 64])
        kv_heads, share = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4])
        heads = kv_heads * share
        if rng.random() < 0.35:                                    # few new tokens over a cache
            queries, keys = _spread(rng, 1, 32), _spread(rng, 33, 40000)
            batch = _spread(rng, 1, max(1, min(32, 2 ** 27 // (keys * kv_heads * dim * 4))))
            mask, train = rng.choice(["none", "lengths", "causal"]), False
        else:
            queries = _spread(rng, 16, 4000)
            keys = queries if rng.random() < 0.75 else _spread(rng, 16, 4000)
            heads = max(heads, 6 // kv_heads * kv_heads) if heads < 6 else heads
            batch = _spread(rng, 1, max(1, min(48, 2 ** 28 // (queries * keys * heads))))
            mask = rng.choice(["none", "lengths", "rows", "groups", "causal"] if queries == keys else ["none", "lengths", "rows"])
            train = rng.random() < 0.6
        case = _attn("", batch, queries, keys, heads, kv_heads, dim, 2 * dim, dtype, mask, train)
    else:
        dim = rng.choice([8, 16, 24, 32, 48, 64, 80, 96, 128, 256])
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 4])
        dtype = BF16 if rng.random() < 0.7 else FP32
        tokens = 2 ** (27 if dtype == BF16 else 26) // ((heads + kv_heads) * dim)
        length = _spread(rng, 1, min(12000, tokens))
        batch = _spread(rng, 1, max(1, min(64, tokens // length)))
        case = _norm("", batch, length, heads, kv_heads, dim, rng.choice([dim, dim, max(8, dim // 16 * 8)]), dtype,
                     length + _spread(rng, 1, 100000), rng.random() < 0.4, rng.random() < 0.4, rng.random() < 0.6)
    del case["name"]
    return case


def _lengths(case):
    """Tokens that are valid in each sequence of a batch: between half of them and all."""
    full = case["keys"]
    return [full - int(full * 0.5 * ((b * 0.6180339887) % 1.0)) for b in range(case["batch"])]


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _blocked(case, gen):
    """The mask that goes with the call, True = may not attend: [queries, keys], or None."""
    n, m = case["queries"], case["keys"]
    if case["mask"] == "groups":               # denoising groups see themselves and the matching queries; those see only themselves
        dn = n * 2 // 5
        size = max(1, dn // 6)
        group = torch.arange(n, device="cuda") // size
        group = torch.where(torch.arange(n, device="cuda") < dn, group, -1)
        seen = (group[:, None] == group[None, :]) | (group[None, :] == -1)
        return ~seen
    if case["mask"] == "rows":                 # scattered pairs, and rows that may see nothing at all
        out = torch.rand(n, m, generator=gen, device="cuda") < 0.4
        out[torch.rand(n, generator=gen, device="cuda") < 0.1] = True
        return out
    return None


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    if case["op"] == "norm_rotate":
        b, n, h, g, d = case["batch"], case["length"], case["heads"], case["kv_heads"], case["dim"]
        packed = _normal(gen, b, n, (h + 2 * g) * d, dtype=dtype)          # the projection's output: q | k | v
        q = packed[..., :h * d].view(b, n, h, d)
        k = packed[..., h * d:(h + g) * d].view(b, n, g, d)
        angle = torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / case["rot"])
        state = {"case": case, "q": q, "k": k, "qw": 1 + 0.2 * _normal(gen, d), "kw": 1 + 0.2 * _normal(gen, d),
                 "cos": angle.cos().float(), "sin": angle.sin().float(), "places": None}
        if case["placed"]:
            state["places"] = torch.randint(0, case["table"], (b, n), generator=gen, device="cuda", dtype=torch.int32)
        if case["train"]:
            state["dq"], state["dk"] = _normal(gen, b, n, h, d, dtype=dtype), _normal(gen, b, n, g, d, dtype=dtype)
            for name in ("q", "k", "qw", "kw"):
                state[name].requires_grad_(True)
        return state
    b, n, m, h, g, d, dv = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "dim", "vdim"))
    # queries and keys as their norms leave them, values with the means that a projection's bias gives them
    if n == m:                                                             # self-attention: slices of one projection's output
        packed = _normal(gen, b, n, (2 * h + 2 * g) * d + g * dv, dtype=dtype)
        q = packed[..., :2 * h * d].view(b, n, h, 2, d)
        k = packed[..., 2 * h * d:2 * (h + g) * d].view(b, n, g, 2, d)
        v = packed[..., 2 * (h + g) * d:].view(b, n, g, dv)
    else:                                                                  # caches of their own
        q, k, v = _normal(gen, b, n, h, 2, d, dtype=dtype), _normal(gen, b, m, g, 2, d, dtype=dtype), _normal(gen, b, m, g, dv, dtype=dtype)
    v += 0.5 * _normal(gen, g, dv, dtype=dtype)
    state = {"case": case, "q": q, "k": k, "v": v, "lam": 0.1 * _normal(gen, 4, h, d), "weight": 1 + 0.2 * _normal(gen, dv),
             "blocked": _blocked(case, gen), "lengths": None, "start": None}
    # parameters of the activations' type, as in a model that is held in it
    state["lam"], state["weight"] = state["lam"].to(dtype), state["weight"].to(dtype)
    if case["mask"] == "lengths":
        state["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
    if case["mask"] == "causal":
        state["start"] = m - n
    if case["train"]:
        state["dy"] = (_normal(gen, b, n, h, dv) + 0.5 * _normal(gen, h, dv)).to(dtype)
        for name in ("q", "k", "v", "lam", "weight"):
            state[name].requires_grad_(True)
    return state


INIT, EPS = 0.4, 1e-5


# ------------------------------------------------------------------------------------------------------- one pass of a case
def _attention_own(s):
    from custom_d_fine_amd import kernels
    causal = s["start"] is not None
    return kernels.diff_attention(s["q"], s["k"], s["v"], s["lam"], INIT, norm_weight=s["weight"], norm_eps=EPS, attn_mask=s["blocked"],
                                  kv_lengths=s["lengths"], causal=causal, query_start=s["start"] if causal else 0)


def _attention_plain(s):
    q, k, v, lam = s["q"].float(), s["k"].float(), s["v"].float(), s["lam"].float()
    b, n, h, _, d = q.shape
    m, g = k.shape[1], k.shape[2]
    hidden = torch.zeros(1, 1, 1, 1, 1, 1, dtype=torch.bool, device=q.device)               # b, g, share, map, n, m
    if s["blocked"] is not None:
        hidden = hidden | s["blocked"]
    if s["lengths"] is not None:
        hidden = hidden | (torch.arange(m, device=q.device) >= s["lengths"][:, None]).view(b, 1, 1, 1, 1, m)
    if s["start"] is not None:
        hidden = hidden | (torch.arange(m, device=q.device) > torch.arange(n, device=q.device)[:, None] + s["start"])
    rows = q.view(b, n, g, h // g, 2, d).permute(0, 2, 4, 3, 1, 5).reshape(b * g * 2, h // g * n, d)
    cols = k.permute(0, 2, 3, 4, 1).reshape(b * g * 2, d, m)
    score = (torch.bmm(rows, cols) * d ** -0.5).view(b, g, 2, h // g, n, m).transpose(2, 3)
    score = score.masked_fill(hidden, -math.inf)
    top = score.detach().amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    weight = (lam[0] * lam[1]).sum(-1).exp() - (lam[2] * lam[3]).sum(-1).exp() + INIT       # [h]
    p = p[:, :, :, 0] - weight.view(1, g, h // g, 1, 1) * p[:, :, :, 1]
    vals = v.permute(0, 2, 1, 3).reshape(b * g, m, -1)
    u = torch.bmm(p.reshape(b * g, h // g * n, m), vals).view(b, g, h // g, n, -1).permute(0, 3, 1, 2, 4).reshape(b, n, h, -1)
    u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * s["weight"].float() * (1 - INIT)
    return u.to(s["q"].dtype)


def _norm_own(s):
    from custom_d_fine_amd import kernels
    return kernels.qk_norm_rotate(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], positions=s["places"], eps=EPS,
                                  interleaved=s["case"]["paired"])


def _norm_plain_one(x, weight, cos, sin, paired):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight
    r = 2 * cos.shape[-1]
    c, t = cos.unsqueeze(-2), sin.unsqueeze(-2)
    if paired:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack([a * c - b * t, b * c + a * t], -1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat([a * c - b * t, b * c + a * t], -1)
    return torch.cat([turned, y[..., r:]], -1).to(x.dtype)


def _norm_plain(s):
    places = s["places"].long() if s["places"] is not None else torch.arange(s["q"].shape[1], device="cuda")
    cos, sin, paired = s["cos"][places], s["sin"][places], s["case"]["paired"]
    return _norm_plain_one(s["q"], s["qw"], cos, sin, paired), _norm_plain_one(s["k"], s["kw"], cos, sin, paired)


def run(state):
    case = state["case"]
    if case["op"] == "norm_rotate":
        q, k = _norm_own(state) if own else _norm_plain(state)
        if not case["train"]:
            return {"q": q, "k": k}
        grads = torch.autograd.grad([q, k], [state["q"], state["k"], state["qw"], state["kw"]], [state["dq"], state["dk"]])
        return {"q": q.detach(), "k": k.detach(), "dq": grads[0], "dk": grads[1], "dqw": grads[2], "dkw": grads[3]}
    y = _attention_own(state) if own else _attention_plain(state)
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [state["q"], state["k"], state["v"], state["lam"], state["weight"]], state["dy"])
    return {"y": y.detach(), "dq": grads[0], "dk": grads[1], "dv": grads[2], "dlam": grads[3], "dweight": grads[4]}


def _pairs(case):
    """(query, key) pairs of one head that are looked at, over the batch."""
    b, n, m = case["batch"], case["queries"], case["keys"]
    if case["mask"] == "lengths":
        return n * sum(_lengths(case))
    if case["mask"] == "causal":
        return b * (n * (m - n) + n * (n + 1) // 2)
    if case["mask"] == "rows":
        return b * n * m * 0.54
    if case["mask"] == "groups":
        dn = n * 2 // 5
        return b * (n * (n - dn) + dn * max(1, dn // 6))
    return b * n * m


def work(case):
    size = 2 if case["dtype"] == BF16 else 4
    if case["op"] == "norm_rotate":
        values = case["batch"] * case["length"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        rows = case["batch"] * case["length"] if case["placed"] else case["length"]
        table = min(rows, case["table"]) * case["rot"] * 4
        # forward: read, write; with its backward: inputs once, both outputs' gradients, both results of each direction
        return {"bytes": values * size * (4 if case["train"] else 2) + table, "flops": values * (24 if case["train"] else 8)}
    b, n, h, g, d, dv = (case[x] for x in ("batch", "queries", "heads", "kv_heads", "dim", "vdim"))
    keys = sum(_lengths(case)) if case["mask"] == "lengths" else b * case["keys"]
    q, kv, out = b * n * h * 2 * d, keys * g * (2 * d + dv), b * n * h * dv
    mask = n * case["keys"] if case["mask"] in ("groups", "rows") else 0
    flops = _pairs(case) * h * (4 * d + 2 * dv)
    if case["train"]:
        return {"bytes": size * (2 * q + 2 * kv + 2 * out) + mask, "flops": flops + _pairs(case) * h * (8 * d + 4 * dv)}
    return {"bytes": size * (q + kv + out) + mask, "flops": flops}


# ----------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_norm(x, weight, cos, sin, paired, upstream):
    d, r = x.shape[-1], 2 * cos.shape[-1]
    # the rotation of one token as a d x d matrix would be [[c, -s], [s, c]] on each pair (i, j) and one elsewhere
    i = torch.arange(r // 2, device=x.device)
    i, j = (2 * i, 2 * i + 1) if paired else (i, i + r // 2)
    inv = 1.0 / ((x ** 2).sum(-1, keepdim=True) / d + EPS).sqrt()
    hat = x * inv
    n = hat * weight
    y = n.clone()
    y[..., i] = n[..., i] * cos - n[..., j] * sin
    y[..., j] = n[..., i] * sin + n[..., j] * cos
    if upstream is None:
        return y, None, None
    dn = upstream.clone()
    dn[..., i] = upstream[..., i] * cos + upstream[..., j] * sin
    dn[..., j] = upstream[..., j] * cos - upstream[..., i] * sin
    dhat = dn * weight
    dx = inv * (dhat - hat * (dhat * hat).sum(-1, keepdim=True) / d)
    return y, dx, (dn * hat).reshape(-1, d).sum(0)


def exact(case, seed):
    s = prepare(case, seed)
    f = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    if case["op"] == "norm_rotate":
        rows = s["places"].long() if s["places"] is not None else torch.arange(case["length"], device="cuda").expand(case["batch"], -1)
        cos, sin = f["cos"][rows][:, :, None], f["sin"][rows][:, :, None]
        q, dq, dqw = _exact_norm(f["q"], f["qw"], cos, sin, case["paired"], f.get("dq"))
        k, dk, dkw = _exact_norm(f["k"], f["kw"], cos, sin, case["paired"], f.get("dk"))
        return {"q": q, "k": k, "dq": dq, "dk": dk, "dqw": dqw, "dkw": dkw} if case["train"] else {"q": q, "k": k}
    b, n, m, h, g, d, dv = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "dim", "vdim"))
    dot1, dot2 = (f["lam"][0] * f["lam"][1]).sum(-1), (f["lam"][2] * f["lam"][3]).sum(-1)
    y = torch.zeros(b, n, h, dv, device="cuda", dtype=torch.float64)
    out = {"y": y}
    if case["train"]:
        out.update(dq=torch.zeros_like(f["q"]), dk=torch.zeros_like(f["k"]), dv=torch.zeros_like(f["v"]),
                   dlam=torch.zeros_like(f["lam"]), dweight=torch.zeros_like(f["weight"]))
    lens = _lengths(case) if case["mask"] == "lengths" else [m] * b
    step = max(1, min(b, 2 ** 26 // (n * m)))                              # batch entries at a time
    for at in range(0, b, step):
        e = slice(at, min(b, at + step))
        seen = torch.arange(m, device="cuda") < torch.tensor(lens[e], device="cuda")[:, None, None]
        seen = seen.expand(-1, n, m).clone()
        if s["blocked"] is not None:
            seen &= ~s["blocked"]
        if case["mask"] == "causal":
            seen &= torch.arange(m, device="cuda") - torch.arange(n, device="cuda")[:, None] <= m - n
        for head in range(h):
            kv = head // (h // g)
            lam = dot1[head].exp() - dot2[head].exp() + INIT
            maps, vals = [], f["v"][e, :, kv].contiguous()
            for t in range(2):
                logit = torch.bmm(f["q"][e, :, head, t].contiguous(), f["k"][e, :, kv, t].transpose(1, 2).contiguous()) / math.sqrt(d)
                logit.masked_fill_(~seen, -math.inf)
                a = torch.softmax(logit, -1)
                maps.append(torch.nan_to_num_(a, nan=0.0))                 # a row that sees nothing takes nothing
                del logit, a
            o1, o2 = torch.bmm(maps[0], vals), torch.bmm(maps[1], vals)
            u = o1 - lam * o2
            inv = 1.0 / ((u ** 2).sum(-1, keepdim=True) / dv + EPS).sqrt()
            y[e, :, head] = (1 - INIT) * u * inv * f["weight"]
            if not case["train"]:
                continue
            dy = (1 - INIT) * f["dy"][e, :, head]
            out["dweight"] += (dy * u * inv).sum((0, 1))
            t = dy * f["weight"]
            du = inv * (t - u * inv ** 2 * (t * u).sum(-1, keepdim=True) / dv)
            out["dv"][e, :, kv] += torch.bmm((maps[0] - lam * maps[1]).transpose(1, 2).contiguous(), du)
            da = torch.bmm(du, vals.transpose(1, 2).contiguous())
            for t, (a, o, c) in enumerate(((maps[0], o1, 1.0), (maps[1], o2, -lam))):
                ds = c * a * (da - (du * o).sum(-1, keepdim=True)) / math.sqrt(d)
                out["dq"][e, :, head, t] = torch.bmm(ds, f["k"][e, :, kv, t].contiguous())
                out["dk"][e, :, kv, t] += torch.bmm(ds.transpose(1, 2).contiguous(), f["q"][e, :, head, t].contiguous())
            dl = -(du * o2).sum()
            out["dlam"][0, head] += dl * dot1[head].exp() * f["lam"][1, head]
            out["dlam"][1, head] += dl * dot1[head].exp() * f["lam"][0, head]
            out["dlam"][2, head] -= dl * dot2[head].exp() * f["lam"][3, head]
            out["dlam"][3, head] -= dl * dot2[head].exp() * f["lam"][2, head]
    return out
