"""The operators on the tokens of rendered views (`mvtn_amd.tokens`), in their plain form and as the framework's calls: what they compute,
on which sizes, and what one pass cannot do without.

Tokens are the 16 x 16 patches of 224 x 224 views, 14 x 14 = 196 a view: an object of 12 views has 2352 tokens, one of 20 has 3920.  Three
operators: rotary positions with several axes ("rotate"), attention over an object's tokens ("attend"), and the norms around a block with
its gate and residual scale ("norm")."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---- cases ----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one object, one token a view (pooled features of 12 views): a call whose latency counts
        dict(name="rotate_12_tokens", op="rotate", batch=1, tokens=12, heads=12, dim=64, sections="16,16", periods="360,360", base=100.0,
             interleaved=False, type="fp32", far=180.0, grad="none"),
        # queries and keys of a training batch (16 objects x 12 views) rotated by camera and patch: forward and backward, cameras learned
        dict(name="rotate_batch_cameras", op="rotate", batch=16, tokens=2352, heads=24, dim=64, sections="8,8,8,8", periods="360,360,0,0", base=100.0,
             interleaved=False, type="bf16", far=180.0, grad="positions"),
        # three axes (frame, row, column) of a long odd sequence, far positions, part of each head left as it is, neighbouring pairs; x's gradient only
        dict(name="rotate_video_odd", op="rotate", batch=3, tokens=10007, heads=5, dim=80, sections="9,11,13", periods="0,0,0", base=10000.0,
             interleaved=True, type="fp16", far=100000.0, grad="x"),
        # attention within each view: 192 views of 196 tokens, evaluation
        dict(name="attend_views_eval", op="attend", batch=192, queries=196, keys=196, heads=12, kv_heads=12, dim=64, groups=1, drop=0.0, type="bf16",
             backward=False),
        # attention over all tokens of an object, a training step of 16 objects x 12 views with view dropout
        dict(name="attend_objects_train", op="attend", batch=16, queries=2352, keys=2352, heads=12, kv_heads=12, dim=64, groups=12, drop=0.25,
             type="bf16", backward=True),
        # the largest: 8 objects (one GPU's share of 64) x 20 views, heads of 128, training
        dict(name="attend_largest_train", op="attend", batch=8, queries=3920, keys=3920, heads=16, kv_heads=16, dim=128, groups=1, drop=0.0,
             type="bf16", backward=True),
        # one query per object pools all its tokens: few rows, a long axis; training, 64 objects x 20 views
        dict(name="attend_pool_train", op="attend", batch=64, queries=1, keys=3920, heads=16, kv_heads=4, dim=128, groups=20, drop=0.25, type="bf16",
             backward=True),
        # the 12 views' pooled features of two objects, some object with every view dropped, odd head size, shared heads: latency
        dict(name="attend_small_odd", op="attend", batch=2, queries=13, keys=36, heads=6, kv_heads=2, dim=40, groups=12, drop=0.6, type="fp16",
             backward=True),
        # the pooled features of 12 views: latency
        dict(name="norm_12_tokens", op="norm", batch=1, tokens=12, dim=384, kind="layer", post=False, gate="none", views=1, drop=0.0, residual="fp32",
             branch="fp32", weights="fp32", backward=False),
        # a block's end in a training batch, 16-bit residual stream, both norms, a gate per object, views dropped whole
        dict(name="norm_batch_train", op="norm", batch=16, tokens=2352, dim=768, kind="rms", post=True, gate="object", views=12, drop=0.25,
             residual="bf16", branch="bf16", weights="bf16", backward=True),
        # the whole evaluation batch of 64 objects x 20 views, 32-bit residual stream under 16-bit branches
        dict(name="norm_largest_eval", op="norm", batch=64, tokens=3920, dim=1024, kind="layer", post=False, gate="channel", views=1, drop=0.0,
             residual="fp32", branch="bf16", weights="fp32", backward=False),
        # odd width, 32-bit residual stream, training
        dict(name="norm_odd_train", op="norm", batch=5, tokens=1961, dim=837, kind="layer", post=True, gate="object", views=1, drop=0.0, residual="fp32",
             branch="fp16", weights="fp32", backward=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "attend", "norm"])
    if op == "rotate":
        axes = rng.randint(1, 4)
        sections = [rng.randint(2, 16) for _ in range(axes)]
        pairs = sum(sections)
        dim = 2 * pairs + rng.choice([0, 0, 2, 6, 16])
        heads, batch = rng.choice([1, 3, 8, 12, 16, 24]), rng.randint(1, 16)
        tokens = _log(rng, 1, max(2, min(20000, 60000000 // (batch * heads * dim))))
        periods = [rng.choice([0, 360]) for _ in range(axes)]
        return dict(op=op, batch=batch, tokens=tokens, heads=heads, dim=dim, sections=",".join(map(str, sections)), periods=",".join(map(str, periods)),
                    base=rng.choice([100.0, 10000.0]), interleaved=rng.random() < 0.5, type=rng.choice(["bf16", "fp16", "fp32"]),
                    far=float(_log(rng, 10, 100000)), grad=rng.choice(["none", "x", "positions"]))
    if op == "attend":
        dim = rng.choice([32, 40, 64, 64, 72, 96, 128, 128])
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        heads = kv_heads * rng.choice([1, 1, 1, 2, 4])
        groups = rng.choice([1, 4, 12, 20])
        keys = groups * _log(rng, 1, 4000 // groups)
        queries = keys if rng.random() < 0.6 else _log(rng, 1, 4000)
        most = 8 * 16 * 3920 * 3920 * 128
        batch = min(_log(rng, 1, 64), max(1, most // (heads * queries * keys * 128)))
        return dict(op=op, batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads, dim=dim, groups=groups,
                    drop=0.0 if groups == 1 else rng.choice([0.0, 0.25, 0.5]), type=rng.choice(["bf16", "bf16", "fp16"]), backward=rng.random() < 0.6)
    batch, dim = rng.randint(1, 32), rng.choice([rng.randint(1, 400), 384, 512, 768, 1024, rng.randint(400, 2100), 2048])
    views = rng.choice([1, 4, 12, 20])
    tokens = views * _log(rng, 1, max(2, min(400, 60000000 // (batch * dim * views))))
    residual, branch, weights = rng.choice([("bf16", "bf16", "bf16"), ("fp16", "fp16", "fp16"), ("fp32", "fp32", "fp32"), ("fp32", "bf16", "fp32"),
                                            ("fp32", "fp16", "fp32")])
    return dict(op=op, batch=batch, tokens=tokens, dim=dim, kind=rng.choice(["rms", "layer"]), post=rng.random() < 0.5,
                gate=rng.choice(["none", "channel", "object"]), views=views, drop=0.0 if views == 1 else 0.25, residual=residual, branch=branch,
                weights=weights, backward=rng.random() < 0.6)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _numbers(text):
    return [int(x) for x in text.split(",")]


def _turns(case):
    """Turns per unit of position of every pair, 64 bits, and the pair's axis: whole harmonics on a periodic axis, a geometric ladder of radians
    on an open one."""
    turns, axis = [], []
    for a, (n, period) in enumerate(zip(_numbers(case["sections"]), _numbers(case["periods"]))):
        turns += [(j + 1) / period if period else case["base"] ** (-j / n) / (2 * math.pi) for j in range(n)]
        axis += [a] * n
    return torch.tensor(turns, dtype=torch.float64), torch.tensor(axis)


def _view_scale(g, batch, views, drop):
    """View dropout's draws: 0 for a dropped view, 1 / (1 - drop) for the others."""
    kept = torch.rand(batch, views, generator=g, device="cuda") >= drop
    return kept.float() / (1.0 - drop)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, type="fp32", scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(TYPES[type])

    s = {"case": case}
    if case["op"] == "rotate":
        b, n, h, d = case["batch"], case["tokens"], case["heads"], case["dim"]
        axes = len(_numbers(case["sections"]))
        s["x"] = normal(b, n, h, d, type=case["type"])
        u = torch.rand(b, n, axes, generator=g, device="cuda") * 2 - 1
        # cameras' angles are real numbers; rows, columns and frames are whole ones
        periodic = torch.tensor(_numbers(case["periods"]), device="cuda") > 0
        s["positions"] = torch.where(periodic, u * 180.0, (u * case["far"]).round())
        s["turns"], s["axis"] = (t.cuda() for t in _turns(case))
        if case["grad"] != "none":
            s["dy"] = normal(b, n, h, d, type=case["type"])
    elif case["op"] == "attend":
        b, q, k, h, e, d, t = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "dim", "type"))
        s["q"], s["k"], s["v"] = normal(b, q, h, d, type=t), normal(b, k, e, d, type=t), normal(b, k, e, d, type=t)
        s["keep"] = _view_scale(g, b, case["groups"], case["drop"]) != 0 if case["drop"] else None
        if case["drop"] >= 0.6:
            s["keep"][-1] = False
        if case["backward"]:
            s["do"] = normal(b, q, h, d, type=t)
    else:
        b, n, d = case["batch"], case["tokens"], case["dim"]
        s["residual"], s["branch"] = normal(b, n, d, type=case["residual"], scale=2.0, mean=0.1), normal(b, n, d, type=case["branch"], mean=0.1)
        w = case["weights"]
        s["weight"], s["bias"] = normal(d, type=w, scale=0.2, mean=1.0), normal(d, type=w, scale=0.2) if case["kind"] == "layer" else None
        s["post"] = normal(d, type=w, scale=0.2, mean=1.0) if case["post"] else None
        s["gate"] = None if case["gate"] == "none" else normal(d, type=w, scale=0.3) if case["gate"] == "channel" else normal(b, d, type=w, scale=0.3)
        s["scale"] = _view_scale(g, b, case["views"], case["drop"]) if case["drop"] else None
        if case["backward"]:
            s["dy"], s["dz"] = normal(b, n, d, type=case["residual"]), normal(b, n, d, type=case["branch"])
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _rotate(state) if op == "rotate" else _attend(state) if op == "attend" else _norm(state)


def _own(s):
    from mvtn_amd import tokens
    c = s["case"]
    if c["op"] == "rotate":
        rotary = s.get("rotary")
        if rotary is None:
            rotary = s["rotary"] = tokens.TokenRotary(_numbers(c["sections"]), base=c["base"], periods=_numbers(c["periods"]), interleaved=c["interleaved"])
        if c["grad"] == "none":
            return rotary(s["x"], s["positions"])
        x, p = s["x"].detach().requires_grad_(), s["positions"].detach()
        leaves = [x, p.requires_grad_()] if c["grad"] == "positions" else [x]
        y = rotary(x, p)
        return (y.detach(),) + torch.autograd.grad(y, leaves, s["dy"])
    if c["op"] == "attend":
        if not c["backward"]:
            return tokens.attend_tokens(s["q"], s["k"], s["v"], keep=s["keep"])
        leaves = [s[x].detach().requires_grad_() for x in ("q", "k", "v")]
        o = tokens.attend_tokens(*leaves, keep=s["keep"])
        return (o.detach(),) + torch.autograd.grad(o, leaves, s["do"])
    names = [x for x in ("residual", "branch", "weight", "bias", "post", "gate") if s[x] is not None]
    leaves = {x: s[x].detach().requires_grad_() if c["backward"] else s[x] for x in names}
    y, z = tokens.add_norm_tokens(leaves["residual"], leaves["branch"], leaves["weight"], leaves.get("bias"), post_weight=leaves.get("post"),
                                  gate=leaves.get("gate"), scale=s["scale"], kind=c["kind"])
    if not c["backward"]:
        return y, z
    return (y.detach(), z.detach()) + torch.autograd.grad((y, z), [leaves[x] for x in names], (s["dy"], s["dz"]))


def _pairs(x, n, interleaved):
    return (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])


def _joined(a, b, rest, interleaved):
    both = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((both, rest), -1)


def _rotate(s):
    c, n = s["case"], s["turns"].numel()
    part = s["positions"].double()[..., s["axis"]] * s["turns"]
    angle = (part - part.round()) * (2 * math.pi)
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    x = s["x"].float()
    x1, x2 = _pairs(x, n, c["interleaved"])
    y = _joined(x1 * cos - x2 * sin, x1 * sin + x2 * cos, x[..., 2 * n:], c["interleaved"]).to(s["x"].dtype)
    if c["grad"] == "none":
        return y
    dy = s["dy"].float()
    d1, d2 = _pairs(dy, n, c["interleaved"])
    e1, e2 = d1 * cos + d2 * sin, d2 * cos - d1 * sin
    dx = _joined(e1, e2, dy[..., 2 * n:], c["interleaved"]).to(s["x"].dtype)
    if c["grad"] == "x":
        return y, dx
    slope = (x1 * e2 - x2 * e1).sum(2) * (2 * math.pi * s["turns"]).float()
    of_axis = (s["axis"][:, None] == torch.arange(s["positions"].shape[-1], device=slope.device)).float()
    return y, dx, torch.matmul(slope, of_axis)


def _attend(s):
    c = s["case"]
    b, h, e, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    scale = d ** -0.5
    q = s["q"].float().reshape(b, -1, e, h // e, d).permute(0, 2, 3, 1, 4)         # (B, kv heads, heads of a group, queries, D)
    k, v = (s[x].float().permute(0, 2, 1, 3)[:, :, None] for x in ("k", "v"))      # (B, kv heads, 1, keys, D)
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    if s["keep"] is not None:
        gone = ~s["keep"].repeat_interleave(c["keys"] // c["groups"], 1)[:, None, None, None]
        p.masked_fill_(gone, -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    o = torch.matmul(p, v)

    def back(x, heads):
        return x.permute(0, 3, 1, 2, 4).reshape(b, -1, heads, d).to(s["q"].dtype)

    if not c["backward"]:
        return back(o, h)
    do = s["do"].float().reshape(b, -1, e, h // e, d).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2, keepdim=True)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    dq, dk = torch.matmul(ds, k).mul_(scale), torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True).mul_(scale)
    return back(o, h), back(dq, h), back(dk, e), back(dv, e)


EPS = 1e-6


def _normed(x, kind):
    """(x - mean) / std and 1 / std of the rows (no mean for rms)."""
    x = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return x * r, r


def _normed_backward(g, hat, r, kind):
    g = g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True) if kind == "layer" else g - hat * (g * hat).mean(-1, keepdim=True)
    return g * r


def _norm(s):
    c, kind = s["case"], s["case"]["kind"]
    a, dim = s["branch"].float(), c["dim"]
    if s["scale"] is not None:
        scale = s["scale"].repeat_interleave(c["tokens"] // c["views"], 1)[..., None]
    else:
        scale = torch.ones((), device=a.device)
    gate = torch.ones((), device=a.device) if s["gate"] is None else s["gate"].float()[:, None] if c["gate"] == "object" else s["gate"].float()
    post = torch.ones((), device=a.device) if s["post"] is None else s["post"].float()
    hat, r = _normed(a, kind) if s["post"] is not None else (a, None)
    y = s["residual"].float() + scale * (gate * (post * hat))
    yhat, yr = _normed(y, kind)
    w = s["weight"].float()
    z = yhat * w
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, z = y.to(s["residual"].dtype), z.to(s["branch"].dtype)
    if not c["backward"]:
        return y, z
    dz = s["dz"].float()
    dy = s["dy"].float() + _normed_backward(dz * w, yhat, yr, kind)
    dn = scale * gate * dy
    da = _normed_backward(dn * post, hat, r, kind) if s["post"] is not None else dn
    out = [y, z, dy.to(y.dtype), da.to(s["branch"].dtype), (dz * yhat).sum((0, 1)).to(s["weight"].dtype)]
    if s["bias"] is not None:
        out.append(dz.sum((0, 1)).to(s["bias"].dtype))
    if s["post"] is not None:
        out.append((dn * hat).sum((0, 1)).to(s["post"].dtype))
    if s["gate"] is not None:
        dgate = scale * (post * hat) * dy
        out.append((dgate.sum(1) if c["gate"] == "object" else dgate.sum((0, 1))).to(s["gate"].dtype))
    return tuple(out)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    if case["op"] == "rotate":
        size, pos = case["batch"] * case["tokens"] * case["heads"] * case["dim"] * BYTES[case["type"]], case["batch"] * case["tokens"] * 4 * (1 + case["sections"].count(","))
        n = case["batch"] * case["tokens"] * case["heads"] * sum(_numbers(case["sections"]))
        if case["grad"] == "none":
            return {"bytes": 2 * size + pos, "flops": 6 * n}
        # forward: x -> y; backward: dy -> dx, and x again where the positions' gradient is asked for
        return {"bytes": 4 * size + 2 * pos + (size + pos if case["grad"] == "positions" else 0), "flops": (12 if case["grad"] == "x" else 16) * n}
    if case["op"] == "attend":
        e = BYTES[case["type"]]
        rows = case["batch"] * case["queries"] * case["heads"] * case["dim"]
        cols = case["batch"] * case["keys"] * case["kv_heads"] * case["dim"]
        product = 2 * rows * case["keys"] * (1 - case["drop"])
        if not case["backward"]:
            return {"bytes": (2 * rows + 2 * cols) * e, "flops": 2 * product}
        # forward: q, k, v -> o; backward: q, k, v, o, do -> dq, dk, dv; 2 products forward, 5 backward
        return {"bytes": (6 * rows + 6 * cols) * e, "flops": 7 * product}
    n = case["batch"] * case["tokens"] * case["dim"]
    r, b = BYTES[case["residual"]], BYTES[case["branch"]]
    if not case["backward"]:
        return {"bytes": 2 * n * (r + b), "flops": 14 * n}
    # forward: residual, branch -> y, z; backward: y, branch, dy, dz -> their gradients
    return {"bytes": n * (2 * (r + b) + (r + b + r + b) + (r + b)), "flops": 40 * n}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "attend": _exact_attend, "norm": _exact_norm}[case["op"]](case, s)


def _exact_rotate(case, s):
    """Pairs as complex numbers: y = x e^(i angle); the gradients follow from y = x e^(i angle) by the product rule."""
    n = s["turns"].numel()

    def complex_of(t):
        t = t.double()
        return torch.complex(t[..., 0:2 * n:2].contiguous(), t[..., 1:2 * n:2].contiguous()) if case["interleaved"] else \
            torch.complex(t[..., :n].contiguous(), t[..., n:2 * n].contiguous())

    def real_of(z, t):
        out = t.double().clone()
        if case["interleaved"]:
            out[..., 0:2 * n:2], out[..., 1:2 * n:2] = z.real, z.imag
        else:
            out[..., :n], out[..., n:2 * n] = z.real, z.imag
        return out

    angle = torch.remainder(s["positions"].double()[:, :, s["axis"]] * s["turns"], 1.0) * (2 * math.pi)
    e = torch.polar(torch.ones_like(angle), angle)[:, :, None, :]
    y = complex_of(s["x"]) * e
    if case["grad"] == "none":
        return real_of(y, s["x"])
    dy = complex_of(s["dy"])
    dx = real_of(dy * e.conj(), s["dy"])
    if case["grad"] == "x":
        return real_of(y, s["x"]), dx
    slope = (dy.conj() * (y * 1j)).real.sum(2) * (2 * math.pi) * s["turns"]
    dpos = torch.stack([slope[..., s["axis"] == a].sum(-1) for a in range(s["positions"].shape[-1])], -1)
    return real_of(y, s["x"]), dx, dpos


def _exact_attend(case, s):
    """Object by object and head by head (groups of heads together), from softmax's definition over the kept keys only."""
    outs = []
    ratio = case["heads"] // case["kv_heads"]
    c = case["dim"] ** -0.5
    for b in range(case["batch"]):
        kept = torch.ones(case["keys"], dtype=torch.bool, device="cuda")
        if s["keep"] is not None:
            kept = s["keep"][b][torch.arange(case["keys"], device="cuda") // (case["keys"] // case["groups"])]
        at = kept.nonzero()[:, 0]
        q = s["q"][b].double().transpose(0, 1)                                                     # (heads, queries, D)
        k, v = (s[x][b][at].double().repeat_interleave(ratio, 1).transpose(0, 1) for x in ("k", "v"))   # (heads, kept, D)
        p = torch.softmax((q @ k.mT) * c, -1) if at.numel() else q.new_zeros(*q.shape[:2], 0)
        o = p @ v
        got = [o.transpose(0, 1)]
        if case["backward"]:
            do = s["do"][b].double().transpose(0, 1)
            dp = do @ v.mT
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            got.append((ds @ k * c).transpose(0, 1))
            for g in (ds.mT @ q * c, p.mT @ do):
                full = g.new_zeros(case["keys"], case["kv_heads"], case["dim"])
                full[at] = g.reshape(case["kv_heads"], ratio, -1, case["dim"]).sum(1).transpose(0, 1)
                got.append(full)
        outs.append(got)
    outs = [torch.stack(x) for x in zip(*outs)]
    return tuple(outs) if case["backward"] else outs[0]


def _exact_norm(case, s):
    """The forward in 64 bits as written in the definition, the gradients by automatic differentiation of it; in parts of the batch, each
    object's own gradients as they are and the shared ones summed."""
    shared = [x for x in ("weight", "bias", "post") if s[x] is not None] + (["gate"] if case["gate"] == "channel" else [])
    sums, rows = {x: 0.0 for x in shared}, []
    for b in range(case["batch"]):
        t = {x: s[x].double() for x in shared}
        t |= {"residual": s["residual"][b].double(), "branch": s["branch"][b].double()}
        if case["gate"] == "object":
            t["gate"] = s["gate"][b].double()
        with torch.enable_grad():
            t = {x: u.requires_grad_(case["backward"]) for x, u in t.items()}

            def norm(u):
                if case["kind"] == "layer":
                    u = u - u.mean(1, keepdim=True)
                return u / torch.sqrt((u ** 2).mean(1, keepdim=True) + EPS)

            n = norm(t["branch"]) * t["post"] if "post" in t else t["branch"]
            if "gate" in t:
                n = n * t["gate"]
            if s["scale"] is not None:
                n = n * s["scale"][b].double().repeat_interleave(case["tokens"] // case["views"])[:, None]
            y = t["residual"] + n
            z = norm(y) * t["weight"]
            if "bias" in t:
                z = z + t["bias"]
            got = {"y": y.detach(), "z": z.detach()}
            if case["backward"]:
                grads = torch.autograd.grad((y, z), list(t.values()), (s["dy"][b].double(), s["dz"][b].double()))
                for x, u in zip(t, grads):
                    if x in shared:
                        sums[x] = sums[x] + u
                    else:
                        got[x] = u
        rows.append(got)
    full = {x: torch.stack([r[x] for r in rows]) for x in rows[0]} | (sums if case["backward"] else {})
    order = ["y", "z"] + ([x for x in ("residual", "branch", "weight", "bias", "post", "gate") if x in full] if case["backward"] else [])
    return tuple(full[x] for x in order)
