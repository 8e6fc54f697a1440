"""
The cases that the adapter, layer-norm and rotary operators are measured on, their plain torch forms and their 64-bit values.

``listed`` / ``draw`` give cases, ``prepare`` makes a case's inputs, ``run`` makes one pass (plain torch operations, or this
package's operators when ``own`` is set), ``work`` counts the bytes and operations a pass cannot do without and ``exact``
evaluates the definitions in 64 bits.
"""

import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # serving, smallest calls: one row per request through the modulation linear of a block (hidden -> 6 hidden)
        {"name": "lora rows of 24 requests", "op": "lora", "train": False, "rows": 24, "requests": 24, "adapters": 16, "k": 3072, "n": 18432, "rank": 16, "dtype": "bf16", "rest": 0},
        # serving: the fused QKV projection of four images of different sizes, three adapters
        {"name": "lora qkv of 4 images", "op": "lora", "train": False, "rows": 7577, "requests": 4, "adapters": 3, "k": 3072, "n": 9216, "rank": 32, "dtype": "bf16", "rest": 0},
        # serving: the second MLP linear, nine ragged requests, some without an adapter, rows behind the last request
        {"name": "lora mlp of 9 requests", "op": "lora", "train": False, "rows": 5003, "requests": 9, "adapters": 8, "k": 12288, "n": 3072, "rank": 64, "dtype": "fp16", "rest": 37},
        # training on small images: square output projection, four adapters over five samples
        {"name": "lora train output", "op": "lora", "train": True, "rows": 1333, "requests": 5, "adapters": 4, "k": 2048, "n": 2048, "rank": 16, "dtype": "fp16", "rest": 5},
        # training: two full-size samples of one adapter each through the QKV projection
        {"name": "lora train qkv", "op": "lora", "train": True, "rows": 9216, "requests": 2, "adapters": 2, "k": 3072, "n": 9216, "rank": 64, "dtype": "bf16", "rest": 0},
        # rotation of the text rows of two prompts
        {"name": "rotary text rows", "op": "rotary", "train": False, "batch": 2, "text": 77, "frames": 0, "height": 0, "width": 0, "heads": 24, "kv_heads": 24, "dim": 128, "axes": "16,56,56", "half": False, "packed": False, "dtype": "bf16"},
        # one image's joint text and image rows, Q and K as views of the packed QKV projection
        {"name": "rotary image views", "op": "rotary", "train": False, "batch": 1, "text": 512, "frames": 1, "height": 64, "width": 64, "heads": 24, "kv_heads": 24, "dim": 128, "axes": "16,56,56", "half": False, "packed": True, "dtype": "bf16"},
        # training on a video clip: time, height and width, half-split pairs, fewer K heads
        {"name": "rotary video train", "op": "rotary", "train": True, "batch": 1, "text": 226, "frames": 21, "height": 30, "width": 52, "heads": 24, "kv_heads": 8, "dim": 128, "axes": "44,42,42", "half": True, "packed": False, "dtype": "fp16"},
        # the (sin, cos) table of one large image and its text, as the fused QKV epilogue reads it
        {"name": "rotary table", "op": "table", "text": 256, "frames": 1, "height": 83, "width": 83, "axes": "16,56,56"},
        # smallest training call of a norm: the rows of two prompts, everything in 32 bits
        {"name": "norm train small", "op": "norm", "batch": 2, "rows": 77, "dim": 1152, "mod": False, "dtype": "fp32", "wdtype": "fp32"},
        # adaptive norm of two full-size samples: scale and shift per sample
        {"name": "norm train modulated", "op": "norm", "batch": 2, "rows": 4608, "dim": 3072, "mod": True, "dtype": "bf16", "wdtype": "bf16"},
        # norm with weight and bias over a video's rows, weights kept in 32 bits
        {"name": "norm train video", "op": "norm", "batch": 1, "rows": 32761, "dim": 5120, "mod": False, "dtype": "fp16", "wdtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    limit = max(_bytes(c) for c in listed())
    while True:
        op = rng.choice(["lora", "lora", "lora", "rotary", "rotary", "table", "norm", "norm"])
        if op == "lora":
            train = rng.random() < 0.5
            rows = _log(rng, 16 if train else 1, 12000)
            c = {"op": op, "train": train, "rows": rows, "requests": min(rows, _log(rng, 1, 16 if train else 64)), "adapters": _log(rng, 1, 16),
                 "k": 8 * _log(rng, 32, 1536), "n": 8 * _log(rng, 32, 2304), "rank": rng.choice([16, 16, 32, 32, 48, 64, 128]),
                 "dtype": rng.choice(["bf16", "fp16"]), "rest": rng.choice([0, 0, 1, 13])}
            c["rest"] = min(c["rest"], rows - c["requests"])
        elif op in ("rotary", "table"):
            frames = rng.choice([0, 1, 1, _log(rng, 2, 24)])
            c = {"op": op, "text": _log(rng, 1, 512) if frames == 0 else rng.choice([0, _log(rng, 1, 512)]), "frames": frames,
                 "height": _log(rng, 4, 80) if frames else 0, "width": _log(rng, 4, 80) if frames else 0}
            dim = rng.choice([64, 72, 96, 128, 128, 128])
            a = 2 * rng.randint(2, dim // 8)
            b = 2 * rng.randint(4, (dim - a) // 4)
            c["axes"] = rng.choice(["%d,%d,%d" % (a, b, b), "%d,%d,%d" % (a, b, dim - a - b), "%d,%d" % (dim // 2, dim // 2)])
            if op == "rotary":
                heads = rng.choice([1, 4, 10, 12, 16, 24, 30])
                c.update({"train": rng.random() < 0.4, "batch": rng.choice([1, 1, 2, 3]), "heads": heads, "kv_heads": rng.choice([heads, heads, 1, max(1, heads // 2)]),
                          "dim": dim, "half": rng.random() < 0.4, "packed": rng.random() < 0.4, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])})
        else:
            dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
            c = {"op": op, "batch": rng.choice([1, 1, 2, 3]), "rows": _log(rng, 1, 33000), "dim": rng.choice([_log(rng, 8, 8200), 8 * _log(rng, 8, 1024), 128 * _log(rng, 1, 64)]),
                 "mod": rng.random() < 0.5, "dtype": dt, "wdtype": rng.choice([dt, "fp32"])}
        if _bytes(c) <= limit:
            return c


def _requests(case):
    """Lengths and adapters of a case's requests: ragged, every fifth request without an adapter when some rows are left over."""
    rng = random.Random("%d %d %d" % (case["rows"], case["requests"], case["adapters"]))
    total, n = case["rows"] - case["rest"], case["requests"]
    if total == n:
        lengths = [1] * n
    else:
        cuts = sorted(rng.sample(range(1, total), n - 1))
        lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    return lengths, [-1 if case["rest"] and i % 5 == 4 else i % case["adapters"] for i in range(n)]


def _tokens(case):
    return case["text"] + case["frames"] * case["height"] * case["width"]


def _axes(case):
    return [int(a) for a in case["axes"].split(",")]


def _bytes(case):
    op = case["op"]
    if op == "lora":
        t, k, n, r = case["rows"], case["k"], case["n"], case["rank"]
        used = len({a for a in _requests(case)[1] if a >= 0})
        if case["train"]:  # x, base and dy read, out and dx written; every used factor read, every factor's gradient written
            return 2 * t * (2 * k + 3 * n) + 2 * (used + case["adapters"]) * r * (k + n)
        return 2 * t * (k + 2 * n) + 2 * used * r * (k + n)
    if op == "rotary":
        b = 2 * case["batch"] * _tokens(case) * (case["heads"] + case["kv_heads"]) * case["dim"] * SIZES[case["dtype"]]
        return b * (2 if case["train"] else 1)
    if op == "table":
        return _tokens(case) * (4 * sum(_axes(case)) + 4 * len(_axes(case)))
    g = case["batch"] if case["mod"] else 1
    return 4 * case["batch"] * case["rows"] * case["dim"] * SIZES[case["dtype"]] + 4 * g * case["dim"] * SIZES[case["wdtype"]]


def work(case):
    op = case["op"]
    if op == "lora":
        lengths, adapters = _requests(case)
        live = sum(t for t, a in zip(lengths, adapters) if a >= 0)
        flops = 2 * live * case["rank"] * (case["k"] + case["n"]) * (3 if case["train"] else 1)
    elif op == "rotary":
        flops = 3 * case["batch"] * _tokens(case) * (case["heads"] + case["kv_heads"]) * sum(_axes(case)) * (2 if case["train"] else 1)
    elif op == "table":
        flops = 2 * _tokens(case) * sum(_axes(case))
    else:
        flops = 20 * case["batch"] * case["rows"] * case["dim"]
    return {"bytes": _bytes(case), "flops": flops}


# ----------------------------------------------------------------------------------------------------------------- inputs
def _ids(case, dev):
    """Position ids (S, axes): text rows first, numbered behind the largest extent of the grid, then the grid's rows
    (frame, y, x); the last axes of them where there are fewer than three."""
    n = len(_axes(case))
    f, h, w, text = case["frames"], case["height"], case["width"], case["text"]
    grid = torch.stack(torch.meshgrid(torch.arange(f, device=dev), torch.arange(h, device=dev), torch.arange(w, device=dev), indexing="ij"), -1).reshape(-1, 3)
    first = max(f, h, w)
    rows = torch.arange(first, first + text, device=dev)[:, None].expand(text, 3)
    return torch.cat([rows, grid])[:, 3 - n:].to(torch.float32).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, scale=1.0, add=0.0, dtype="fp32"):
        return (torch.randn(shape, generator=g, device=dev) * scale + add).to(DTYPES[dtype])

    op, s = case["op"], {"case": case}
    if op == "lora":
        t, k, n, r, dt = case["rows"], case["k"], case["n"], case["rank"], case["dtype"]
        lengths, adapters = _requests(case)
        ends = [0]
        for v in lengths:
            ends.append(ends[-1] + v)
        s["offsets"] = torch.tensor(ends, dtype=torch.int32, device=dev)
        s["adapters"] = torch.tensor(adapters, dtype=torch.int32, device=dev)
        s["x"], s["base"] = normal(t, k, dtype=dt), normal(t, n, dtype=dt)
        s["down"] = normal(case["adapters"], r, k, scale=k**-0.5, dtype=dt)
        s["up"] = normal(case["adapters"], n, r, scale=0.5 * r**-0.5, dtype=dt)
        s["scale"] = torch.rand(case["adapters"], generator=g, device=dev) + 0.5
        if case["train"]:
            s["dy"] = normal(t, n, dtype=dt)
            for v in ("x", "down", "up"):
                s[v].requires_grad_(True)
    elif op in ("rotary", "table"):
        s["ids"] = _ids(case, dev) + float(int(seed) % 7)  # crops and clips start anywhere
        s["axes"] = _axes(case)
        if op == "rotary":
            b, t, h, hk, d, dt = case["batch"], _tokens(case), case["heads"], case["kv_heads"], case["dim"], case["dtype"]
            if case["packed"]:
                qkv = normal(b, t, (h + 2 * hk) * d, dtype=dt)
                s["q"], s["k"] = qkv[..., : h * d].view(b, t, h, d), qkv[..., h * d : (h + hk) * d].view(b, t, hk, d)
            else:
                s["q"], s["k"] = normal(b, t, h, d, dtype=dt), normal(b, t, hk, d, dtype=dt)
            if case["train"]:
                s["q"], s["k"] = s["q"].detach().requires_grad_(True), s["k"].detach().requires_grad_(True)
                s["dq"], s["dk"] = normal(b, t, h, d, dtype=dt), normal(b, t, hk, d, dtype=dt)
    else:
        b, t, d = case["batch"], case["rows"], case["dim"]
        shape = (b, d) if case["mod"] else (d,)
        s["x"] = (normal(b, t, d, scale=2.0) * (1 + 4 * (torch.rand(d, generator=g, device=dev) < 0.02)) + 0.5).to(DTYPES[case["dtype"]]).requires_grad_(True)
        s["w"] = normal(*shape, scale=0.2, add=0.0 if case["mod"] else 1.0, dtype=case["wdtype"]).requires_grad_(True)
        s["b"] = normal(*shape, scale=0.2, dtype=case["wdtype"]).requires_grad_(True)
        s["add"] = 1.0 if case["mod"] else 0.0
        s["dy"] = normal(b, t, d, dtype=case["dtype"])
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _plain_lora(s):
    down, up, scale, dt = s["down"].float(), s["up"].float(), s["scale"], s["x"].dtype
    a, r, k = down.shape
    n = up.shape[1]
    x = s["x"].float()
    row = torch.arange(x.shape[0], device=x.device)
    request = (row[:, None] >= s["offsets"][None, 1:]).sum(1)
    adapter = torch.cat([s["adapters"], s["adapters"].new_full((1,), -1)])[request]  # -1 behind the last request
    weight = (adapter[:, None] == torch.arange(a, device=x.device)[None]).float() * scale
    weight = weight[:, :, None].expand(-1, -1, r).reshape(-1, a * r)
    down, up = down.reshape(a * r, k), up.permute(0, 2, 1).reshape(a * r, n)
    h = (x @ down.t()) * weight
    out = (s["base"].float() + h @ up).to(dt)
    if "dy" not in s:
        return out
    dy = s["dy"].float()
    g = (dy @ up.t()) * weight
    d_up = (h.t() @ dy).reshape(a, r, n).permute(0, 2, 1)
    return {"out": out, "dx": (g @ down).to(dt), "ddown": (g.t() @ x).reshape(a, r, k).to(dt), "dup": d_up.to(dt)}


def _angles(ids, axes):
    parts = [ids[:, i, None].double() / 10000.0 ** (torch.arange(0, d, 2, device=ids.device, dtype=torch.float64) / d) for i, d in enumerate(axes)]
    return torch.cat(parts, 1)


def _rotate(x, cos, sin, half):
    r = 2 * cos.shape[1]
    xf = x.float()
    cos, sin = cos[:, None], sin[:, None]
    if half:
        a, b = xf[..., : r // 2], xf[..., r // 2 : r]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = xf[..., 0:r:2], xf[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([y, xf[..., r:]], -1).to(x.dtype)


def _plain_rotary(s):
    half = s["case"]["half"]
    a = _angles(s["ids"], s["axes"])
    cos, sin = torch.cos(a).float(), torch.sin(a).float()
    out = [_rotate(s["q"], cos, sin, half), _rotate(s["k"], cos, sin, half)]
    if "dq" in s:
        out += [_rotate(s["dq"], cos, -sin, half), _rotate(s["dk"], cos, -sin, half)]
    return out


def _plain_norm(s):
    x, dy, w, b = s["x"].float(), s["dy"].float(), s["w"].float(), s["b"].float()
    mod = w.dim() == 2
    scale = (w[:, None] if mod else w) + s["add"]
    shift = b[:, None] if mod else b
    d = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-6)
    xhat = d * rstd
    v = dy * scale
    dx = rstd * (v - v.mean(-1, keepdim=True) - xhat * (v * xhat).mean(-1, keepdim=True))
    over = 1 if mod else (0, 1)
    return {"y": (xhat * scale + shift).to(s["x"].dtype), "dx": dx.to(s["x"].dtype),
            "dw": (dy * xhat).sum(over).to(s["w"].dtype), "db": dy.sum(over).to(s["b"].dtype)}


def _run_plain(s):
    op = s["case"]["op"]
    with torch.no_grad():
        if op == "lora":
            return _plain_lora(s)
        if op == "rotary":
            return _plain_rotary(s)
        if op == "table":
            a = _angles(s["ids"], s["axes"])
            return torch.stack([torch.sin(a), torch.cos(a)], -1).float()[:, :, None]
        return _plain_norm(s)


# ------------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    op = s["case"]["op"]
    if op == "lora":
        from nunchaku_rocm_b200.ops.lora import lora_batched

        out = lora_batched(s["x"], s["down"], s["up"], s["offsets"], s["adapters"], base=s["base"], scale=s["scale"])
        if "dy" not in s:
            return out
        dx, ddown, dup = torch.autograd.grad(out, (s["x"], s["down"], s["up"]), s["dy"])
        return {"out": out, "dx": dx, "ddown": ddown, "dup": dup}
    if op == "rotary":
        from nunchaku_rocm_b200.ops.rotary import rotary_axes

        q, k = rotary_axes(s["q"], s["k"], s["ids"], s["axes"], interleaved=not s["case"]["half"])
        if "dq" not in s:
            return [q, k]
        return [q, k, *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]
    if op == "table":
        from nunchaku_rocm_b200.ops.rotary import rotary_table

        return rotary_table(s["ids"], s["axes"])
    from nunchaku_rocm_b200.ops.elementwise import layer_norm

    y = layer_norm(s["x"], s["w"], s["b"], weight_add=s["add"])
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "lora":
            lengths, adapters = _requests(case)
            x, down, up, out = s["x"].double(), s["down"].double(), s["up"].double(), s["base"].double()
            dy = s["dy"].double() if case["train"] else None
            dx, ddown, dup = torch.zeros_like(x), torch.zeros_like(down), torch.zeros_like(up)
            at = 0
            for n, a in zip(lengths, adapters):
                rows = slice(at, at + n)
                at += n
                if a < 0:
                    continue
                h = torch.einsum("tk,rk->tr", x[rows], down[a])
                out[rows] += s["scale"][a].double() * torch.einsum("tr,nr->tn", h, up[a])
                if case["train"]:
                    g = s["scale"][a].double() * torch.einsum("tn,nr->tr", dy[rows], up[a])
                    dx[rows] = torch.einsum("tr,rk->tk", g, down[a])
                    ddown[a] += torch.einsum("tr,tk->rk", g, x[rows])
                    dup[a] += s["scale"][a].double() * torch.einsum("tn,tr->nr", dy[rows], h)
            return {"out": out, "dx": dx, "ddown": ddown, "dup": dup} if case["train"] else out
        if op in ("rotary", "table"):
            turns = []
            for i, d in enumerate(s["axes"]):
                for j in range(d // 2):
                    turns.append(s["ids"][:, i].double() * 10000.0 ** (-2.0 * j / d))
            z = torch.polar(torch.ones_like(torch.stack(turns, 1)), torch.stack(turns, 1))
            if op == "table":
                return torch.stack([z.imag, z.real], -1)[:, :, None]

            def rotated(t, z):
                t, r = t.double(), 2 * z.shape[1]
                pairs = torch.complex(t[..., : r // 2], t[..., r // 2 : r]) if case["half"] else torch.complex(t[..., :r:2], t[..., 1:r:2])
                p = pairs * z[:, None]
                y = torch.cat([p.real, p.imag], -1) if case["half"] else torch.view_as_real(p).reshape(*p.shape[:-1], r)
                return torch.cat([y, t[..., r:]], -1)

            out = [rotated(s["q"], z), rotated(s["k"], z)]
            if case["train"]:
                out += [rotated(s["dq"], z.conj()), rotated(s["dk"], z.conj())]
            return out
    x, w, b = (s[v].detach().double().requires_grad_(True) for v in ("x", "w", "b"))
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    per_row = (lambda v: v.unsqueeze(1)) if case["mod"] else (lambda v: v)
    y = (x - mean) * torch.rsqrt(var + 1e-6) * (per_row(w) + s["add"]) + per_row(b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
