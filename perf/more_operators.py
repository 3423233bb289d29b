"""What a training step of a model with experts needs beside its norms, sorted rows and 8-bit products, as cases
that can be timed: products in 16-bit floats with one matrix or one per expert, with their gradients; the softmax
cross entropy of a vocabulary's logits from the rows before them, with its gradients; dropout with a mask that is
never stored, added to a residual.

`own` selects between the framework's operators and their plain forms in elementary torch operations.
Nothing here needs the framework while `own` is false.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one linear layer for a few generated tokens: the weights are read once, latency counts
        {"name": "products, 4 tokens", "op": "product", "rows": 4, "groups": 1, "n": 8192, "k": 4096, "dtype": "bf16",
         "drop": 0.0, "pad": 0, "grad": False},
        # the experts' product for a generated batch: a few rows for each expert
        {"name": "products, a generated batch", "op": "product", "rows": 256, "groups": 64, "n": 1024, "k": 2048,
         "dtype": "bf16", "drop": 0.0, "pad": 0, "grad": False},
        # the experts' product in a training step, forward and both gradients
        {"name": "products, a training batch", "op": "product", "rows": 16384, "groups": 16, "n": 4096, "k": 4096,
         "dtype": "bf16", "drop": 0.0, "pad": 0, "grad": True},
        # odd sizes that no wide load fits, some rows of the batch without an expert, forward and both gradients
        {"name": "products, odd sizes", "op": "product", "rows": 3001, "groups": 20, "n": 1003, "k": 1021,
         "dtype": "f16", "drop": 0.1, "pad": 0, "grad": True},
        # how likely a few given tokens are: the vocabulary's weights are read once
        {"name": "loss, 16 tokens", "op": "loss", "rows": 16, "vocab": 50257, "d": 2048, "dtype": "bf16",
         "ignored": 0.0, "grad": False},
        # a training step's loss over a large vocabulary with both gradients
        {"name": "loss, a training batch", "op": "loss", "rows": 8192, "vocab": 128000, "d": 4096, "dtype": "bf16",
         "ignored": 0.0, "grad": True},
        # a padded batch: a part of the rows has no target; a vocabulary of odd size
        {"name": "loss, a padded batch", "op": "loss", "rows": 3001, "vocab": 50257, "d": 1000, "dtype": "f16",
         "ignored": 0.2, "grad": True},
        # a few rows, where latency counts
        {"name": "dropout, 8 rows", "op": "dropout", "rows": 8, "d": 4096, "dtype": "bf16", "p": 0.1, "pad": 0,
         "residual": True, "grad": False},
        # the end of a layer in a training step, added to the residual, and its gradient
        {"name": "dropout, a training batch", "op": "dropout", "rows": 16384, "d": 8192, "dtype": "bf16", "p": 0.1,
         "pad": 0, "residual": True, "grad": True},
        # rows of an odd width inside a wider buffer
        {"name": "dropout, odd rows", "op": "dropout", "rows": 5003, "d": 1021, "dtype": "f16", "p": 0.35, "pad": 3,
         "residual": True, "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, odd):
    n = _log(rng, lo, hi)
    return n if rng.random() < odd else (n + 63) // 64 * 64


def draw(rng):
    op = rng.choice(["product", "product", "loss", "loss", "dropout"])
    if op == "dropout":
        d = _size(rng, 64, 20000, 0.5)
        return {"op": op, "rows": _log(rng, 1, min(40000, 100_000_000 // d)), "d": d,
                "dtype": rng.choice(["bf16", "f16", "f32"]), "p": round(rng.uniform(0.0, 0.9), 3),
                "pad": rng.choice([0, 0, 8, rng.randrange(1, 40)]), "residual": rng.random() < 0.6,
                "grad": rng.random() < 0.6}
    dtype, grad = rng.choice(["bf16", "f16"]), rng.random() < 0.6
    if op == "product":
        groups = rng.choice([1, _log(rng, 2, 128)])
        n, k = _size(rng, 64, 8192, 0.25), _size(rng, 64, 8192, 0.25)
        n = max(64, min(n, 250_000_000 // (groups * k)))
        rows = _log(rng, 1, min(20000, 200_000_000_000 // (n * k)))
        return {"op": op, "rows": rows, "groups": groups, "n": n, "k": k, "dtype": dtype, "grad": grad,
                "drop": rng.choice([0.0, 0.0, round(rng.uniform(0.0, 0.9), 3)]), "pad": rng.choice([0, 0, 8])}
    d, vocab = _size(rng, 64, 4096, 0.25), _size(rng, 1000, 128000, 0.5)
    rows = _log(rng, 1, min(8192, 3_000_000_000_000 // (vocab * d)))
    return {"op": op, "rows": rows, "vocab": vocab, "d": d, "dtype": dtype, "grad": grad,
            "ignored": rng.choice([0.0, 0.0, round(rng.uniform(0.0, 0.9), 3)])}


def _normal(shape, gen):
    return torch.randn(shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s, op, dev, t = dict(case), case["op"], "cuda", TYPES[case["dtype"]]
    if op == "product":
        m, n, k, e, pad = case["rows"], case["n"], case["k"], case["groups"], case["pad"]
        s["x"] = _normal((m, k + pad), gen).to(t)[:, :k]
        s["w"] = torch.empty(e, n, k, dtype=t, device=dev)
        for g in range(e):
            s["w"][g] = _normal((n, k), gen) / math.sqrt(k)
        s["y"] = torch.zeros(m, n, dtype=t, device=dev)
        there = m - int(m * case["drop"])  # rows that have an expert; the padding is behind them
        liked = torch.softmax(0.7 * _normal((e,), gen), 0)  # some experts are chosen more often than others
        counts = torch.bincount(torch.multinomial(liked, there, replacement=True, generator=gen), minlength=e)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["most"], s["there"] = int(counts.max()), there
        if case["grad"]:
            s["dy"] = _normal((m, n + pad), gen).to(t)[:, :n]
            s["dx"], s["dw"] = torch.zeros(m, k, dtype=t, device=dev), torch.zeros(e, n, k, dtype=t, device=dev)
    elif op == "loss":
        m, v, d = case["rows"], case["vocab"], case["d"]
        s["w"] = torch.empty(v, d, dtype=t, device=dev)
        for at in range(0, v, 16384):
            s["w"][at:at + 16384] = _normal((min(16384, v - at), d), gen) * (1.5 / math.sqrt(d))
        # frequent tokens come often, and the model knows some of the targets better than others
        target = (v * torch.rand(m, generator=gen, device=dev) ** 3).long().clamp_(max=v - 1)
        known = 6 * torch.rand(m, 1, generator=gen, device=dev)
        s["h"] = (_normal((m, d), gen) + known * s["w"][target].float() / 1.5).to(t)
        target[m - int(m * case["ignored"]):] = -1
        s["targets"] = target.to(torch.int32)
        s["loss"], s["lse"] = (torch.zeros(m, device=dev) for _ in range(2))
        if case["grad"]:
            # the mean over the rows with a target; in f16 with the factor that a training loop scales its loss by
            scale = (1024.0 if t == torch.float16 else 1.0) / max(1, int((target >= 0).sum()))
            s["dloss"] = torch.full((m,), scale, device=dev)
            s["dh"], s["dw"] = torch.zeros(m, d, dtype=t, device=dev), torch.zeros(v, d, dtype=t, device=dev)
    else:
        rows, d, pad = case["rows"], case["d"], case["pad"]
        s["x"] = _normal((rows, d + pad), gen).to(t)[:, :d]
        s["residual_in"] = _normal((rows, d + pad), gen).to(t)[:, :d] if case["residual"] else None
        s["rng"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), generator=gen, device=dev)  # key and place in its stream
        s["y"] = torch.zeros(rows, d, dtype=t, device=dev)
        if case["grad"]:
            s["dy"] = _normal((rows, d + pad), gen).to(t)[:, :d]
            s["dx"] = torch.zeros(rows, d, dtype=t, device=dev)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------


def _product(s):
    t, off, m = s["x"].dtype, s["offsets"].long(), s["there"]
    row = torch.arange(m, device=off.device)
    g = torch.searchsorted(off, row, right=True) - 1
    at = row - off[g]
    x = torch.zeros(s["groups"], s["most"], s["k"], device=off.device)
    x[g, at] = s["x"][:m].float()
    w = s["w"].float()
    y = torch.zeros(s["rows"], s["n"], device=off.device)
    y[:m] = torch.bmm(x, w.transpose(1, 2))[g, at]
    out = {"y": y.to(t)}
    if s["grad"]:
        dy = torch.zeros(s["groups"], s["most"], s["n"], device=off.device)
        dy[g, at] = s["dy"][:m].float()
        dx = torch.zeros(s["rows"], s["k"], device=off.device)
        dx[:m] = torch.bmm(dy, w)[g, at]
        out.update(dx=dx.to(t), dw=torch.bmm(dy.transpose(1, 2), x).to(t))
    return out


def _loss(s):
    t, h, w, target = s["h"].dtype, s["h"].float(), s["w"].float(), s["targets"].long()
    there = target >= 0
    at = target.clamp(min=0)[:, None]
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    lse = top + torch.log(e.sum(1, keepdim=True))
    # the others' sum by itself: where the target is nearly certain, lse - logit would be what rounding leaves
    mine = e.gather(1, at)
    others = e.scatter_(1, at, 0.0).sum(1, keepdim=True)
    loss = (top - logits.gather(1, at)) + torch.log1p(others + (mine - 1))
    out = {"loss": torch.where(there, loss[:, 0], torch.zeros_like(loss[:, 0])), "lse": lse[:, 0]}
    if s["grad"]:
        g = torch.where(there, s["dloss"], torch.zeros_like(s["dloss"]))[:, None]
        p = torch.exp(logits - lse) * g
        p.scatter_add_(1, at, -g)
        out.update(dh=(p @ w).to(t), dw=(p.t() @ h).to(t))
    return out


def _philox(key, place, rows, blocks):
    """Philox 4x32-10 at the counters (block, row, low word of place, high word of place): eight 16-bit numbers
    each. Products of 32-bit words wrap in 64 bits, of which every bit is right."""
    low = 0xFFFFFFFF
    k0, k1 = key & low, (key >> 32) & low
    shape = (rows, blocks)
    dev = key.device
    c0 = torch.arange(blocks, device=dev)[None, :].expand(shape)
    c1 = torch.arange(rows, device=dev)[:, None].expand(shape)
    c2, c3 = (place & low).expand(shape), ((place >> 32) & low).expand(shape)

    def a_round(c0, c1, c2, c3, k0, k1):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        return ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low

    for i in range(10):
        c0, c1, c2, c3 = a_round(c0, c1, c2, c3, (k0 + i * 0x9E3779B9) & low, (k1 + i * 0xBB67AE85) & low)
    words = torch.stack([c0, c1, c2, c3], 2)
    return torch.stack([words & 0xFFFF, words >> 16], 3).reshape(rows, blocks * 8)


def _dropout(s):
    t, d = s["x"].dtype, s["d"]
    limit = int(round(s["p"] * 65536))
    kept = _philox(s["rng"][0], s["rng"][1], s["rows"], (d + 7) // 8)[:, :d] >= limit
    scale = 65536.0 / (65536 - limit)
    zero = torch.zeros((), device=kept.device)
    y = torch.where(kept, s["x"].float() * scale, zero)
    if s["residual"]:
        y = y + s["residual_in"].float()
    out = {"y": y.to(t)}
    if s["grad"]:
        out["dx"] = torch.where(kept, s["dy"].float() * scale, zero).to(t)
    return out


# ---- the framework's operators ------------------------------------------------------------------------------

_kept = {}


def _plan(s):
    """The context of the program, the records of this state's sizes and the loss's scratch, made once."""
    import flow_b200 as fb
    if "ctx" not in _kept:
        _kept["ctx"] = fb.Context((0,), sync=False)
    ctx, op = _kept["ctx"], s["op"]
    if op == "product":
        site = fb.product_site(s["rows"], s["n"], s["k"], s["x"].dtype, groups=s["groups"], ldx=s["x"].stride(0),
                               lddy=s["dy"].stride(0) if s["grad"] else 0)
    elif op == "loss":
        site = fb.loss_site(s["rows"], s["vocab"], s["d"], s["h"].dtype)
        s["work"] = torch.empty(ctx.linear_loss_workspace(site, grad=s["grad"]), dtype=torch.uint8, device="cuda")
    else:
        res = s["residual_in"]
        fwd = fb.dropout_site(s["rows"], s["d"], s["x"].dtype, s["p"], ldx=s["x"].stride(0),
                              ldr=res.stride(0) if res is not None else 0)
        bwd = fb.dropout_site(s["rows"], s["d"], s["x"].dtype, s["p"], ldx=s["dy"].stride(0)) if s["grad"] else None
        site = fwd, bwd
    s["plan"] = ctx, site
    return s["plan"]


def _run_own(s):
    ctx, site = s.get("plan") or _plan(s)
    op = s["op"]
    if op == "product":
        ctx.product(site, s["x"], s["w"], s["y"], offsets=s["offsets"])
        out = {"y": s["y"]}
        if s["grad"]:
            ctx.product_grad(site, s["x"], s["w"], s["dy"], s["dx"], s["dw"], offsets=s["offsets"])
            out.update(dx=s["dx"], dw=s["dw"])
        return out
    if op == "loss":
        ctx.linear_loss(site, s["h"], s["w"], s["targets"], s["loss"], s["lse"], s["work"])
        out = {"loss": s["loss"], "lse": s["lse"]}
        if s["grad"]:
            ctx.linear_loss_grad(site, s["h"], s["w"], s["targets"], s["lse"], s["dloss"], s["dh"], s["dw"], s["work"])
            out.update(dh=s["dh"], dw=s["dw"])
        return out
    fwd, bwd = site
    ctx.dropout(fwd, s["x"], s["residual_in"], s["y"], s["rng"])
    out = {"y": s["y"]}
    if s["grad"]:
        ctx.dropout(bwd, s["dy"], None, s["dx"], s["rng"])  # the gradient is the same call on dy
        out["dx"] = s["dx"]
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"product": _product, "loss": _loss, "dropout": _dropout}[state["op"]](state)


def work(case):
    op, es = case["op"], SIZE[case["dtype"]]
    if op == "product":
        m, n, k = case["rows"] - int(case["rows"] * case["drop"]), case["n"], case["k"]
        weights = min(case["groups"], m) * n * k
        b, f = (m * k + weights + m * n) * es + 4 * (case["groups"] + 1), 2 * m * n * k
        if case["grad"]:
            b += (m * n + m * k + case["groups"] * n * k) * es
            f *= 3
        return {"bytes": b, "flops": f}
    if op == "loss":
        m, v, d = case["rows"], case["vocab"], case["d"]
        b, f = (m * d + v * d) * es + 12 * m, 2 * m * v * d + 4 * m * v
        if case["grad"]:
            b += (m * d + v * d) * es + 4 * m
            f = 3 * f
        return {"bytes": b, "flops": f}
    n = case["rows"] * case["d"]
    arrays = 2 + (1 if case["residual"] else 0) + (2 if case["grad"] else 0)
    return {"bytes": n * arrays * es + 16, "flops": n * (6 if case["grad"] else 3)}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------


def _exact_product(s):
    ends, dev = s["offsets"].tolist(), s["x"].device
    y = torch.zeros(s["rows"], s["n"], dtype=torch.float64, device=dev)
    out = {"y": y}
    if s["grad"]:
        out["dx"] = torch.zeros(s["rows"], s["k"], dtype=torch.float64, device=dev)
        out["dw"] = torch.zeros(s["groups"], s["n"], s["k"], dtype=torch.float64, device=dev)
    for g in range(s["groups"]):
        rows = slice(ends[g], ends[g + 1])
        x, w = s["x"][rows].double(), s["w"][g].double()
        y[rows] = torch.einsum("ik,nk->in", x, w)
        if s["grad"]:
            dy = s["dy"][rows].double()
            out["dx"][rows] = torch.einsum("in,nk->ik", dy, w)
            out["dw"][g] = torch.einsum("in,ik->nk", dy, x)
    return out


def _exact_loss(s):
    m, v, d = s["rows"], s["vocab"], s["d"]
    w, dev = s["w"].double(), s["h"].device
    loss, lse = (torch.zeros(m, dtype=torch.float64, device=dev) for _ in range(2))
    out = {"loss": loss, "lse": lse}
    if s["grad"]:
        out["dh"], out["dw"] = (torch.zeros(n, d, dtype=torch.float64, device=dev) for n in (m, v))
    for lo in range(0, m, 1024):
        rows = slice(lo, min(m, lo + 1024))
        h, target = s["h"][rows].double(), s["targets"][rows].long()
        logits = torch.einsum("id,vd->iv", h, w)
        lse[rows] = torch.logsumexp(logits, 1)
        there = torch.nonzero(target >= 0)[:, 0]
        loss[rows] = loss[rows].index_copy(0, there, lse[rows][there] - logits[there, target[there]])
        if s["grad"]:
            g = torch.zeros_like(logits)
            g[there] = torch.softmax(logits[there], 1)
            g[there, target[there]] -= 1
            g *= s["dloss"][rows].double()[:, None]
            out["dh"][rows] = torch.einsum("iv,vd->id", g, w)
            out["dw"] += torch.einsum("iv,id->vd", g, h)
    return out


def _mask(key, place, rows, d, limit):
    """Which elements Philox 4x32-10 keeps, with products of 16-bit halves."""
    key, place = key % 2 ** 64, place % 2 ** 64
    low = 0xFFFFFFFF

    def wide(a, b):  # 32-bit a (tensor) times 32-bit b: high and low word
        ah, al, bh, bl = a >> 16, a & 0xFFFF, b >> 16, b & 0xFFFF
        mid = ah * bl + (al * bl >> 16)
        lowmid = (mid & 0xFFFF) + al * bh
        return ah * bh + (mid >> 16) + (lowmid >> 16), ((lowmid & 0xFFFF) << 16) | (al * bl & 0xFFFF)

    col = torch.arange(d, device="cuda")
    out = torch.empty(rows, d, dtype=torch.bool, device="cuda")
    for lo in range(0, rows, 1024):
        r = torch.arange(lo, min(rows, lo + 1024), device="cuda")[:, None]
        x = [torch.arange((d + 7) // 8, device="cuda")[None, :] + 0 * r, r + 0 * torch.arange((d + 7) // 8, device="cuda")]
        x += [torch.full_like(x[0], place & low), torch.full_like(x[0], place >> 32)]
        k = [key & low, key >> 32]
        for _ in range(10):
            (h0, l0), (h1, l1) = wide(x[0], 0xD2511F53), wide(x[2], 0xCD9E8D57)
            x = [h1 ^ x[1] ^ k[0], l1, h0 ^ x[3] ^ k[1], l0]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        word = torch.stack(x)[col % 8 // 2, :, col // 8].t()
        out[lo:lo + 1024] = (word >> 16 * (col % 2)) % 65536 >= limit
    return out


def _exact_dropout(s):
    limit = int(round(s["p"] * 65536))
    kept = _mask(int(s["rng"][0]), int(s["rng"][1]), s["rows"], s["d"], limit)
    factor = kept.double().mul_(65536 / (65536 - limit))
    out = {"y": s["x"].double() * factor}
    if s["residual"]:
        out["y"] += s["residual_in"].double()
    if s["grad"]:
        out["dx"] = s["dy"].double() * factor
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"product": _exact_product, "loss": _exact_loss, "dropout": _exact_dropout}[s["op"]](s)
