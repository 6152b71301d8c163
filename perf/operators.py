"""What is measured of the training-step operators: the combine with dropout in
its epilogue, the expert balance loss and the clipped policy loss, each with its
gradient. `run` computes a case in plain torch, or with the framework's kernels
where `own` is true; `exact` computes it in 64 bits, written apart."""
import math

import torch

own = False

_TORCH = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
_ctx = None


def _context():
    """One device context for the process, on a torch stream, as a training program keeps it."""
    global _ctx
    if _ctx is None:
        import xucg_amd
        _ctx = xucg_amd.DevContext.on_torch_stream(torch.cuda.current_device())
    return _ctx


# ---- the cases -------------------------------------------------------------------------------

def _drop(name, dt, rows, cols, nsrc=1, p=0.1, offset=0, bias=True, residual=True, out_dt=None):
    return dict(name=name, op="dropout", dt=dt, out_dt=out_dt or dt, rows=rows, cols=cols, nsrc=nsrc, p=p,
                offset=offset, bias=bias, residual=residual)


def _drop_grad(name, dt, rows, cols, p=0.1, offset=0, bias=True, out_dt=None):
    return dict(name=name, op="dropout_grad", dt=dt, out_dt=out_dt or dt, rows=rows, cols=cols, p=p, offset=offset,
                bias=bias)


def _balance(name, dt, tokens, experts, topk, grad, padded=True, base=False):
    return dict(name=name, op="balance_grad" if grad else "balance", dt=dt, tokens=tokens, experts=experts,
                topk=topk, padded=padded, **({"base": base} if grad else {}))


def _policy(name, dt, rows, cols, grad, per_sequence=False, kl=True, adv_per_row=True):
    return dict(name=name, op="policy_grad" if grad else "policy", dt=dt, rows=rows, cols=cols,
                per_sequence=per_sequence, kl=kl, adv_per_row=adv_per_row)


def listed():
    return [
        # a few tokens of a small layer: what a call costs
        _drop("drop-f32-4x1024", "float32", 4, 1024),
        # the sum of four tensor-parallel members' partial products, one layer's tokens
        _drop("drop-bf16-4src-4096x4096", "bfloat16", 4096, 4096, nsrc=4),
        # a shard that begins in the middle of a row, widths that are no multiple of a vector
        _drop("drop-f16-2src-odd", "float16", 1237, 1023, nsrc=2, p=0.25, offset=1237 * 1023 * 3 + 5),
        # the largest: one long batch, residual stream in 32 bits
        _drop("drop-bf16-f32res-16384x8192", "bfloat16", 16384, 8192, out_dt="float32"),
        # the backward pass with the bias' gradient: ordinary, and ragged in 32 bits
        _drop_grad("dropgrad-bf16-8192x4096", "bfloat16", 8192, 4096),
        _drop_grad("dropgrad-f32-odd", "float32", 777, 2049, p=0.2, offset=12345),
        # one small batch of a router with few experts
        _balance("balance-f32-64x8", "float32", 64, 8, 2, False),
        # many experts and a long padded batch; its gradient joined to the gates'
        _balance("balance-bf16-65536x256", "bfloat16", 65536, 256, 8, False),
        _balance("balancegrad-bf16-49999x160", "bfloat16", 49999, 160, 6, True, base=True),
        # a handful of short answers
        _policy("policy-f32-8x200", "float32", 8, 200, False),
        # many answers with long reasoning, the mean over all tokens
        _policy("policy-f32-1024x8192", "float32", 1024, 8192, False),
        # the gradient, each answer weighing the same, an odd length
        _policy("policygrad-bf16-513x12345", "bfloat16", 513, 12345, True, per_sequence=True, adv_per_row=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dropout", "dropout", "dropout_grad", "balance", "balance_grad", "policy", "policy_grad"])
    dt = rng.choice(["bfloat16", "float16", "float32"])
    if op in ("dropout", "dropout_grad"):
        cols = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        nsrc = rng.choice([1, 1, 2, 3, 4, 8])
        rows = _log(rng, 1, max(1, min(16384, (1 << 25) // cols)))
        out_dt = rng.choice([dt, "float32"])
        offset = rng.choice([0, 0, rows * cols * rng.randint(1, 7), rng.randint(1, 1 << 40)])
        p = rng.choice([0.05, 0.1, 0.2, 0.5, 0.0])
        if op == "dropout":
            c = _drop("", dt, rows, cols, nsrc, p, offset, rng.random() < 0.7, rng.random() < 0.8, out_dt)
        else:
            c = _drop_grad("", dt, rows, cols, p, offset, rng.random() < 0.7, out_dt)
    elif op in ("balance", "balance_grad"):
        experts = rng.choice([8, 16, 32, 60, 64, 128, 160, 256, 384, rng.randint(2, 512)])
        topk = rng.randint(1, min(8, experts))
        c = _balance("", dt, _log(rng, 1, 65536), experts, topk, op == "balance_grad", rng.random() < 0.6,
                     rng.random() < 0.5)
    else:
        cols = _log(rng, 1, 16384)
        c = _policy("", dt, _log(rng, 1, max(1, min(2048, (1 << 23) // cols))), cols, op == "policy_grad",
                    rng.random() < 0.5, rng.random() < 0.7, rng.random() < 0.5)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------

BALANCE_COEF, Z_COEF = 0.01, 0.001
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.05


def _normal(gen, shape, dt, std=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * std).to(_TORCH[dt])


def _prefix_mask(gen, rows, cols):
    """Answers of different lengths in one batch, one of them empty where there are several."""
    n = torch.randint(1, cols + 1, (rows, 1), device="cuda", generator=gen)
    if rows > 3:
        n[rows // 2] = 0
    return (torch.arange(cols, device="cuda") < n).to(torch.uint8)


def prepare(case, seed):
    c = dict(case)
    ctx = _context() if own else None
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case=c, ctx=ctx)
    op, dt = c["op"], c["dt"]
    if op in ("dropout", "dropout_grad"):
        shape = (c["rows"], c["cols"])
        s["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) & ((1 << 63) - 1)
        s["tag"] = 3 * seed + 1
        s["bias"] = _normal(gen, shape[1:], dt, 0.5) if c["bias"] else None
        if op == "dropout":
            s["srcs"] = [_normal(gen, shape, dt) for _ in range(c["nsrc"])]
            s["residual"] = _normal(gen, shape, c["out_dt"]) if c["residual"] else None
            s["out"] = torch.empty(shape, dtype=_TORCH[c["out_dt"]], device="cuda")
        else:
            s["grad"] = _normal(gen, shape, c["out_dt"])
            s["dsrc"] = torch.empty(shape, dtype=_TORCH[dt], device="cuda")
            s["dbias"] = torch.empty(shape[1], device="cuda") if c["bias"] else None
            if own:
                s["ws"] = torch.empty(ctx.sum_dropout_grad_workspace(*shape), dtype=torch.uint8, device="cuda")
    elif op in ("balance", "balance_grad"):
        t, e, k = c["tokens"], c["experts"], c["topk"]
        # some experts are liked better than others
        s["logits"] = ((torch.randn((t, e), device="cuda", generator=gen) * 1.5
                        + torch.randn((1, e), device="cuda", generator=gen) * 0.5)).to(_TORCH[dt])
        s["index"] = torch.topk(s["logits"].float(), k, dim=1).indices
        s["mask"] = None
        if c["padded"]:
            s["mask"] = (torch.rand(t, device="cuda", generator=gen) < 0.85).to(torch.uint8)
            s["mask"][0] = 1
        s["counts"] = torch.empty(e + 1, dtype=torch.int64, device="cuda")
        s["sums"] = torch.empty(e + 1, device="cuda")
        s["loss"] = torch.empty(3, device="cuda")
        if op == "balance_grad":
            live = torch.ones(t, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"] != 0
            # the counts of a group of two members: this one's tokens, and as many of another
            s["counts"] = torch.zeros(e + 1, dtype=torch.int64, device="cuda")
            s["counts"][:e] = torch.bincount(s["index"][live].reshape(-1), minlength=e) * 2
            s["counts"][e] = live.sum() * 2
            s["base"] = _normal(gen, (t, e), dt, 1e-6) if c["base"] else None
            s["grad_loss"] = torch.rand(1, device="cuda", generator=gen) + 0.5
            s["dlogits"] = torch.empty_like(s["logits"])
        if own:
            s["ws"] = torch.empty(ctx.balance_workspace(t, e), dtype=torch.uint8, device="cuda")
    else:
        shape = (c["rows"], c["cols"])
        old = -torch.rand(shape, device="cuda", generator=gen).log().abs() - 0.01
        s["logp"] = (old + torch.randn(shape, device="cuda", generator=gen) * 0.15).to(_TORCH[dt])
        s["old"] = old.to(_TORCH[dt])
        s["ref"] = (old + torch.randn(shape, device="cuda", generator=gen) * 0.2).to(_TORCH[dt]) if c["kl"] else None
        s["adv"] = torch.randn(shape[:1] if c["adv_per_row"] else shape, device="cuda", generator=gen)
        s["mask"] = _prefix_mask(gen, *shape)
        s["row_tokens"] = s["mask"].sum(1).to(torch.int32)
        s["sums"] = torch.empty(2, device="cuda")
        s["counts"] = torch.empty(3, dtype=torch.int64, device="cuda")
        s["loss"] = torch.empty(3, device="cuda")
        if op == "policy_grad":
            s["counts"] = torch.stack([s["row_tokens"].sum(), (s["row_tokens"] > 0).sum(),
                                       torch.zeros((), dtype=torch.int64, device="cuda")]) * 2
            s["grad_loss"] = torch.rand(1, device="cuda", generator=gen) + 0.5
            s["dlogp"] = torch.empty_like(s["logp"])
        if own:
            s["ws"] = torch.empty(ctx.policy_workspace(*shape), dtype=torch.uint8, device="cuda")
    return s


# ---- one pass --------------------------------------------------------------------------------

def _run_own(s):
    c, ctx = s["case"], s["ctx"]
    op, dt = c["op"], c["dt"]
    if op == "dropout":
        ctx.sum_dropout(dt, s["out"], s["srcs"], c["rows"], c["cols"], c["p"], s["seed"], tag=s["tag"],
                        offset=c["offset"], bias=s["bias"], residual=s["residual"], out_dt=c["out_dt"])
        return {"out": s["out"]}
    if op == "dropout_grad":
        ctx.sum_dropout_grad(dt, s["dsrc"], s["grad"], c["rows"], c["cols"], c["p"], s["seed"], tag=s["tag"],
                             offset=c["offset"], dbias=s["dbias"], grad_dt=c["out_dt"], workspace=s["ws"])
        return {"dsrc": s["dsrc"], "dbias": s["dbias"]}
    if op == "balance":
        ctx.balance(dt, s["logits"], s["index"], c["tokens"], c["experts"], c["topk"], s["counts"], s["sums"],
                    mask=s["mask"], loss=s["loss"], balance_coef=BALANCE_COEF, z_coef=Z_COEF, workspace=s["ws"])
        return {"counts": s["counts"], "sums": s["sums"], "loss": s["loss"]}
    if op == "balance_grad":
        ctx.balance_grad(dt, s["dlogits"], s["logits"], c["tokens"], c["experts"], c["topk"], s["counts"],
                         mask=s["mask"], base=s["base"], grad_loss=s["grad_loss"], balance_coef=BALANCE_COEF,
                         z_coef=Z_COEF)
        return {"dlogits": s["dlogits"]}
    if op == "policy":
        ctx.policy(dt, s["logp"], s["old"], s["adv"], c["rows"], c["cols"], s["sums"], s["counts"], ref=s["ref"],
                   mask=s["mask"], row_tokens=s["row_tokens"], adv_per_row=c["adv_per_row"],
                   per_sequence=c["per_sequence"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF,
                   loss=s["loss"], workspace=s["ws"])
        return {"sums": s["sums"], "counts": s["counts"], "row_tokens": s["row_tokens"], "loss": s["loss"]}
    ctx.policy_grad(dt, s["dlogp"], s["logp"], s["old"], s["adv"], c["rows"], c["cols"], s["counts"], ref=s["ref"],
                    mask=s["mask"], row_tokens=s["row_tokens"], adv_per_row=c["adv_per_row"],
                    per_sequence=c["per_sequence"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF,
                    grad_loss=s["grad_loss"])
    return {"dlogp": s["dlogp"]}


_M32 = 0xFFFFFFFF


def _keep(seed, tag, offset, n, threshold):
    """Philox-4x32 with ten rounds: eight 16-bit numbers for eight neighbouring elements."""
    first = offset // 8
    c0 = torch.arange(first, (offset + n + 7) // 8, device="cuda")
    c0, c1 = c0 & _M32, c0 >> 32
    c2, c3 = torch.full_like(c0, tag & _M32), torch.full_like(c0, tag >> 32)
    k0, k1 = seed & _M32, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _M32) ^ c1 ^ k0, b & _M32, ((a >> 32) & _M32) ^ c3 ^ k1, a & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    words = torch.stack((c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16), 1)
    return words.reshape(-1)[offset - first * 8:][:n] >= threshold


def _plain_dropout(s):
    c = s["case"]
    n, threshold = c["rows"] * c["cols"], round(c["p"] * 65536)
    keep = _keep(s["seed"], s["tag"], c["offset"], n, threshold).reshape(c["rows"], c["cols"])
    scale = 65536 / (65536 - threshold)
    if c["op"] == "dropout_grad":
        d = torch.where(keep, s["grad"].float() * scale, 0.0)
        dbias = d.sum(0, dtype=torch.float64).float() if c["bias"] else None
        return {"dsrc": d.to(_TORCH[c["dt"]]), "dbias": dbias}
    x = s["srcs"][0].float()
    for src in s["srcs"][1:]:
        x = x + src.float()
    if s["bias"] is not None:
        x = x + s["bias"].float()
    x = torch.where(keep, x * scale, 0.0)
    if s["residual"] is not None:
        x = x + s["residual"].float()
    return {"out": x.to(_TORCH[c["out_dt"]])}


def _softmax(logits):
    x = logits.float()
    top = x.max(1, keepdim=True).values
    w = torch.exp(x - top)
    total = w.sum(1, keepdim=True)
    return w / total, (top + torch.log(total))[:, 0]


def _balance_loss(counts, sums, experts, topk):
    n = counts[experts].double()
    balance = (counts[:experts].double() * sums[:experts].double()).sum() * (BALANCE_COEF * experts / topk) / (n * n)
    z = sums[experts].double() * Z_COEF / n
    return torch.stack((balance + z, balance, z)).float()


def _plain_balance(s):
    c = s["case"]
    e = c["experts"]
    p, lse = _softmax(s["logits"])
    live = torch.ones_like(lse) if s["mask"] is None else (s["mask"] != 0).float()
    if c["op"] == "balance":
        counts = torch.zeros(e + 1, dtype=torch.int64, device="cuda")
        ones = live.to(torch.int64)
        counts.scatter_add_(0, s["index"].reshape(-1), ones[:, None].expand(-1, c["topk"]).reshape(-1))
        counts[e] = ones.sum()
        sums = torch.cat(((p * live[:, None]).sum(0, dtype=torch.float64),
                          (lse * lse * live).sum(0, keepdim=True, dtype=torch.float64)))
        return {"counts": counts, "sums": sums.float(), "loss": _balance_loss(counts, sums, e, c["topk"])}
    n = s["counts"][e].float()
    share = (s["counts"][:e].double() * e / s["counts"][:e].sum() - 1).float()  # near nought where experts are used alike
    share = share * (s["counts"][:e].sum().double() / e).float()
    d = p * (share - (p * share).sum(1, keepdim=True)) * (BALANCE_COEF * e / c["topk"] / (n * n))
    d = d + p * lse[:, None] * (2 * Z_COEF / n)
    d = torch.where(live[:, None] > 0, d * s["grad_loss"], 0.0)
    if s["base"] is not None:
        d = d + s["base"].float()
    return {"dlogits": d.to(s["logits"].dtype)}


def _expm1_less(q):
    """exp(q) - q - 1, which loses everything near nought in 32 bits."""
    q = q.double()
    return (torch.expm1(q) - q).float()


def _plain_policy(s):
    c = s["case"]
    logp, live = s["logp"].float(), s["mask"] != 0
    adv = s["adv"][:, None] if c["adv_per_row"] else s["adv"]
    d = logp - s["old"].float()
    up = (adv > 0) & (d > math.log1p(CLIP_HIGH))
    down = (adv < 0) & (d < math.log1p(-CLIP_LOW))
    ratio = torch.exp(d)
    if c["op"] == "policy":
        ratio = torch.where(up, 1 + CLIP_HIGH, torch.where(down, 1 - CLIP_LOW, ratio))
        pg = torch.where(live, -adv * ratio, 0.0)
        kl = torch.where(live, _expm1_less(s["ref"].float() - logp), 0.0) if c["kl"] else torch.zeros_like(pg)
        rows = live.sum(1)
        weight = 1.0 / rows.clamp(min=1).double() if c["per_sequence"] else torch.ones_like(rows).double()
        sums = torch.stack(((pg.sum(1, dtype=torch.float64) * weight).sum(),
                            (kl.sum(1, dtype=torch.float64) * weight).sum()))
        counts = torch.stack((rows.sum(), (rows > 0).sum(), (live & (up | down)).sum()))
        mean = sums / (counts[1] if c["per_sequence"] else counts[0])
        loss = torch.stack((mean[0] + KL_COEF * mean[1], mean[0], mean[1]))
        return {"sums": sums.float(), "counts": counts, "row_tokens": rows.to(torch.int32), "loss": loss.float()}
    g = torch.where(up | down, 0.0, -adv * ratio)
    if c["kl"]:
        g = g - KL_COEF * torch.expm1(s["ref"].float() - logp)
    weight = s["grad_loss"] / s["counts"][0]
    if c["per_sequence"]:
        weight = s["grad_loss"] / (s["row_tokens"].clamp(min=1) * s["counts"][1])[:, None]
    return {"dlogp": torch.where(live, g * weight, 0.0).to(s["logp"].dtype)}


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op.startswith("dropout"):
        return _plain_dropout(state)
    return _plain_balance(state) if op.startswith("balance") else _plain_policy(state)


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    c = case
    s = _SIZE[c["dt"]]
    if c["op"] == "dropout":
        n, o = c["rows"] * c["cols"], _SIZE[c["out_dt"]]
        return {"bytes": n * (c["nsrc"] * s + o * (2 if c["residual"] else 1)) + (c["cols"] * s if c["bias"] else 0),
                "flops": n * (c["nsrc"] + 3)}
    if c["op"] == "dropout_grad":
        n, o = c["rows"] * c["cols"], _SIZE[c["out_dt"]]
        return {"bytes": n * (s + o) + (c["cols"] * 4 if c["bias"] else 0), "flops": n * 2}
    if c["op"].startswith("balance"):
        t, e, k = c["tokens"], c["experts"], c["topk"]
        mask = t if c["padded"] else 0
        if c["op"] == "balance":
            return {"bytes": t * e * s + t * k * 8 + mask + (e + 1) * 12 + 12, "flops": 5 * t * e}
        return {"bytes": t * e * s * (3 if c["base"] else 2) + mask + (e + 1) * 8, "flops": 9 * t * e}
    n = c["rows"] * c["cols"]
    read = n * (s * (3 if c["kl"] else 2) + 1) + (c["rows"] if c["adv_per_row"] else n) * 4 + c["rows"] * 4
    return {"bytes": read + 44, "flops": 16 * n} if c["op"] == "policy" else {"bytes": read + n * s, "flops": 12 * n}


# ---- in 64 bits ------------------------------------------------------------------------------

def _mul32(a, b):
    """High and low word of the product of 32-bit numbers, by halves of the second."""
    low, high = a * (b & 0xFFFF), a * (b >> 16)
    mid = high + (low >> 16)
    return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _exact_keep(seed, tag, offset, n, threshold):
    place = offset + torch.arange(n, device="cuda")
    group = torch.arange(offset // 8, (offset + n - 1) // 8 + 1, device="cuda")
    x = [group % 2 ** 32, group // 2 ** 32, torch.zeros_like(group) + tag % 2 ** 32, torch.zeros_like(group) + tag // 2 ** 32]
    for r in range(10):
        key = ((seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32)
        h0, l0 = _mul32(x[0], 0xD2511F53)
        h1, l1 = _mul32(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ key[0], l1, h0 ^ x[3] ^ key[1], l0]
    table = torch.stack(x)
    lane = place % 8
    word = table[lane // 2, place // 8 - offset // 8]
    return (word >> (16 * (lane % 2))) % 65536 >= threshold


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] in ("dropout", "dropout_grad"):
        threshold = round(c["p"] * 65536)
        keep = _exact_keep(s["seed"], s["tag"], c["offset"], c["rows"] * c["cols"], threshold).view(c["rows"], c["cols"])
        factor = keep.double() * (65536 / (65536 - threshold))
        if c["op"] == "dropout_grad":
            d = factor * s["grad"].double()
            return {"dsrc": d, "dbias": d.sum(0) if c["bias"] else None}
        total = sum(x.double() for x in s["srcs"]) + (s["bias"].double() if c["bias"] else 0)
        return {"out": factor * total + (s["residual"].double() if c["residual"] else 0)}
    if c["op"] in ("balance", "balance_grad"):
        e, k = c["experts"], c["topk"]
        x = s["logits"].double()
        lse = torch.logsumexp(x, 1)
        p = torch.exp(x - lse[:, None])
        live = torch.ones_like(lse) if s["mask"] is None else s["mask"].double()
        if c["op"] == "balance":
            used = torch.bincount(s["index"][live > 0].reshape(-1), minlength=e).double()
            n, prob, zsum = live.sum(), live @ p, live @ lse.square()
            balance, z = BALANCE_COEF * e * torch.dot(used / (k * n), prob / n), Z_COEF * zsum / n
            return {"counts": None, "sums": torch.cat((prob, zsum[None])), "loss": torch.stack((balance + z, balance, z))}
        n, used = s["counts"][e].double(), s["counts"][:e].double()
        slope = BALANCE_COEF * e * (used / (k * n)) / n
        d = p * (slope - (p @ slope)[:, None]) + 2 * Z_COEF / n * lse[:, None] * p
        d = d * live[:, None] * s["grad_loss"].double()
        return {"dlogits": d + (s["base"].double() if c["base"] else 0)}
    live = s["mask"].double()
    adv = (s["adv"][:, None] if c["adv_per_row"] else s["adv"]).double()
    # whether a token is clipped goes by the difference in 32 bits: that is the operator's definition
    side = s["logp"].float() - s["old"].float()
    cut = torch.where(adv > 0, side > math.log1p(CLIP_HIGH), (adv < 0) & (side < math.log1p(-CLIP_LOW)))
    ratio = (s["logp"].double() - s["old"].double()).exp()
    q = s["ref"].double() - s["logp"].double() if c["kl"] else None
    rows = live.sum(1)
    each = live / rows.clamp(min=1)[:, None] if c["per_sequence"] else live
    if c["op"] == "policy":
        pg = -adv * torch.where(cut, torch.where(adv > 0, 1 + CLIP_HIGH, 1 - CLIP_LOW).double(), ratio)
        kl = torch.expm1(q) - q if c["kl"] else torch.zeros_like(pg)
        sums = torch.stack(((each * pg).sum(), (each * kl).sum()))
        mean = sums / ((rows > 0).sum() if c["per_sequence"] else rows.sum())
        return {"sums": sums, "counts": None, "row_tokens": None, "loss": torch.stack((mean[0] + KL_COEF * mean[1], mean[0], mean[1]))}
    d = -adv * ratio * (~cut)
    if c["kl"]:
        d = d - KL_COEF * torch.expm1(q)
    return {"dlogp": d * each * s["grad_loss"].double() / s["counts"][1 if c["per_sequence"] else 0]}
