"""Workloads of the sublayer operators: the projection with per-request low-rank adapters (``gemm_peak_lora``) and
the norms around a block fused with its gate and the scaled residual (``rms_norm_residual_fwd`` / ``_bwd``).

``run`` computes a case with elementary torch operations in 32 bits, or, where ``own`` is true, with the calls of
the package; ``exact`` evaluates the definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one decoded token of one request at a benchmark width: launch latency
        dict(name="norm_fwd_1", op="fwd", rows=1, h=4096, dtype="bf16", post=True, pre=True, gates=0, res_scale="none"),
        # a decode batch, every token with its own gate
        dict(name="norm_fwd_64", op="fwd", rows=64, h=8192, dtype="fp16", post=True, pre=True, gates=64,
             res_scale="one"),
        # prompts: 17 sequences of 59 tokens, one gate per sequence, learned residual scale per channel
        dict(name="norm_fwd_1003", op="fwd", rows=1003, h=5120, dtype="fp16", post=True, pre=True, gates=17,
             res_scale="column"),
        # a training step: the row count and width of the RMSNorm benchmark, 8 sequences
        dict(name="norm_fwd_32768", op="fwd", rows=32768, h=4096, dtype="bf16", post=True, pre=True, gates=8,
             res_scale="one"),
        # gradients of a short batch: 4 sequences of 59 tokens
        dict(name="norm_bwd_236", op="bwd", rows=236, h=2048, dtype="bf16", post=True, pre=True, gates=4,
             res_scale="one"),
        # gradients with one gate per token, an odd number of tokens
        dict(name="norm_bwd_4099", op="bwd", rows=4099, h=5120, dtype="fp16", post=True, pre=True, gates=4099,
             res_scale="none"),
        # gradients of a training step at the wide benchmark width, everything learned
        dict(name="norm_bwd_16384", op="bwd", rows=16384, h=8192, dtype="bf16", post=True, pre=True, gates=8,
             res_scale="column"),
        # one decoded token, one adapter
        dict(name="lora_1", op="lora", m=1, n=4096, k=4096, rank=16, pool=8, active=1, order="mixed", dtype="bf16",
             terms=False),
        # a decode batch of many requests: 32 adapters in use among 64 tokens, some tokens without one
        dict(name="lora_64", op="lora", m=64, n=14336, k=4096, rank=16, pool=64, active=32, order="mixed",
             dtype="bf16", terms=False),
        # a wider decode batch on the down projection, larger rank, with the norm's row scale, bias and residual
        dict(name="lora_128", op="lora", m=128, n=4096, k=14336, rank=64, pool=32, active=20, order="mixed",
             dtype="fp16", terms=True),
        # a few prompts of uneven length, sizes that are no multiple of any tile
        dict(name="lora_1003", op="lora", m=1003, n=4104, k=5128, rank=24, pool=16, active=5, order="runs",
             dtype="fp16", terms=False),
        # prompts of 8 requests at once at the largest benchmark projection of this kind
        dict(name="lora_4096", op="lora", m=4096, n=14336, k=4096, rank=16, pool=16, active=8, order="runs",
             dtype="bf16", terms=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["fwd", "bwd", "lora"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "lora":
        while True:
            m = _log_uniform(rng, 1, 4096)
            n, k = (8 * _log_uniform(rng, 32, 1792) for _ in range(2))
            if m * n * k <= 4096 * 14336 * 4096:
                break
        pool = _log_uniform(rng, 1, 64)
        return dict(op=op, m=m, n=n, k=k, rank=rng.choice([8, 16, 24, 32, 64, 128]), pool=pool,
                    active=rng.randint(1, min(pool, m)), order=rng.choice(["mixed", "runs"]), dtype=dtype,
                    terms=rng.random() < 0.5)
    while True:
        rows, h = _log_uniform(rng, 1, 32768), 8 * _log_uniform(rng, 8, 2048)
        if rows * h <= 1 << 27:
            break
    divisors = [d for d in range(1, rows + 1) if rows % d == 0]
    post = rng.random() < 0.8
    return dict(op=op, rows=rows, h=h, dtype=dtype, post=post, pre=not post or rng.random() < 0.8,
                gates=rng.choice([0, 1, rng.choice(divisors), rows]), res_scale=rng.choice(["none", "one", "column"]))


# ------------------------------------------------------------------ inputs ----

def _ids(case, g):
    """Adapter of every token: each adapter in use occurs, about an eighth of the remaining tokens have none."""
    m, pool, active = case["m"], case["pool"], case["active"]
    chosen = torch.randperm(pool, generator=g, device="cuda")[:active]
    if case["order"] == "mixed":
        place = torch.arange(m, device="cuda") % active
    else:
        place = (torch.rand(m, generator=g, device="cuda") ** 1.5 * active).long().clamp(max=active - 1)
        place[:active] = torch.arange(active, device="cuda")
    none = torch.rand(m, generator=g, device="cuda") < 0.125
    none[:active] = False
    ids = torch.where(none, torch.full_like(place, -1), chosen[place])
    order = torch.randperm(m, generator=g, device="cuda") if case["order"] == "mixed" else torch.argsort(ids, stable=True)
    return ids[order].int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    st = {"case": case}
    if case["op"] == "lora":
        m, n, k, r, pool = (case[x] for x in ("m", "n", "k", "rank", "pool"))
        st["x"] = normal(m, k)
        st["w"] = normal(n, k, std=0.02)
        st["a"] = normal(pool, r, k, std=k ** -0.5)
        st["b"] = normal(pool, n, r, std=0.02)
        st["scale"] = 0.5 + 1.5 * torch.rand(pool, generator=g, device="cuda")
        st["ids"] = _ids(case, g)
        st["row_scale"] = st["bias"] = st["residual"] = None
        if case["terms"]:
            st["row_scale"] = 0.5 + torch.rand(m, generator=g, device="cuda")
            st["bias"] = normal(n)
            st["residual"] = normal(m, n)
        st["d"] = torch.empty(m, n, dtype=dt, device="cuda")
        return st
    rows, h = case["rows"], case["h"]
    st["u"] = normal(rows, h)
    st["residual"] = normal(rows, h)
    st["gamma_post"] = normal(h, std=0.1, mean=1.0, dtype=torch.float32) if case["post"] else None
    st["gamma_pre"] = normal(h, std=0.1, mean=1.0, dtype=torch.float32) if case["pre"] else None
    st["gate"] = normal(case["gates"], h, std=0.5) if case["gates"] else None
    st["res_scale"] = None
    if case["res_scale"] != "none":
        st["res_scale"] = normal(1 if case["res_scale"] == "one" else h, std=0.1, mean=1.0, dtype=torch.float32)
    if case["op"] == "fwd":
        st["s"] = torch.empty(rows, h, dtype=dt, device="cuda")
        st["y"] = torch.empty_like(st["s"]) if case["pre"] else None
        return st
    st["s"] = _forward(st)[0].to(dt)
    # the loss's slope along the stream it changes is not zero on average
    st["ds"] = (normal(rows, h).float() + 0.1 * st["residual"].float()).to(dt)
    st["dy"] = normal(rows, h) if case["pre"] else None
    for name in ("gamma_post", "gate", "res_scale", "gamma_pre"):
        st["d" + name] = None if st[name] is None else torch.empty_like(st[name])
    st["du"], st["dresidual"] = torch.empty_like(st["u"]), torch.empty_like(st["u"])
    return st


# ------------------------------------------------------------- plain forms ----

def _rstd(v):
    return 1.0 / torch.sqrt(v.square().mean(dim=-1, keepdim=True) + EPS)


def _per_row(gate, rows):
    """The gate of every row: consecutive rows / gates rows share one."""
    return gate.float().repeat_interleave(rows // gate.shape[0], dim=0)


def _forward(st):
    """(s, y) in 32 bits."""
    u = st["u"].float()
    p = u if st["gamma_post"] is None else u * _rstd(u) * st["gamma_post"]
    if st["gate"] is not None:
        p = p * _per_row(st["gate"], u.shape[0])
    res = st["residual"].float()
    s = p + (res if st["res_scale"] is None else res * st["res_scale"])
    return s, None if st["gamma_pre"] is None else s * _rstd(s) * st["gamma_pre"]


def _backward(st):
    rows = st["u"].shape[0]
    s, u, big = st["s"].float(), st["u"].float(), st["ds"].float()
    out = {}
    if st["gamma_pre"] is not None:
        rs = _rstd(s)
        shat, dy = s * rs, st["dy"].float()
        gy = dy * st["gamma_pre"]
        big = big + rs * (gy - shat * (gy * shat).mean(dim=-1, keepdim=True))
        out["dgamma_pre"] = (dy * shat).sum(dim=0)
    if st["res_scale"] is None:
        out["dresidual"] = big
    else:
        out["dresidual"] = big * st["res_scale"]
        dscale = big * st["residual"].float()
        out["dres_scale"] = dscale.sum(dim=0) if st["res_scale"].numel() > 1 else dscale.sum(dtype=torch.float64).float().view(1)
    e = big if st["gate"] is None else big * _per_row(st["gate"], rows)
    ru = None if st["gamma_post"] is None else _rstd(u)
    uhat = u if ru is None else u * ru
    if st["gate"] is not None:
        p = uhat if ru is None else uhat * st["gamma_post"]
        out["dgate"] = (big * p).view(st["gate"].shape[0], -1, u.shape[1]).sum(dim=1)
    if ru is None:
        out["du"] = e
    else:
        out["dgamma_post"] = (e * uhat).sum(dim=0)
        ge = e * st["gamma_post"]
        out["du"] = ru * (ge - uhat * (ge * uhat).mean(dim=-1, keepdim=True))
    return {k: v.to(torch.float32 if k in ("dgamma_pre", "dgamma_post", "dres_scale") else st["u"].dtype)
            for k, v in out.items()}


def _lora(st):
    x, a, b = st["x"].float(), st["a"].float(), st["b"].float()
    pool, r, k = a.shape
    mine = st["ids"].long()[:, None] == torch.arange(pool, device=x.device)[None, :]          # [m, pool]
    v = (x @ a.view(pool * r, k).t()).view(-1, pool, r) * (mine * st["scale"])[:, :, None]
    y = x @ st["w"].float().t() + v.view(-1, pool * r) @ b.transpose(1, 2).reshape(pool * r, -1)
    if st["row_scale"] is not None:
        y = y * st["row_scale"][:, None] + st["bias"].float() + st["residual"].float()
    return y.to(st["x"].dtype)


def run(st):
    op = st["case"]["op"]
    if own:
        import PeakGemm

        if op == "lora":
            PeakGemm.gemm_peak_lora(st["d"], st["x"], st["w"], st["a"], st["b"], st["ids"], scale=st["scale"],
                                    row_scale=st["row_scale"], bias=st["bias"], residual=st["residual"])
            return {"d": st["d"]}
        params = {n: st[n] for n in ("gamma_post", "gate", "res_scale", "gamma_pre")}
        if op == "fwd":
            PeakGemm.rms_norm_residual_fwd(st["s"], st["y"], st["u"], st["residual"], eps=EPS, **params)
            return {"s": st["s"], "y": st["y"]}
        grads = {"d" + n: st["d" + n] for n in params}
        PeakGemm.rms_norm_residual_bwd(st["du"], st["dresidual"], st["dy"], st["ds"], st["s"], st["u"],
                                       residual=st["residual"], eps=EPS, **params, **grads)
        return {k: v for k, v in dict(du=st["du"], dresidual=st["dresidual"], **grads).items() if v is not None}
    if op == "lora":
        return {"d": _lora(st)}
    if op == "fwd":
        s, y = _forward(st)
        return {"s": s.to(st["u"].dtype), "y": None if y is None else y.to(st["u"].dtype)}
    return _backward(st)


# -------------------------------------------------------------------- work ----

def work(case):
    if case["op"] == "lora":
        m, n, k, r = case["m"], case["n"], case["k"], case["rank"]
        extra = 2 * m * n + 2 * n + 4 * m if case["terms"] else 0
        return {"bytes": 2 * (m * k + n * k + m * n) + 2 * case["active"] * r * (n + k) + 4 * m + 4 * case["active"] + extra,
                "flops": 2 * m * n * k + 2 * m * r * (n + k)}
    rows, h = case["rows"], case["h"]
    column = {"none": 0, "one": 1, "column": h}[case["res_scale"]]
    vectors = 4 * (h * (case["post"] + case["pre"]) + column)
    if case["op"] == "fwd":
        tensors = 4 if case["pre"] else 3                                  # u, residual, s, y
        return {"bytes": 2 * tensors * rows * h + 2 * case["gates"] * h + vectors, "flops": 12 * rows * h}
    # ds, u, du, dresidual; s and dy with the norm before the next block; residual for the residual scale's gradient
    tensors = 4 + 2 * case["pre"] + (column > 0)
    if not case["post"] and not case["gates"]:
        tensors -= 1                                                        # u is not needed
    return {"bytes": 2 * tensors * rows * h + 4 * case["gates"] * h + 2 * vectors, "flops": 30 * rows * h}


# ------------------------------------------------------------------- exact ----

def exact(case, seed):
    """The definitions, in 64 bits."""
    st = prepare(case, seed)
    d = {k: v.double() for k, v in st.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "lora":
        y = torch.matmul(d["x"], d["w"].mT)
        for a in st["ids"].unique().tolist():
            if a >= 0:
                t = (st["ids"] == a).nonzero()[:, 0]
                y[t] += torch.matmul(torch.matmul(d["x"][t], d["a"][a].mT), d["b"][a].mT) * d["scale"][a]
        if case["terms"]:
            y = d["row_scale"].unsqueeze(1) * y + d["bias"] + d["residual"]
        return {"d": y}
    rows, h = case["rows"], case["h"]

    def grouped(t):                              # [groups, rows of a group, h]
        return t.reshape(max(1, case["gates"]), -1, h)

    gate = d["gate"][:, None, :] if case["gates"] else torch.ones(1, 1, 1, dtype=torch.float64, device="cuda")
    inv_u = (d["u"].pow(2).sum(-1, keepdim=True) / h + EPS).pow(-0.5) if case["post"] else torch.ones_like(d["u"][:, :1])
    gp = d.get("gamma_post", torch.ones(1, dtype=torch.float64, device="cuda"))
    alpha = d.get("res_scale", torch.ones(1, dtype=torch.float64, device="cuda"))
    if case["op"] == "fwd":
        s = alpha * d["residual"] + (gate * grouped(d["u"] * inv_u * gp)).reshape(rows, h)
        y = s * (s.pow(2).sum(-1, keepdim=True) / h + EPS).pow(-0.5) * d["gamma_pre"] if case["pre"] else None
        return {"s": s, "y": y}
    out, total = {}, d["ds"]
    if case["pre"]:
        inv_s = (d["s"].pow(2).sum(-1, keepdim=True) / h + EPS).pow(-0.5)
        w = d["dy"] * d["gamma_pre"]
        # d(s * inv_s) = inv_s ds - s inv_s^3 <s, ds> / h
        total = total + inv_s * w - d["s"] * inv_s.pow(3) * ((w * d["s"]).sum(-1, keepdim=True) / h)
        out["dgamma_pre"] = (d["dy"] * d["s"] * inv_s).sum(0)
    out["dresidual"] = alpha * total
    if case["res_scale"] != "none":
        dscale = (total * d["residual"]).sum(0)
        out["dres_scale"] = dscale if case["res_scale"] == "column" else dscale.sum().reshape(1)
    if case["gates"]:
        out["dgate"] = grouped(total * d["u"] * inv_u * gp).sum(1)
    e = (gate * grouped(total)).reshape(rows, h)
    if case["post"]:
        out["dgamma_post"] = (e * d["u"] * inv_u).sum(0)
        w = e * gp
        out["du"] = inv_u * w - d["u"] * inv_u.pow(3) * ((w * d["u"]).sum(-1, keepdim=True) / h)
    else:
        out["du"] = e
    return out
