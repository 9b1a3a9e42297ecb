"""Performance cases of the optimizer-step operators beside the whole-matrix Newton-Schulz.

Three operators, each in its plain torch form (``own = False``) and as the
calls a user makes of ``muon_fused`` (``own = True``):

* ``heads``   per-head Newton-Schulz orthogonalisation of attention projections;
* ``adamw``   AdamW over a list of tensors (embeddings, norms, biases);
* ``normed``  decay + neuron-wise normalised update of a list of matrices.
"""

import math

import torch

own = False

NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LR, WD, BETAS, EPS = 0.003, 0.1, (0.9, 0.95), 1e-8


def listed():
    return [
        # one small projection: the latency of a single call
        {"name": "heads_one_small", "op": "heads", "batch": 1, "rows": 512, "cols": 512,
         "heads": 8, "dim": 0, "dtype": "bf16", "steps": 5},
        # query projection of the 8B-class shape set, 32 heads of 128 rows
        {"name": "heads_query", "op": "heads", "batch": 1, "rows": 4096, "cols": 4096,
         "heads": 32, "dim": 0, "dtype": "bf16", "steps": 5},
        # output projection of the same set: each head is a block of columns
        {"name": "heads_output", "op": "heads", "batch": 1, "rows": 4096, "cols": 4096,
         "heads": 32, "dim": 1, "dtype": "bf16", "steps": 5},
        # fused query/key/value projections of eight layers in one call
        {"name": "heads_qkv_layers", "op": "heads", "batch": 8, "rows": 6144, "cols": 4096,
         "heads": 48, "dim": 0, "dtype": "bf16", "steps": 5},
        # odd sizes: 72-row heads, an input length that no vector width divides, fp16
        {"name": "heads_odd", "op": "heads", "batch": 3, "rows": 1080, "cols": 1001,
         "heads": 15, "dim": 0, "dtype": "fp16", "steps": 5},
        # the norm weights of ten layers: launch-bound
        {"name": "adamw_norms", "op": "adamw", "sizes": "20*4096", "dtype": "fp32",
         "moments": "fp32", "step": 7},
        # an embedding, a head bias and odd vectors, 16-bit weights with 32-bit moments
        {"name": "adamw_mixed", "op": "adamw",
         "sizes": "32003x2048,32003,2048x16,1,7,1001,65537", "dtype": "bf16", "moments": "fp32",
         "step": 1000},
        # a large embedding in 32 bits
        {"name": "adamw_embedding", "op": "adamw", "sizes": "65536x4096,4096", "dtype": "fp32",
         "moments": "fp32", "step": 3},
        # one small matrix
        {"name": "normed_small", "op": "normed", "count": 1, "rows": 896, "cols": 1152,
         "dtype": "bf16"},
        # the four attention projections of the 1B-class set, 32-bit master weights
        {"name": "normed_attention", "op": "normed", "count": 4, "rows": 2048, "cols": 2048,
         "dtype": "fp32"},
        # down projections of the 8B-class set, longer than the L2 holds together
        {"name": "normed_down", "op": "normed", "count": 6, "rows": 4096, "cols": 14336,
         "dtype": "bf16"},
        # odd rows and columns: no 16-byte row starts
        {"name": "normed_odd", "op": "normed", "count": 5, "rows": 1003, "cols": 2731,
         "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["heads", "adamw", "normed"])
    if op == "heads":
        d = rng.choice([16, 32, 48, 64, 72, 80, 96, 112, 128, rng.randint(16, 128)])
        heads = _log(rng, 1, 64)
        other = _log(rng, 64, 8192)
        limit = 8 * 6144 * 4096
        batch = min(_log(rng, 1, 16), max(1, limit // (d * heads * other)))
        dim = rng.randint(0, 1)
        return {"op": op, "batch": batch, "rows": d * heads if dim == 0 else other,
                "cols": other if dim == 0 else d * heads, "heads": heads, "dim": dim,
                "dtype": rng.choice(["bf16", "fp16"]), "steps": 5}
    if op == "adamw":
        sizes = [str(_log(rng, 1, 100000)) for _ in range(rng.randint(1, 10))]
        if rng.random() < 0.7:
            sizes.append("%dx%d" % (_log(rng, 1000, 65536), _log(rng, 64, 4096)))
        rng.shuffle(sizes)
        return {"op": op, "sizes": ",".join(sizes), "dtype": rng.choice(["fp32", "bf16", "fp16"]),
                "moments": "fp32", "step": _log(rng, 1, 100000)}
    rows, cols = _log(rng, 32, 16384), _log(rng, 32, 16384)
    limit = 6 * 4096 * 14336
    return {"op": op, "count": min(_log(rng, 1, 8), max(1, limit // (rows * cols))), "rows": rows,
            "cols": cols, "dtype": rng.choice(["fp32", "bf16", "fp16"])}


def _shapes(text):
    """Tensor shapes of a list: "32003x2048,7" a matrix and a vector, "20*4096" twenty vectors."""
    out = []
    for item in text.split(","):
        count, _, shape = item.rpartition("*")
        out += [tuple(int(x) for x in shape.split("x"))] * int(count or 1)
    return out


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "heads":
        # a momentum direction: noise plus a few strong directions with a decaying spectrum
        b, r, c = case["batch"], case["rows"], case["cols"]
        g = _randn(gen, b, r, c)
        s = 4.0 / torch.arange(1, 17, device="cuda", dtype=torch.float32)
        g += (_randn(gen, b, r, 16) * s) @ _randn(gen, b, 16, c)
        g *= 1e-3
        g = g.to(DTYPES[case["dtype"]])
        return {"case": case, "G": g if b > 1 else g[0]}
    dt = DTYPES[case["dtype"]]
    if case["op"] == "adamw":
        mt = DTYPES[case["moments"]]
        st = {"case": case, "p": [], "g": [], "m": [], "v": []}
        for shape in _shapes(case["sizes"]):
            st["p"].append((_randn(gen, *shape) * 0.02).to(dt))
            st["g"].append((_randn(gen, *shape) * 1e-3).to(dt))
            st["m"].append((_randn(gen, *shape) * 3e-4).to(mt))
            st["v"].append(((_randn(gen, *shape) * 1e-3).square() + 1e-8).to(mt))
        return st
    r, c = case["rows"], case["cols"]
    st = {"case": case, "p": [], "v": []}
    u = torch.empty(case["count"], r, c, device="cuda", dtype=torch.bfloat16)
    for i in range(case["count"]):
        # orthogonalised rows have a mean square near 1/max(r, c), some rows more, some less
        spread = torch.exp(0.5 * _randn(gen, r, 1))
        u[i] = _randn(gen, r, c) * spread / math.sqrt(max(r, c))
        st["v"].append((spread[:, 0].square() * torch.exp(0.3 * _randn(gen, r))) / max(r, c))
        st["p"].append((_randn(gen, r, c) * 0.02).to(dt))
    st["u"] = u
    return st


# ----------------------------------------------------------------- plain forms
def _plain_heads(G, heads, steps, dim):
    g = G if G.dim() == 3 else G[None]
    b, r, c = g.shape
    x = g.float()
    # (batch, heads, head side, other side)
    x = x.view(b, heads, r // heads, c) if dim == 0 else x.view(b, r, heads, c // heads).permute(0, 2, 3, 1)
    x = x / (x.square().sum(dim=(2, 3), keepdim=True).sqrt() + 1e-7)
    for _ in range(steps):
        a = x @ x.transpose(2, 3)
        x = NS_A * x + (NS_B * a + NS_C * (a @ a)) @ x
    x = x if dim == 0 else x.permute(0, 3, 1, 2)
    return x.reshape(G.shape).to(torch.bfloat16)


def _plain_adamw(p, g, m, v, step):
    scale = (1 - BETAS[0] ** step) / (1 - BETAS[1] ** step) ** 0.5
    gf = g.float()
    m.copy_(m.float() + (1 - BETAS[0]) * (gf - m.float()))
    v.copy_(v.float() + (1 - BETAS[1]) * (gf * gf - v.float()))
    p.copy_(p.float() * (1 - LR * WD) - (LR / scale) * (m.float() / (EPS + v.float().sqrt())))


def _plain_normed(p, u, v):
    uf = u.float()
    v.copy_(BETAS[1] * v + (1 - BETAS[1]) * uf.square().mean(dim=1))
    o = uf / (v.sqrt() + EPS)[:, None]
    step = LR * 0.2 * math.sqrt(u.numel()) / (o.square().sum().sqrt() + 1e-7)
    p.copy_(p.float() * (1 - LR * WD) - step * o)


def run(state):
    case = state["case"]
    if case["op"] == "heads":
        if own:
            from muon_fused import fused_newton_schulz_heads

            return fused_newton_schulz_heads(state["G"], case["heads"], case["steps"],
                                             dim=case["dim"])
        return _plain_heads(state["G"], case["heads"], case["steps"], case["dim"])
    if case["op"] == "adamw":
        if own:
            from muon_fused import fused_adamw

            fused_adamw(state["p"], state["g"], state["m"], state["v"], case["step"], lr=LR, wd=WD,
                        betas=BETAS, eps=EPS)
        else:
            for p, g, m, v in zip(state["p"], state["g"], state["m"], state["v"]):
                _plain_adamw(p, g, m, v, case["step"])
        return state["p"], state["m"], state["v"]
    if own:
        from muon_fused import fused_normed_update

        fused_normed_update(state["p"], state["u"], state["v"], lr=LR, wd=WD, beta2=BETAS[1],
                            eps=EPS)
    else:
        for p, u, v in zip(state["p"], state["u"], state["v"]):
            _plain_normed(p, u, v)
    return state["p"], state["v"]


def work(case):
    if case["op"] == "heads":
        b, r, c, h, k = case["batch"], case["rows"], case["cols"], case["heads"], case["steps"]
        d, n = (r // h, c) if case["dim"] == 0 else (c // h, r)
        # one triangle of the Gram matrix, four symmetric d x d products an iteration, one product with G
        per = d * (d + 1) * n + 4 * k * d ** 3 + 2 * d * d * n
        return {"bytes": 4 * b * r * c, "flops": b * h * per}
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case["sizes"]))
        e, me = DTYPES[case["dtype"]].itemsize, DTYPES[case["moments"]].itemsize
        return {"bytes": n * (3 * e + 4 * me), "flops": 15 * n}
    n = case["count"] * case["rows"] * case["cols"]
    e = DTYPES[case["dtype"]].itemsize
    return {"bytes": n * (2 + 2 * e) + 8 * case["count"] * case["rows"], "flops": 5 * n}


# ---------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "heads":
        g = st["G"].double()
        g = g if g.dim() == 3 else g.unsqueeze(0)
        blocks = torch.stack(g.chunk(case["heads"], dim=1 + case["dim"]), dim=1)
        if case["dim"] == 1:
            blocks = blocks.mT
        x = blocks / (torch.linalg.vector_norm(blocks, dim=(2, 3), keepdim=True) + 1e-7)
        for _ in range(case["steps"]):
            gram = x @ x.mT
            ax = gram @ x
            x = NS_A * x + NS_B * ax + NS_C * (gram @ ax)
        if case["dim"] == 1:
            x = x.mT
        return torch.cat(x.unbind(1), dim=1 + case["dim"]).reshape(st["G"].shape)
    if case["op"] == "adamw":
        b1, b2 = BETAS
        corr1, corr2 = 1 - b1 ** case["step"], 1 - b2 ** case["step"]
        m = [b1 * m.double() + (1 - b1) * g.double() for m, g in zip(st["m"], st["g"])]
        v = [b2 * v.double() + (1 - b2) * g.double() ** 2 for v, g in zip(st["v"], st["g"])]
        p = [(1 - LR * WD) * p.double() - LR * corr2 ** 0.5 / corr1 * mi / (EPS + vi ** 0.5)
             for p, mi, vi in zip(st["p"], m, v)]
        return p, m, v
    out_p, out_v = [], []
    for p, u, v in zip(st["p"], st["u"], st["v"]):
        u64 = u.double()
        v64 = BETAS[1] * v.double() + (1 - BETAS[1]) * (u64 * u64).sum(1) / u.shape[1]
        n64 = torch.div(u64, (v64 ** 0.5 + EPS).unsqueeze(1))
        eta = 0.2 * LR * (u.shape[0] * u.shape[1]) ** 0.5 / (torch.linalg.matrix_norm(n64) + 1e-7)
        out_p.append((1 - LR * WD) * p.double() - eta * n64)
        out_v.append(v64)
    return out_p, out_v
