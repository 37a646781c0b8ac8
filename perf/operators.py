"""Measured operators of the mixture-of-experts training and serving path.

Each case is one pass of a public entry point of the package, forward or
forward and backward, beside a plain form of the same operator in elementary
torch operations (32 bits, rounded once at the end).

Kinds
  route    moe_route: softmax, top-k and the stable sort of the chosen pairs by
           expert; with grad, the gradient of the logits as well
  product  grouped_matmul: products with the expert weights over ragged groups of
           rows; with grad, the gradients of the rows and of the weights as well
  combine  moe_combine: each token's weighted sum of its experts' rows; with
           grad, the gradients of the rows and of the weights as well
  distill  topk_distill_loss (how = "loss", or with its gradient how = "train"),
           topk_distill_loss_and_grad (how = "both"): the divergence of a
           student's logits from a teacher's top logits

The expert sizes are those of the repository's mixture-of-experts configuration
(64 experts, gate and up 1024 x 2048 each, down 2048 x 1024), 8 experts a token.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
# What a float32 sum of a teacher's probabilities can leave of 1 by rounding
# alone: a remainder below it is none.
REST = 1e-6


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quant-2bit_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import bcjr
    return bcjr


# ---------------------------------------------------------------------- cases

def _route(T, E, k, dtype, norm, padded, grad):
    """padded: a tenth of the tokens is padding, and some experts are masked."""
    return {"kind": "route", "T": T, "E": E, "k": k, "dtype": dtype, "norm": norm, "padded": padded, "grad": grad}


def _product(T, E, k, K, N, dtype, wtype, gather, grad):
    """gather: rows are taken from T tokens; else T * k rows are in order already."""
    return {"kind": "product", "T": T, "E": E, "k": k, "K": K, "N": N, "dtype": dtype, "wtype": wtype,
            "gather": gather, "grad": grad}


def _combine(T, E, k, N, dtype, grad):
    return {"kind": "combine", "T": T, "E": E, "k": k, "N": N, "dtype": dtype, "grad": grad}


def _distill(T, V, K, dtype, tau, rest, how):
    """rest: the teacher's mass outside its top entries is known, and counts."""
    return {"kind": "distill", "T": T, "V": V, "K": K, "dtype": dtype, "tau": tau, "rest": rest, "how": how}


def listed():
    return [
        # one step of decoding a batch of 8 sequences
        dict(_route(8, 64, 8, "bf16", False, False, False), name="route_decode"),
        # a training batch: padding at the sequences' ends, some experts masked
        dict(_route(16384, 64, 8, "f32", True, True, True), name="route_train"),
        # gate and up of a layer for the tokens of 4 decoding sequences
        dict(_product(4, 64, 8, 2048, 2048, "bf16", "bf16", True, False), name="product_decode"),
        # down of a layer for 64 decoding sequences, about 8 rows an expert
        dict(_product(64, 64, 8, 1024, 2048, "bf16", "bf16", False, False), name="product_batch"),
        # down of a layer for a prompt of 4096 tokens
        dict(_product(4096, 64, 8, 1024, 2048, "bf16", "bf16", False, False), name="product_prefill"),
        # gate and up of a layer in a quantization-aware training step: the quantizer's weights are float32
        dict(_product(4096, 64, 8, 2048, 2048, "bf16", "f32", True, True), name="product_train"),
        # a small layer of odd sizes, float16, forward and backward
        dict(_product(301, 7, 2, 517, 333, "f16", "f16", True, True), name="product_odd"),
        # the end of a layer in decoding
        dict(_combine(8, 64, 8, 2048, "bf16", False), name="combine_decode"),
        # the end of a layer in a training step
        dict(_combine(4096, 64, 8, 2048, "bf16", True), name="combine_train"),
        # scoring a handful of positions, a float32 head
        dict(_distill(16, 32000, 32, "f32", 1.0, False, "loss"), name="distill_score"),
        # a training step's loss through autograd, a vocabulary of odd size, softened
        dict(_distill(4096, 50257, 64, "bf16", 2.0, False, "train"), name="distill_train"),
        # a training step that takes loss and gradient in one call, large vocabulary, the teacher's rest counted
        dict(_distill(8192, 131072, 128, "bf16", 1.0, True, "both"), name="distill_both"),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 1 if n == 3072 else n


def _dim(rng, lo, hi):
    """A row length: as often a multiple of 64 as any number."""
    n = _log_int(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(["route", "product", "product", "combine", "distill", "distill"])
    E = _log_int(rng, 4, 64)
    k = rng.randint(1, min(E, 8))
    if kind == "route":
        E = _log_int(rng, 8, 256)
        return _route(_log_int(rng, 1, 16384), E, k, rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.5,
                      rng.random() < 0.5, rng.random() < 0.5)
    if kind == "product":
        dtype = rng.choice(["bf16", "bf16", "f16"])
        return _product(_log_int(rng, 1, 4096), E, k, _dim(rng, 64, 2048), _dim(rng, 64, 2048), dtype,
                        rng.choice([dtype, "f32"]), rng.random() < 0.5, rng.random() < 0.5)
    if kind == "combine":
        return _combine(_log_int(rng, 1, 4096), E, k, _dim(rng, 64, 2048), rng.choice(["f32", "bf16", "f16"]),
                        rng.random() < 0.5)
    V = _dim(rng, 1000, 131072)
    T = _log_int(rng, 1, max(1, min(8192, (1 << 29) // V)))
    return _distill(T, V, rng.choice([1, 8, 20, 64, 100, 256]), rng.choice(["f32", "bf16", "f16"]),
                    rng.choice([1.0, 2.0, 0.7]), rng.random() < 0.5, rng.choice(["loss", "train", "both"]))


# --------------------------------------------------------------------- inputs

def _routed(T, E, k, g):
    """A routing of T tokens in which some experts are preferred and some hardly
    chosen: (weights, experts, offsets, rows, slots) and the largest group."""
    bias = torch.randn(E, device=DEV, generator=g)
    l = torch.randn(T, E, device=DEV, generator=g) + bias
    top, pick = torch.sort(l, dim=1, descending=True, stable=True)
    pick = pick[:, :k]
    flat = pick.reshape(-1)
    count = torch.bincount(flat, minlength=E)
    order = torch.sort(flat, stable=True)[1]
    offsets = torch.zeros(E + 1, device=DEV, dtype=torch.int32)
    offsets[1:] = count.cumsum(0)
    slots = torch.empty_like(flat)
    slots[order] = torch.arange(T * k, device=DEV)
    return {"weights": torch.softmax(top[:, :k], 1), "experts": pick.int(), "offsets": offsets,
            "rows": (order // k).int(), "slots": slots.reshape(T, k).int(), "cap": int(count.max())}


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)

    def normal(*shape, dtype="f32", scale=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(TYPES[dtype])

    if case["kind"] == "route":
        T, E = case["T"], case["E"]
        s["logits"] = (torch.randn(T, E, device=DEV, generator=g) * 1.5 + torch.randn(E, device=DEV, generator=g)).to(
            TYPES[case["dtype"]])
        s["valid"] = None
        if case["padded"]:
            s["valid"] = torch.rand(T, device=DEV, generator=g) >= 0.1
            s["logits"][torch.rand(T, E, device=DEV, generator=g) < 0.05] = -math.inf
        s["gw"] = normal(T, case["k"])
    elif case["kind"] == "product":
        T, E, k, K, N = (case[n] for n in ("T", "E", "k", "K", "N"))
        s.update(_routed(T, E, k, g))
        s["x"] = normal(T if case["gather"] else T * k, K, dtype=case["dtype"])
        s["w"] = normal(E, N, K, dtype=case["wtype"], scale=K ** -0.5)
        s["gy"] = normal(T * k, N, dtype=case["dtype"]) if case["grad"] else None
    elif case["kind"] == "combine":
        T, E, k, N = (case[n] for n in ("T", "E", "k", "N"))
        s.update(_routed(T, E, k, g))
        s["y"] = normal(T * k, N, dtype=case["dtype"])
        s["go"] = normal(T, N, dtype=case["dtype"]) if case["grad"] else None
    else:
        T, V, K = case["T"], case["V"], case["K"]
        z = normal(T, V, scale=2.0)
        teacher = z + normal(T, V, scale=0.7)
        s["values"], s["indices"] = torch.topk(teacher, K, dim=1)
        s["indices"] = s["indices"].int()
        s["lse"] = torch.logsumexp(teacher / case["tau"], 1) if case["rest"] else None
        s["logits"] = z.to(TYPES[case["dtype"]])
        # the weight of each position in the batch's loss; a few positions are prompt, and count nothing.
        # float16 gradients need a loss scale, here 2^15
        s["weight"] = (torch.rand(T, device=DEV, generator=g) >= 0.1).float() * (
            (32768.0 if case["dtype"] == "f16" else 1.0) / T)
    return s


# ----------------------------------------------------------------- plain forms

def _plain_route(s):
    T, E, k = s["T"], s["E"], s["k"]
    l = s["logits"].float()
    if s["valid"] is not None:
        l = torch.where(s["valid"][:, None], l, -math.inf)
    top, pick = torch.sort(l, dim=1, descending=True, stable=True)
    top, pick = top[:, :k], pick[:, :k]
    live = top > -math.inf
    ref = torch.where(live[:, :1], top[:, :1], 0.0)
    e = torch.exp(l - ref)
    chosen = torch.exp(top - ref)
    total = (chosen if s["norm"] else e).sum(1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    weights = chosen / total
    experts = torch.where(live, pick, -1).int()
    key = torch.where(live, pick, E).reshape(-1)
    order = torch.sort(key, stable=True)[1]
    offsets = torch.zeros(E + 1, device=l.device, dtype=torch.int32)
    offsets[1:] = torch.bincount(key, minlength=E + 1)[:E].cumsum(0)
    at = torch.arange(T * k, device=l.device)
    rows = torch.where(at < offsets[E], order // k, -1).int()
    slots = torch.empty_like(order)
    slots[order] = at
    slots = torch.where(live, slots.reshape(T, k), -1).int()
    out = {"weights": weights, "experts": experts, "offsets": offsets, "rows": rows, "slots": slots}
    if s["grad"]:
        wg = weights * s["gw"]
        dot = wg.sum(1, keepdim=True)
        if s["norm"]:
            d = torch.zeros_like(l).scatter_add(1, pick, wg - weights * dot)
        else:
            d = (-(e / total) * dot).scatter_add(1, pick, wg)
        out["glogits"] = d.to(s["logits"].dtype)
    return out


def _plain_product(s):
    E, cap, M = s["E"], s["cap"], s["T"] * s["k"]
    offsets = s["offsets"].long()
    x, w = s["x"].float(), s["w"].to(s["x"].dtype).float()
    if s["gather"]:
        x = x[s["rows"].long()]
    # every group in a padded block of the largest group's height; row M is empty
    step = torch.arange(cap, device=x.device)
    at = offsets[:-1, None] + step
    at = torch.where(step < (offsets[1:] - offsets[:-1])[:, None], at, M)

    def blocks(rows):
        return torch.cat([rows, rows.new_zeros(1, rows.shape[1])])[at]

    def unblocked(b):
        out = b.new_zeros(M + 1, b.shape[2])
        out[at.reshape(-1)] = b.reshape(E * cap, -1)
        return out[:M]

    xb = blocks(x)
    y = unblocked(xb @ w.transpose(1, 2)).to(s["x"].dtype)
    if not s["grad"]:
        return {"y": y}
    gb = blocks(s["gy"].float())
    gx = unblocked(gb @ w)
    if s["gather"]:
        gx = gx[s["slots"].long()].sum(1)
    gw = gb.transpose(1, 2) @ xb
    return {"y": y, "gx": gx.to(s["x"].dtype), "gw": gw.to(s["w"].dtype)}


def _plain_combine(s):
    slots, w = s["slots"].long(), s["weights"]
    y = s["y"].float()
    picked = y[slots]
    out = {"out": (w[:, :, None] * picked).sum(1).to(s["y"].dtype)}
    if s["grad"]:
        go = s["go"].float()
        gy = torch.empty_like(y)
        gy[slots.reshape(-1)] = (w[:, :, None] * go[:, None, :]).reshape(-1, y.shape[1])
        out["gy"] = gy.to(s["y"].dtype)
        out["gweights"] = (picked * go[:, None, :]).sum(2)
    return out


def _plain_distill(s):
    tau = s["tau"]
    z = s["logits"].float() / tau
    t = s["values"].float() / tau
    at = s["indices"].long()
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    logp = torch.gather(z, 1, at) - top - torch.log(total)
    if s["rest"]:
        q = torch.exp(t - s["lse"][:, None])
        qr = 1.0 - q.sum(1, keepdim=True)
        qr = torch.where(qr > REST, qr, 0.0)
        pr = e.scatter(1, at, 0.0).sum(1, keepdim=True) / total
        loss = (q * (torch.log(q) - logp)).sum(1) + torch.where(qr > 0, qr * (torch.log(qr) - torch.log(pr)), 0.0)[:, 0]
        mass = q.sum(1, keepdim=True) + qr
        outside = mass - torch.where(qr > 0, qr / pr, 0.0)
    else:
        q = torch.exp(t - t.max(1, keepdim=True).values)
        q = q / q.sum(1, keepdim=True)
        loss = (q * (torch.log(q) - logp)).sum(1)
        mass = outside = torch.ones_like(total)
    if s["how"] == "loss":
        return {"loss": loss}
    g = s["weight"][:, None] / tau
    p = e / total
    d = (p * (g * outside)).scatter(1, at, g * (torch.gather(p, 1, at) * mass - q))
    return {"loss": loss, "glogits": d.to(s["logits"].dtype)}


# ------------------------------------------------------------ the package's own

def _own_route(s):
    b = _package()
    if not s["grad"]:
        r = b.moe_route(s["logits"], s["k"], renormalize=s["norm"], valid=s["valid"])
        return {"weights": r.weights, "experts": r.experts, "offsets": r.offsets, "rows": r.rows, "slots": r.slots}
    logits = s["logits"].detach().requires_grad_()
    r = b.moe_route(logits, s["k"], renormalize=s["norm"], valid=s["valid"])
    (gl,) = torch.autograd.grad(r.weights, logits, s["gw"])
    return {"weights": r.weights.detach(), "experts": r.experts, "offsets": r.offsets, "rows": r.rows,
            "slots": r.slots, "glogits": gl}


def _own_product(s):
    b = _package()
    rows, slots = (s["rows"], s["slots"]) if s["gather"] else (None, None)
    if not s["grad"]:
        return {"y": b.grouped_matmul(s["x"], s["w"], s["offsets"], rows=rows, slots=slots)}
    x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
    y = b.grouped_matmul(x, w, s["offsets"], rows=rows, slots=slots)
    gx, gw = torch.autograd.grad(y, (x, w), s["gy"])
    return {"y": y.detach(), "gx": gx, "gw": gw}


def _own_combine(s):
    b = _package()
    if not s["grad"]:
        return {"out": b.moe_combine(s["y"], s["weights"], s["rows"], s["slots"])}
    y, w = s["y"].detach().requires_grad_(), s["weights"].detach().requires_grad_()
    out = b.moe_combine(y, w, s["rows"], s["slots"])
    gy, gw = torch.autograd.grad(out, (y, w), s["go"])
    return {"out": out.detach(), "gy": gy, "gweights": gw}


def _own_distill(s):
    b = _package()
    if s["how"] == "both":
        loss, d = b.topk_distill_loss_and_grad(s["logits"], s["values"], s["indices"], s["weight"],
                                               temperature=s["tau"], teacher_lse=s["lse"])
        return {"loss": loss, "glogits": d}
    if s["how"] == "loss":
        return {"loss": b.topk_distill_loss(s["logits"], s["values"], s["indices"], temperature=s["tau"],
                                            teacher_lse=s["lse"])}
    logits = s["logits"].detach().requires_grad_()
    loss = b.topk_distill_loss(logits, s["values"], s["indices"], temperature=s["tau"], teacher_lse=s["lse"])
    (d,) = torch.autograd.grad(loss, logits, s["weight"])
    return {"loss": loss.detach(), "glogits": d}


PLAIN = {"route": _plain_route, "product": _plain_product, "combine": _plain_combine, "distill": _plain_distill}
OWN = {"route": _own_route, "product": _own_product, "combine": _own_combine, "distill": _own_distill}


def run(state):
    if own:
        return OWN[state["kind"]](state)
    with torch.no_grad():
        return PLAIN[state["kind"]](state)


# ----------------------------------------------------------------------- work

def work(case):
    c = case
    if c["kind"] == "route":
        T, E, k, b = c["T"], c["E"], c["k"], SIZE[c["dtype"]]
        n = T * E * b + T * k * 16 + (E + 1) * 4 + (T if c["padded"] else 0)
        if c["grad"]:
            n += T * E * b + T * k * 4
        return {"bytes": n, "flops": 4 * T * E}
    if c["kind"] == "product":
        T, E, k, K, N = (c[n] for n in ("T", "E", "k", "K", "N"))
        M, b, wb = T * k, SIZE[c["dtype"]], SIZE[c["wtype"]]
        x = (T if c["gather"] else M) * K * b
        # few tokens do not reach every expert: those that even choices would reach
        used = E * (1 - (1 - k / E) ** T)
        n = x + used * N * K * wb + M * N * b + (E + 1) * 4 + (M * 4 if c["gather"] else 0)
        if c["grad"]:
            n += M * N * b + x + E * N * K * wb
        return {"bytes": n, "flops": (6 if c["grad"] else 2) * M * N * K}
    if c["kind"] == "combine":
        T, k, N, b = c["T"], c["k"], c["N"], SIZE[c["dtype"]]
        n = (T * k + T) * N * b + T * k * 8
        if c["grad"]:
            n += (T * k + T) * N * b + T * k * 4
        return {"bytes": n, "flops": (6 if c["grad"] else 2) * T * k * N}
    T, V, K, b = c["T"], c["V"], c["K"], SIZE[c["dtype"]]
    n = T * V * b + T * K * 8 + T * 4 + (T * 4 if c["rest"] else 0)
    if c["how"] != "loss":
        n += T * V * b + T * 4
    return {"bytes": n, "flops": (4 if c["how"] == "loss" else 7) * T * V}


# ------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "product": _exact_product, "combine": _exact_combine,
                "distill": _exact_distill}[case["kind"]](s)


def _exact_route(s):
    T, E, k = s["T"], s["E"], s["k"]
    l = s["logits"].double().cpu()
    if s["valid"] is not None:
        l[~s["valid"].cpu()] = -math.inf
    p = torch.nan_to_num(torch.softmax(l, 1), nan=0.0)
    chosen = torch.argsort(-l, dim=1, stable=True)[:, :k]
    live = torch.gather(l, 1, chosen) > -math.inf
    w = torch.gather(p, 1, chosen)
    scale = w.sum(1, keepdim=True) if s["norm"] else torch.ones(T, 1, dtype=torch.float64)
    w = torch.where(live, w / torch.where(scale > 0, scale, 1.0), 0.0)
    groups = []
    slots = torch.full((T, k), -1, dtype=torch.int32)
    offsets, n = [0], 0
    for e in range(E):
        t, j = torch.nonzero((chosen == e) & live, as_tuple=True)
        slots[t, j] = torch.arange(n, n + len(t), dtype=torch.int32)
        groups.append(t.int())
        n += len(t)
        offsets.append(n)
    rows = torch.cat(groups + [torch.full((T * k - n,), -1, dtype=torch.int32)])
    out = {"weights": w, "experts": torch.where(live, chosen, -1).int(),
           "offsets": torch.tensor(offsets, dtype=torch.int32), "rows": rows, "slots": slots}
    if s["grad"]:
        gw = s["gw"].double().cpu()
        base = p / torch.where(scale > 0, scale, 1.0)  # the weight that every expert has, chosen or not
        mask = torch.zeros(T, E, dtype=torch.float64).scatter_(1, chosen, live.double())
        up = torch.zeros(T, E, dtype=torch.float64).scatter_(1, chosen, gw)
        in_sum = mask if s["norm"] else torch.ones_like(mask)
        mean = (base * mask * up).sum(1, keepdim=True)
        out["glogits"] = base * (mask * up - in_sum * mean)
    return {n: v.to(DEV) for n, v in out.items()}


def _exact_product(s):
    E = s["E"]
    o = s["offsets"].tolist()
    M, N, K = s["T"] * s["k"], s["N"], s["K"]
    of = s["rows"].long() if s["gather"] else torch.arange(M, device=DEV)
    y = torch.zeros(M, N, device=DEV, dtype=torch.float64)
    if s["grad"]:
        gx = torch.zeros(s["x"].shape, device=DEV, dtype=torch.float64)
        gw = torch.zeros(E, N, K, device=DEV, dtype=torch.float64)
    for e in range(E):
        a, b = o[e], o[e + 1]
        if a == b:
            continue
        xe, we = s["x"][of[a:b]].double(), s["w"][e].to(s["x"].dtype).double()
        y[a:b] = torch.mm(xe, we.t())
        if s["grad"]:
            ge = s["gy"][a:b].double()
            gx.index_add_(0, of[a:b], torch.mm(ge, we))
            gw[e] = torch.mm(ge.t(), xe)
    return {"y": y, "gx": gx, "gw": gw} if s["grad"] else {"y": y}


def _exact_combine(s):
    T, k = s["T"], s["k"]
    w, y = s["weights"].double(), s["y"].double()
    out = torch.zeros(T, s["N"], device=DEV, dtype=torch.float64)
    for j in range(k):
        out += w[:, j, None] * y[s["slots"][:, j].long()]
    if not s["grad"]:
        return {"out": out}
    go = s["go"].double()
    gy, gw = torch.zeros_like(y), torch.zeros_like(w)
    for j in range(k):
        at = s["slots"][:, j].long()
        gy[at] = w[:, j, None] * go
        gw[:, j] = torch.linalg.vecdot(go, y[at])
    return {"out": out, "gy": gy, "gweights": gw}


def _exact_distill(s):
    T, tau = s["T"], s["tau"]
    loss = torch.empty(T, device=DEV, dtype=torch.float64)
    d = torch.empty(s["logits"].shape, device=DEV, dtype=torch.float64) if s["how"] != "loss" else None
    step = max(1, (1 << 27) // s["V"])
    for a in range(0, T, step):
        part = slice(a, min(T, a + step))
        at = s["indices"][part].long()
        lp = torch.log_softmax(s["logits"][part].double() / tau, 1)
        t = s["values"][part].double() / tau
        lq = t - s["lse"][part, None].double() if s["rest"] else torch.log_softmax(t, 1)
        q = lq.exp()
        l = (q * (lq - lp.gather(1, at))).sum(1)
        # target - p, with the rest of the teacher's mass shared as the student shares it
        target = torch.zeros_like(lp).scatter(1, at, q)
        mass = torch.ones(q.shape[0], dtype=torch.float64, device=DEV)
        if s["rest"]:
            qr = 1.0 - q.sum(1)
            qr = torch.where(qr > REST, qr, 0.0)
            others = torch.logsumexp(lp.scatter(1, at, -math.inf), 1)
            l = l + torch.where(qr > 0, qr * (qr.log() - others), 0.0)
            mass = q.sum(1) + qr
            target = target + (lp - others[:, None]).exp().scatter(1, at, 0.0) * qr[:, None]
        loss[part] = l
        if d is not None:
            d[part] = (lp.exp() * mass[:, None] - target) * (s["weight"][part, None].double() / tau)
    return {"loss": loss} if d is None else {"loss": loss, "glogits": d}
