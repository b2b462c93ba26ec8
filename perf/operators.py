"""Timed cases of the softmax read-out and of the orthogonalised update.

Four operators: ``log_probs`` (log probabilities of given outcomes under a softmax of each row, with the row's entropy and
its most probable outcomes), ``log_probs_grad`` (the same log probabilities and entropies with the gradient of a loss that
weighs them), ``orthogonalize`` (Newton-Schulz products that carry a matrix's singular values towards 1) and ``muon_step``
(momentum, orthogonalisation and weight update).  With ``own`` the calls go to ``vqa_amd``, else they are computed from
elementary torch operations."""
import math

import torch

own = False

COEFS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
DTYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LARGEST_ROWS = 2048 * 100003     # logits of the largest listed read-out
LARGEST_PRODUCT = 4096 ** 3      # rows * columns * shorter side of the largest listed matrix


def listed():
    return [
        # one batch of the four-qubit Iris classifier: 105 training samples, three classes
        {"name": "score iris", "op": "score", "rows": 105, "width": 3, "top": 3, "scale": 4.0, "type": "f64"},
        # the twelve Z values of a 12-qubit register for a batch of 65536 samples
        {"name": "score 12 outcomes", "op": "score", "rows": 65536, "width": 12, "top": 2, "scale": 4.0, "type": "f64"},
        # one sampling step: one row over the 2^17 outcomes of 17 qubits, with the alternatives shown to the user
        {"name": "score one row", "op": "score", "rows": 1, "width": 131072, "top": 20, "scale": 1.0, "type": "bf16"},
        # scoring a data set: many rows over a wide, odd number of outcomes
        {"name": "score many rows", "op": "score", "rows": 2048, "width": 100003, "top": 8, "scale": 1.0, "type": "bf16"},
        # a training step's loss on 12 outcomes, with an entropy bonus
        {"name": "loss 12 outcomes", "op": "loss", "rows": 65536, "width": 12, "scale": 4.0, "type": "f64"},
        # a training step's loss over a wide read-out
        {"name": "loss wide", "op": "loss", "rows": 4000, "width": 32001, "scale": 1.0, "type": "f32"},
        # the parameters of the 12-qubit depth-10 ansatz: 11 layers of 36 angles
        {"name": "orthogonalize 12 qubits", "op": "orthogonalize", "batch": 1, "rows": 11, "cols": 36, "type": "f64"},
        # 256 trials of the 20-qubit depth-8 ansatz at once
        {"name": "orthogonalize trials", "op": "orthogonalize", "batch": 256, "rows": 9, "cols": 60, "type": "f64"},
        # an ordinary matrix with odd sides, longer than wide
        {"name": "orthogonalize odd", "op": "orthogonalize", "batch": 1, "rows": 1000, "cols": 777, "type": "f32"},
        # the largest matrix
        {"name": "orthogonalize large", "op": "orthogonalize", "batch": 1, "rows": 4096, "cols": 4096, "type": "bf16"},
        # an optimizer step of the 12-qubit ansatz
        {"name": "muon 12 qubits", "op": "muon", "batch": 1, "rows": 11, "cols": 36, "type": "f64"},
        # an optimizer step of a wide layer: 16-bit gradients, 32-bit weights and momentum
        {"name": "muon wide", "op": "muon", "batch": 1, "rows": 1024, "cols": 4096, "type": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "loss", "orthogonalize", "muon"])
    if op in ("score", "loss"):
        kind = rng.choice(["f64", "f32", "bf16", "f16"])
        most = LARGEST_ROWS // {"f64": 4, "f32": 2}.get(kind, 1)
        width = _log_int(rng, 2, 262144)
        rows = _log_int(rng, 1, max(1, min(65536, most // width)))
        case = {"op": op, "rows": rows, "width": width, "scale": round(rng.uniform(0.5, 4.0), 2), "type": kind}
        if op == "score":
            case["top"] = rng.randint(0, min(32, width))
        return case
    kind = rng.choice(["f64", "f32", "bf16", "f16"])
    rows, cols = _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)
    if kind == "f64":  # products in 64 bits run at a small part of the rate
        rows, cols = min(rows, 1500), min(cols, 1500)
    room = LARGEST_PRODUCT // (rows * cols * min(rows, cols)) // 16
    batch = _log_int(rng, 1, max(1, min(256, room)))
    return {"op": op, "batch": batch, "rows": rows, "cols": cols, "type": kind}


def _logits(case, gen):
    """Scores as a model gives them: most outcomes in a broad middle, a few that stand out, every eleventh or so forbidden;
    the rows of a narrow read-out are expectation values in [-1, 1]."""
    r, v, t = case["rows"], case["width"], DTYPES[case["type"]]
    if v <= 64:
        return (2 * torch.rand(r, v, device="cuda", dtype=torch.float64, generator=gen) - 1).to(t)
    z = torch.randn(r, v, device="cuda", generator=gen).mul_(2.5)
    z[torch.rand(r, v, device="cuda", generator=gen) < 0.09] = -math.inf
    return z.to(t)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    if case["op"] in ("score", "loss"):
        r, v = case["rows"], case["width"]
        s["logits"] = _logits(case, gen)
        target = torch.randint(0, v, (r,), device="cuda", generator=gen, dtype=torch.int32)
        if r > 8:  # samples without a label
            target[torch.rand(r, device="cuda", generator=gen) < 0.05] = -1
        s["target"] = target
        if case["op"] == "loss":
            wide = torch.float64 if case["type"] == "f64" else torch.float32
            s["g"] = torch.full((r,), -1.0 / r, device="cuda", dtype=wide)
            s["h"] = -0.01 / r * torch.rand(r, device="cuda", dtype=wide, generator=gen)
        return s
    b, m, n, t = case["batch"], case["rows"], case["cols"], DTYPES[case["type"]]
    k = max(1, min(m, n) // 8)
    wide = torch.float64 if case["type"] == "f64" else torch.float32
    # a gradient: a few strong directions over a noisy floor
    left = torch.randn(b, m, k, device="cuda", dtype=wide, generator=gen)
    right = torch.randn(b, k, n, device="cuda", dtype=wide, generator=gen)
    g = (torch.matmul(left, right) / math.sqrt(k) + 0.5 * torch.randn(b, m, n, device="cuda", dtype=wide, generator=gen)) * 1e-2
    s["g"] = g.to(t)
    if case["op"] == "muon":
        s["w"] = torch.randn(b, m, n, device="cuda", dtype=wide, generator=gen)
        s["m"] = torch.randn(b, m, n, device="cuda", dtype=wide, generator=gen) * 1e-2
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------


def _row_parts(s):
    z = s["logits"]
    x = z.to(torch.float64 if z.dtype == torch.float64 else torch.float32) * s["scale"]
    d = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(dim=1, keepdim=True)
    ls = torch.log(total)
    terms = torch.where(e > 0, e * d, torch.zeros_like(d))
    entropy = (ls - terms.sum(dim=1, keepdim=True) / total)[:, 0]
    d -= ls
    t = s["target"].to(torch.int64)
    given = d.gather(1, t.clamp(min=0)[:, None])[:, 0]
    given = torch.where(t < 0, torch.zeros_like(given), given)
    return d, e, total, given, entropy, t


def _plain_score(s):
    lp, _, _, given, entropy, _ = _row_parts(s)
    k = s["top"]
    # a stable order gives equal values to the lowest index; it is taken on the values as they are stored
    index = torch.sort(s["logits"], dim=1, descending=True, stable=True)[1][:, :k]
    top = lp.gather(1, index)
    index = torch.where(torch.isinf(top), torch.full_like(index, -1), index)
    return {"log_prob": given, "entropy": entropy, "top_log_prob": top, "top_index": index.to(torch.int32)}


def _plain_loss(s):
    lp, e, total, given, entropy, t = _row_parts(s)
    p = e / total
    del e
    g = torch.where(t < 0, torch.zeros_like(s["g"]), s["g"])
    bonus = torch.where(p > 0, p * (lp + entropy[:, None]), torch.zeros_like(p))
    dz = -g[:, None] * p - s["h"][:, None] * bonus
    dz.scatter_add_(1, t.clamp(min=0)[:, None], g[:, None])
    return {"log_prob": given, "entropy": entropy, "d_logits": (dz * s["scale"]).to(s["logits"].dtype)}


def _newton_schulz(u):
    """In u's type; the shorter side first, so that the products stay small."""
    norm = torch.sqrt((u.double() * u.double()).sum(dim=(1, 2), keepdim=True)) + EPS
    x = (u.double() / norm).to(u.dtype)
    turned = x.shape[1] > x.shape[2]
    if turned:
        x = x.transpose(1, 2).contiguous()
    a, b, c = COEFS
    for _ in range(STEPS):
        y = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * y + c * torch.matmul(y, y), x)
    return x.transpose(1, 2).contiguous() if turned else x


def _plain_orthogonalize(s):
    g = s["g"]
    return _newton_schulz(g if g.dtype == torch.float64 else g.float()).to(g.dtype)


MUON = {"lr": 0.02, "mu": 0.95, "weight_decay": 0.01}


def _plain_muon(s):
    g, m, w = s["g"].to(s["m"].dtype), s["m"], s["w"]
    m.mul_(MUON["mu"]).add_(g)
    o = _newton_schulz(g + MUON["mu"] * m)
    rows, cols = w.shape[1:]
    w.mul_(1 - MUON["lr"] * MUON["weight_decay"]).sub_(o * (MUON["lr"] * math.sqrt(max(1.0, rows / cols))))
    return {"weight": w, "momentum": m}


def run(state):
    op = state["op"]
    if own:
        import vqa_amd

        if op == "score":
            r = vqa_amd.log_probs(state["logits"], state["target"], top_k=state["top"], scale=state["scale"])
            return {"log_prob": r.log_prob, "entropy": r.entropy, "top_log_prob": r.top_log_prob, "top_index": r.top_index}
        if op == "loss":
            r = vqa_amd.log_probs_grad(state["logits"], state["target"], state["g"], state["h"], scale=state["scale"])
            return {"log_prob": r.log_prob, "entropy": r.entropy, "d_logits": r.d_logits}
        if op == "orthogonalize":
            return vqa_amd.orthogonalize(state["g"], steps=STEPS, coefs=COEFS, eps=EPS)
        vqa_amd.muon_step(state["w"], state["g"], state["m"], steps=STEPS, coefs=COEFS, eps=EPS, nesterov=True, **MUON)
        return {"weight": state["w"], "momentum": state["m"]}
    if op == "score":
        return _plain_score(state)
    if op == "loss":
        return _plain_loss(state)
    return _plain_orthogonalize(state) if op == "orthogonalize" else _plain_muon(state)


def work(case):
    size = {"f64": 8, "f32": 4}.get(case["type"], 2)
    wide = 8 if case["type"] == "f64" else 4
    if case["op"] in ("score", "loss"):
        r, v = case["rows"], case["width"]
        if case["op"] == "score":
            return {"bytes": r * (v * size + 4 + 2 * wide + case["top"] * (wide + 4)), "flops": 6 * r * v}
        return {"bytes": r * (2 * v * size + 4 + 4 * wide), "flops": 12 * r * v}
    b, m, n = case["batch"], case["rows"], case["cols"]
    k, c = min(m, n), max(m, n)
    # the products with a symmetric result need only one half of it
    flops = b * STEPS * (k * k * c + k * k * k + 2 * k * k * c)
    if case["op"] == "orthogonalize":
        return {"bytes": 2 * b * m * n * size, "flops": flops}
    return {"bytes": b * m * n * (size + 4 * wide), "flops": flops + 6 * b * m * n}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------


def _exact_rows(s):
    """Row by row in blocks: log softmax from logsumexp, entropy as the mean of -log p under p."""
    z, scale, out = s["logits"], s["scale"], []
    step = max(1, 20_000_000 // z.shape[1])
    for lo in range(0, z.shape[0], step):
        x = z[lo:lo + step].double() * scale
        logp = x - torch.logsumexp(x, dim=1, keepdim=True)
        p = torch.exp(logp)
        entropy = -(torch.where(p > 0, logp, torch.zeros_like(p)) * p).sum(dim=1)
        t = s["target"][lo:lo + step].long()
        hit = torch.arange(z.shape[1], device=z.device)[None, :] == t[:, None]
        given = torch.where(hit, logp, torch.zeros_like(logp)).sum(dim=1)
        if s["op"] == "score":
            # the values of the top places do not depend on how ties are broken
            top = torch.topk(logp, s["top"], dim=1).values if s["top"] else logp[:, :0]
            out.append((given, entropy, top))
        else:
            g = torch.where(t < 0, torch.zeros_like(given), s["g"][lo:lo + step].double())
            h = s["h"][lo:lo + step].double()
            slope = torch.where(p > 0, -p * (logp + entropy[:, None]), torch.zeros_like(p))
            out.append((given, entropy, scale * (g[:, None] * (hit.double() - p) + h[:, None] * slope)))
    return [torch.cat(parts) for parts in zip(*out)]


def _exact_orthogonal(u):
    """By the definition on singular values where that is quick, else by products in another order: x (a + b y + c y y)
    with y on the side of x's columns or rows that is shorter."""
    u = u.double()
    m, n = u.shape[1:]
    x = u / (torch.linalg.vector_norm(u, dim=(1, 2), keepdim=True) + EPS)
    a, b, c = COEFS
    if u.shape[0] * min(m, n) <= 256:
        left, sv, right = torch.linalg.svd(x.cpu(), full_matrices=False)
        for _ in range(STEPS):
            sv = sv * (a + sv * sv * (b + c * sv * sv))
        return (left @ (sv[:, :, None] * right)).to(u.device)
    short = min(m, n)
    eye = torch.eye(short, dtype=torch.float64, device=u.device)[None]
    for _ in range(STEPS):
        xt = x.transpose(1, 2).contiguous()
        if m <= n:
            y = torch.matmul(x, xt)
            x = torch.matmul(a * eye + torch.matmul(y, b * eye + c * y), x)
        else:
            y = torch.matmul(xt, x)
            x = torch.matmul(x, a * eye + torch.matmul(y, b * eye + c * y))
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "score":
        given, entropy, top = _exact_rows(s)
        return {"log_prob": given, "entropy": entropy, "top_log_prob": top, "top_index": None}
    if case["op"] == "loss":
        given, entropy, dz = _exact_rows(s)
        return {"log_prob": given, "entropy": entropy, "d_logits": dz}
    if case["op"] == "orthogonalize":
        return _exact_orthogonal(s["g"])
    m = MUON["mu"] * s["m"].double() + s["g"].double()
    o = _exact_orthogonal(s["g"].double() + MUON["mu"] * m)
    rows, cols = case["rows"], case["cols"]
    w = s["w"].double() * (1 - MUON["lr"] * MUON["weight_decay"]) - MUON["lr"] * math.sqrt(max(1.0, rows / cols)) * o
    return {"weight": w, "momentum": m}
