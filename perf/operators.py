"""The dense-head operators (pointnet2_ops.head_ops) as measured work: cases, inputs, plain forms, exact values.

``own`` False: elementary torch operations in 32 bits.  ``own`` True: the calls a user's program makes.

linear     y = act(x W^T + b) [+ residual];    train: also dx, dW, db, d residual for a given dy
labels     log probability of given labels, entropy of each row, top alternatives;  train: also d logits
distill    KL divergence of a teacher's top logits from the student's softmax, per row;  train: also d logits
"""
import math
import os
import sys

import torch

# the package lies one folder below the repository's root, under a name that is no Python identifier
sys.path.insert(1, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "4d-or_amd"))

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_INV_SQRT2 = 0.7071067811865476
_INV_SQRT_2PI = 0.3989422804014327


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the relation head's first layer on one scan: 9 objects give 72 ordered pairs, 256 features -> 512, ReLU, training
        dict(name="linear_scan", op="linear", m=72, k=256, n=512, type="f32", act="relu", bias=True, residual=False, train=True),
        # one token through a square layer of a served network: bound by reading the weight
        dict(name="linear_token", op="linear", m=1, k=4096, n=4096, type="bf16", act="silu", bias=True, residual=True, train=False),
        # odd sizes in every direction, 16-bit training
        dict(name="linear_odd", op="linear", m=1003, k=1001, n=777, type="f16", act="gelu_tanh", bias=True, residual=True, train=True),
        # a batch of clouds' pooled features, exact fp32 (the framework's default type), inference
        dict(name="linear_rows", op="linear", m=8192, k=2048, n=2048, type="f32", act="relu", bias=True, residual=True, train=False),
        # the wide layer of a feed-forward block on a full training batch
        dict(name="linear_wide", op="linear", m=16384, k=2048, n=8192, type="bf16", act="gelu", bias=True, residual=False, train=True),
        # the relations of one scan: 15 predicates, the three best of each pair
        dict(name="labels_scan", op="labels", t=72, v=15, type="f32", top=3, masked=0.0, train=False),
        # one decoded token: log probability and twenty alternatives, a tenth of the vocabulary masked
        dict(name="labels_token", op="labels", t=1, v=131072, type="bf16", top=20, masked=0.1, train=False),
        # policy-gradient training: log probability and entropy with their gradient, an odd vocabulary
        dict(name="labels_train", op="labels", t=4096, v=32003, type="bf16", top=0, masked=0.0, train=True),
        # scoring a long batch over a large vocabulary
        dict(name="labels_score", op="labels", t=8192, v=131072, type="bf16", top=20, masked=0.0, train=False),
        # the relations of one scan learned from a teacher's five best predicates
        dict(name="distill_scan", op="distill", t=72, v=15, k=5, type="f32", temperature=2.0, train=True),
        # the loss alone (validation), half precision, an odd vocabulary
        dict(name="distill_valid", op="distill", t=1021, v=50021, k=32, type="f16", temperature=1.0, train=False),
        # a training batch over a large vocabulary
        dict(name="distill_train", op="distill", t=8192, v=131072, k=64, type="bf16", temperature=2.0, train=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("linear", "labels", "distill"))
    kind = rng.choice(("f32", "bf16", "f16"))
    train = rng.random() < 0.5
    if op == "linear":
        m, k, n = _log_int(rng, 1, 16384), _log_int(rng, 32, 8192), _log_int(rng, 32, 8192)
        if rng.random() < 0.5:                                   # half of the layers have the round sizes of real ones
            k, n = (k + 31) // 32 * 32, (n + 31) // 32 * 32
        most = 2 ** 35 if kind == "f32" else 2 ** 38             # products; fp32 multiplies at a sixteenth of the 16-bit rate
        while m * k * n > most:
            m = (m + 1) // 2
        acts = ["none", "gelu", "gelu_tanh", "silu"]
        if not train or m * n <= 2 ** 18:
            # a pre-activation within its own rounding of zero has slope 0 or 1 by chance: a few in 2^24 of them
            acts.append("relu")
        return dict(op=op, m=m, k=k, n=n, type=kind, act=rng.choice(acts),
                    bias=rng.random() < 0.8, residual=rng.random() < 0.5, train=train)
    t, v = _log_int(rng, 1, 8192), _log_int(rng, 2, 131072)
    while t * v * (2 if kind == "f32" else 1) > 2 ** 30:
        t = (t + 1) // 2
    if op == "labels":
        return dict(op=op, t=t, v=v, type=kind, top=min(v, rng.choice((0, 1, 3, 5, 20, 64))),
                    masked=rng.choice((0.0, 0.1, 0.9)), train=train)
    return dict(op=op, t=t, v=v, k=min(v, _log_int(rng, 1, 64)), type=kind, temperature=rng.choice((1.0, 2.0, 0.7)), train=train)


# ----------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale)

    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return dict(case=case, x=normal(m, k).to(dtype), weight=normal(n, k, scale=k ** -0.5).to(dtype),
                    bias=normal(n, scale=0.1).to(dtype) if case["bias"] else None,
                    residual=normal(m, n).to(dtype) if case["residual"] else None,
                    dy=normal(m, n).to(dtype) if case["train"] else None)
    t, v = case["t"], case["v"]
    logits = torch.empty(t, v, dtype=dtype, device="cuda")
    rows = max(1, 2 ** 27 // v)                                  # logits of a trained network: a broad background and a few peaks
    for r in range(0, t, rows):
        part = normal(min(rows, t - r), v, scale=2.0)
        if case.get("masked"):
            part.masked_fill_(torch.rand(part.shape, generator=gen, device="cuda") < case["masked"], -math.inf)
        peaks = torch.randint(v, (part.size(0), 4), generator=gen, device="cuda")
        part.scatter_reduce_(1, peaks, normal(part.size(0), 4, scale=3.0).add_(6.0), "amax")
        logits[r:r + rows] = part.to(dtype)
    if case["op"] == "labels":
        best = logits.argmax(1)
        anywhere = torch.randint(v, (t,), generator=gen, device="cuda")
        take = torch.rand(t, generator=gen, device="cuda") < 0.7
        return dict(case=case, logits=logits, labels=torch.where(take, best, anywhere),
                    d_log_prob=normal(t) if case["train"] else None, d_entropy=normal(t, scale=0.01) if case["train"] else None)
    # the teacher's best entries: distinct indices, some of them the student's own best, with falling logits
    k = case["k"]
    first = torch.randint(v, (t, 1), generator=gen, device="cuda")
    step = torch.randint(1, max(2, (v - 1) // k + 1), (t, 1), generator=gen, device="cuda") if v > 1 else first * 0
    index = (first + step * torch.arange(k, device="cuda")) % v
    values = normal(t, k, scale=2.0).sort(1, descending=True)[0].to(dtype)
    return dict(case=case, logits=logits, index=index, values=values, d_loss=torch.full((t,), 1.0 / t, device="cuda"))


# ------------------------------------------------------------------------------------------------------- plain forms
def _act_and_slope(z, act):
    if act == "none":
        return z, None
    if act == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * _INV_SQRT2))
        return z * cdf, cdf + z * (_INV_SQRT_2PI * torch.exp(-0.5 * z * z))
    c = 0.7978845608028654
    u = c * (z + 0.044715 * z ** 3)
    t = torch.tanh(u)
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    case, x, w = s["case"], s["x"], s["weight"]
    kind = x.dtype
    x32, w32 = x.float(), w.float()
    z = x32 @ w32.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, slope = _act_and_slope(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y.to(kind)
    if not case["train"]:
        return y
    dz = s["dy"].float()
    if slope is not None:
        dz = dz * slope
    out = dict(y=y, dx=(dz @ w32).to(kind), dw=(dz.t() @ x32).to(kind))
    if s["bias"] is not None:
        out["db"] = dz.sum(0).to(kind)
    if s["residual"] is not None:
        out["dr"] = s["dy"]
    return out


def _plain_labels(s):
    case, logits, labels = s["case"], s["logits"], s["labels"]
    x = logits.float()
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    log_prob = x.gather(1, labels[:, None])[:, 0] - lse[:, 0]
    # masked entries have probability zero and add nothing
    entropy = lse[:, 0] - torch.where(e > 0, e * x, 0.0).sum(1) / total[:, 0]
    out = dict(log_prob=log_prob, entropy=entropy)
    if case["top"]:
        # one whole number per entry: the logit's rank above, the index below (reversed), so equal logits go by their index
        bits = logits.float().add(0.0).view(torch.int32).long()
        rank = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        v = x.size(1)
        index = torch.arange(v, device=x.device)
        best = torch.topk(rank * v + (v - 1 - index), case["top"], dim=1)[0]
        index = v - 1 - best.remainder(v)
        value = x.gather(1, index) - lse
        out.update(top_log_prob=value, top_index=torch.where(value > -math.inf, index, -1))
    if case["train"]:
        p = e / total
        g, h = s["d_log_prob"][:, None], s["d_entropy"][:, None]
        grad = -p * (g + torch.where(e > 0, h * (x - lse + entropy[:, None]), 0.0))
        grad.scatter_add_(1, labels[:, None], g)
        out["d_logits"] = grad.to(logits.dtype)
    return out


def _plain_distill(s):
    case, logits, index = s["case"], s["logits"], s["index"]
    tau = case["temperature"]
    x = logits.float() / tau
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    t = s["values"].float() / tau
    t = t - t.amax(1, keepdim=True)
    log_q = t - torch.log(torch.exp(t).sum(1, keepdim=True))
    q = torch.exp(log_q)
    loss = tau * tau * (q * (log_q - (x.gather(1, index) - torch.log(total)))).sum(1)
    if not case["train"]:
        return loss
    g = s["d_loss"][:, None] * tau
    grad = (e / total) * g
    grad.scatter_add_(1, index, -q * g)
    return dict(loss=loss, d_logits=grad.to(logits.dtype))


# ------------------------------------------------------------------------------------------------- the user's calls
def _own_linear(s):
    from pointnet2_ops import head_ops
    case = s["case"]
    if not case["train"]:
        return head_ops.linear_act(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"])
    leaves = {name: s[name].detach().requires_grad_() for name in ("x", "weight", "bias", "residual") if s[name] is not None}
    y = head_ops.linear_act(leaves["x"], leaves["weight"], leaves.get("bias"), activation=case["act"],
                            residual=leaves.get("residual"))
    grads = torch.autograd.grad(y, list(leaves.values()), s["dy"])
    names = {"x": "dx", "weight": "dw", "bias": "db", "residual": "dr"}
    return dict(y=y.detach(), **{names[name]: g for name, g in zip(leaves, grads)})


def _own_labels(s):
    from pointnet2_ops import head_ops
    case = s["case"]
    if not case["train"]:
        r = head_ops.label_log_probs(s["logits"], s["labels"], top=case["top"])
    else:
        logits = s["logits"].detach().requires_grad_()
        r = head_ops.label_log_probs(logits, s["labels"], top=case["top"])
    out = dict(log_prob=r.log_prob.detach(), entropy=r.entropy.detach())
    if case["top"]:
        out.update(top_log_prob=r.top_log_prob, top_index=r.top_index)
    if case["train"]:
        out["d_logits"], = torch.autograd.grad((r.log_prob, r.entropy), logits, (s["d_log_prob"], s["d_entropy"]))
    return out


def _own_distill(s):
    from pointnet2_ops import head_ops
    case = s["case"]
    if not case["train"]:
        return head_ops.distill_top_k(s["logits"], s["index"], s["values"], temperature=case["temperature"])
    logits = s["logits"].detach().requires_grad_()
    loss = head_ops.distill_top_k(logits, s["index"], s["values"], temperature=case["temperature"])
    grad, = torch.autograd.grad(loss, logits, s["d_loss"])
    return dict(loss=loss.detach(), d_logits=grad)


_PLAIN = {"linear": _plain_linear, "labels": _plain_labels, "distill": _plain_distill}
_OWN = {"linear": _own_linear, "labels": _own_labels, "distill": _own_distill}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# -------------------------------------------------------------------------------------------------------- the floor
def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        read = m * k + n * k + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        write = m * n
        if case["train"]:
            read += m * n
            write += m * k + n * k + (n if case["bias"] else 0)
        return {"bytes": (read + write) * size, "flops": (6 if case["train"] else 2) * m * k * n}
    t, v = case["t"], case["v"]
    entries = t * v * size * (2 if case["train"] else 1)
    if case["op"] == "labels":
        # label in, two statistics out, (log probability, index) of each alternative out, two gradients in
        return {"bytes": entries + t * (8 + 8 + 12 * case["top"] + (8 if case["train"] else 0)),
                "flops": t * v * (10 if case["train"] else 5)}
    return {"bytes": entries + t * (case["k"] * (8 + size) + 4 + (4 if case["train"] else 0)),
            "flops": t * v * (8 if case["train"] else 4)}


# ------------------------------------------------------------------------------------------------------ exact values
def _exact_linear(s, case):
    f64 = {name: None if s[name] is None else s[name].double() for name in ("x", "weight", "bias", "residual", "dy")}
    z = torch.matmul(f64["x"], f64["weight"].t().contiguous())
    if f64["bias"] is not None:
        z += f64["bias"]
    act = case["act"]
    if act == "none":
        y, slope = z.clone(), torch.ones_like(z)
    elif act == "relu":
        y, slope = torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).double()
    elif act == "silu":
        y = z / (1 + torch.exp(-z))
        slope = (1 + torch.exp(-z) * (1 + z)) / (1 + torch.exp(-z)) ** 2
    elif act == "gelu":
        half_erfc = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        y = z * half_erfc
        slope = half_erfc + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    else:
        # (1 + tanh u) / 2 = 1 / (1 + e^(-2u))
        two_u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z.pow(3))
        gate = torch.sigmoid(two_u)
        y = z * gate
        slope = gate + z * gate * (1 - gate) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z.square())
    if f64["residual"] is not None:
        y += f64["residual"]
    if not case["train"]:
        return y
    dz = f64["dy"] * slope
    out = dict(y=y, dx=torch.matmul(dz, f64["weight"]), dw=torch.matmul(dz.t().contiguous(), f64["x"]))
    if f64["bias"] is not None:
        out["db"] = dz.sum(0)
    if f64["residual"] is not None:
        out["dr"] = f64["dy"]
    return out


def _exact_rows(s, case, lo, hi):
    """Rows lo..hi of a labels or distill case in 64 bits."""
    x = s["logits"][lo:hi].double()
    rows = torch.arange(x.size(0), device=x.device)
    if case["op"] == "labels":
        log_p = x - torch.logsumexp(x, 1, keepdim=True)
        p = log_p.exp()
        plogp = torch.where(p > 0, p * log_p, 0.0)
        label = s["labels"][lo:hi]
        out = dict(log_prob=log_p[rows, label], entropy=-plogp.sum(1))
        if case["top"]:
            value, index = torch.sort(x, dim=1, descending=True, stable=True)
            value, index = value[:, :case["top"]], index[:, :case["top"]]
            out["top_log_prob"] = log_p.gather(1, index)
            out["top_index"] = index.masked_fill(value == -math.inf, -1)
        if case["train"]:
            g, h = s["d_log_prob"][lo:hi, None].double(), s["d_entropy"][lo:hi, None].double()
            # d log p_y / d x = [v = y] - p ;  d H / d x = -p (log p + H)
            grad = -g * p - h * (plogp + p * out["entropy"][:, None])
            grad[rows, label] += g[:, 0]
            out["d_logits"] = grad
        return out
    tau = case["temperature"]
    log_p = torch.log_softmax(x / tau, 1)
    log_q = torch.log_softmax(s["values"][lo:hi].double() / tau, 1)
    index = s["index"][lo:hi]
    out = dict(loss=tau * tau * (log_q.exp() * (log_q - log_p.gather(1, index))).sum(1))
    if case["train"]:
        target = torch.zeros_like(x).scatter_add_(1, index, log_q.exp())
        out["d_logits"] = s["d_loss"][lo:hi, None].double() * tau * (log_p.exp() - target)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(s, case)
    rows = max(1, 2 ** 26 // case["v"])
    parts = [_exact_rows(s, case, lo, min(case["t"], lo + rows)) for lo in range(0, case["t"], rows)]
    out = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
    if case["op"] == "distill" and not case["train"]:
        return out["loss"]
    return out
