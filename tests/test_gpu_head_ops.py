"""Dense-head operators on the GPU against plain implementations in 64 bits.

Tolerances are error bounds, elementwise, from the arithmetic the kernels document (u = 2^-24, half a step of the output type
h = eps / 2): an fp32 sum of K products is off by at most (K + 4) u sum |x w| in any order; a stored slope by u, or, in 16-bit fixed
point of step 2^-14, by 2^-15 plus the conversion's own fp32 rounding (2 u);
dz by its own rounding; exponentials and logarithms by a few u of their argument's size (written at `_row_bounds`)."""
import math

import pytest
import torch

from pointnet2_ops import _ext, head_ops as ho

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
NAN, INF = float("nan"), float("inf")


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rnd(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()


def check(got, want, tol, what=""):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64).cpu().expand_as(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs() - tol)
    bad = ~(off <= 0)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist(),
                           tol[bad][:4].tolist())


# ------------------------------------------------------------------------------------------------------------ linear
def act64(z, name):
    """(act, slope) in 64 bits."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    a = math.sqrt(2 / math.pi)
    t = torch.tanh(a * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)


def linear_case(x, w, b, act, r, dy):
    """Exact outputs and their bounds, all in 64 bits on the CPU."""
    dt = x.dtype
    x, w, dy = (t.detach().double().cpu() for t in (x, w, dy))
    b = None if b is None else b.detach().double().cpu()
    r = None if r is None else r.detach().double().cpu()
    K, N, M = x.size(1), w.size(0), x.size(0)
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b, size + b.abs()
    ez = (K + 4) * U * size
    y, d = act64(z, act)
    # |act'| <= 1.2; the activation itself is evaluated to 8 u (1 + |z|) (erf, exp, rcp: a few ulp each)
    ey = 1.2 * ez + (0 if act in ("none", "relu") else 8 * U * (1 + z.abs()))
    if r is not None:
        y, ey = y + r, ey + 2 * U * (y.abs() + r.abs())
    ey = ey + half(dt) * (y.abs() + ey) + tiny(dt)
    # |act''| <= 1.2; relu's slope is either within ez of zero
    ed = torch.zeros_like(z) if act == "none" else ((z.abs() <= ez).double() if act == "relu" else
                                                   1.2 * ez + 16 * U * (1 + z.abs()) + (U * d.abs() if dt == torch.float32 else 2.0 ** -15 + 2 * U * d.abs()))
    dz = dy * d
    edz0 = dy.abs() * ed + U * dz.abs()
    edz = edz0 + (0 if act == "none" else half(dt) * (dz.abs() + edz0) + tiny(dt))
    adz = dz.abs() + edz
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    edx = edz @ w.abs() + (N + 4) * U * (adz @ w.abs())
    edw = edz.t() @ x.abs() + (M + 4) * U * (adz.t() @ x.abs())
    edb = edz0.sum(0) + (M + 4) * U * adz.sum(0)
    out = lambda v, e, t=dt: (v, e + half(t) * (v.abs() + e) + tiny(t))
    return dict(y=(y, ey), dx=out(dx, edx), dw=out(dw, edw), db=(db, edb))


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps      # spacing of the subnormals


SHAPES = [(1, 1, 1), (1, 17, 5), (3, 7, 9), (72, 512, 256), (1, 300, 1001), (130, 65, 33), (64, 64, 64), (257, 129, 2048), (5, 1, 700),
          (1003, 77, 101), (16, 4096, 128), (33, 520, 4104), (300, 264, 72), (256, 256, 32), (512, 776, 328), (640, 1304, 4104), (1032, 136, 1000), (2100, 520, 264),
          # one of every kernel and rule: few columns, 128 x 64 and 128 x 128 (fp32) / 256 x 256 (16-bit) tiles, padded copies, split sums
          (128, 1000, 300), (5000, 20, 100), (2100, 1032, 264), (8200, 1030, 40), (4100, 2900, 72), (1003, 777, 1001), (640, 1301, 4099),
          (20000, 40, 33), (7, 3000, 20000)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_linear_act_forward_and_gradients(shape, dtype):
    M, N, K = shape
    n = SHAPES.index(shape)
    act = ho.ACTIVATIONS[n % 5]
    gen = torch.Generator().manual_seed(n)
    x, w = rnd(gen, M, K, dtype=dtype), rnd(gen, N, K, scale=K ** -0.5, dtype=dtype)
    b = None if n % 4 == 1 else rnd(gen, N, scale=0.3, dtype=torch.float32 if n % 2 else dtype)
    r = rnd(gen, M, N, dtype=dtype) if n % 3 else None
    dy = rnd(gen, M, N, dtype=dtype)
    want = linear_case(x, w, b, act, r, dy)
    leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
    y = ho.linear_act(x, w, b, act, r)
    assert y.dtype == dtype
    check(y, *want["y"], what="y")
    grads = dict(zip([k for k, t in zip(("dx", "dw", "db", "dr"), (x, w, b, r)) if t is not None],
                     torch.autograd.grad(y, leaves, dy)))
    check(grads["dx"], *want["dx"], what="dx")
    check(grads["dw"], *want["dw"], what="dw")
    if b is not None:
        v, e = want["db"]
        assert grads["db"].dtype == b.dtype
        check(grads["db"], v, e + half(b.dtype) * (v.abs() + e) + tiny(b.dtype), what="db")
    if r is not None:
        assert torch.equal(grads["dr"], dy)
    # without a graph the same kernel runs; two runs agree bit for bit
    with torch.no_grad():
        assert torch.equal(ho.linear_act(x, w, b, act, r), y)
    for a, c in zip(torch.autograd.grad(ho.linear_act(x, w, b, act, r), leaves, dy), grads.values()):
        assert torch.equal(a, c)


@pytest.mark.parametrize("act", ho.ACTIVATIONS)
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_act_strides_alignment_and_leading_axes(act, dtype):
    gen = torch.Generator().manual_seed(5)
    big = rnd(gen, 2, 41, 130, dtype=dtype)
    x = big[..., 3:64]                                       # rows at odd starts, row stride 130
    w = rnd(gen, 61, 96, scale=0.2, dtype=dtype).t()         # transposed: (96, 61)
    r = rnd(gen, 41, 1, dtype=dtype)                         # broadcast over scans and columns
    b = rnd(gen, 200, dtype=dtype)[7:103]
    dy = rnd(gen, 2, 41, 96, dtype=dtype)
    xl, wl, rl = (t.detach().requires_grad_() for t in (x, w, r))
    y = ho.linear_act(xl, wl, b, act, rl)
    assert y.shape == (2, 41, 96)
    want = linear_case(x.reshape(82, 61), w, b, act, r.expand(2, 41, 96).reshape(82, 96), dy.reshape(82, 96))
    check(y.reshape(82, 96), *want["y"], what="y")
    dx, dw, dr = torch.autograd.grad(y, (xl, wl, rl), dy)
    check(dx.reshape(82, 61), *want["dx"], what="dx")
    check(dw, *want["dw"], what="dw")
    full = dy.double().cpu()
    check(dr, full.sum((0, 2))[:, None], (192 * 2 * half(dtype)) * full.abs().sum((0, 2))[:, None], what="dr")   # torch's sum, steps of dtype
    # a gradient that arrives expanded (y.sum()), a vector, an empty batch
    g, = torch.autograd.grad(ho.linear_act(xl, w, b, act).sum(), xl)
    want = linear_case(x.reshape(82, 61), w, b, act, None, torch.ones(82, 96, dtype=dtype))
    check(g.reshape(82, 61), *want["dx"], what="dx of sum")
    v = ho.linear_act(x[0, 0], w, b, act)
    assert v.shape == (96,)
    check(v, want["y"][0][0], want["y"][1][0], what="vector")
    e = x[:, :0].detach().requires_grad_()
    out = ho.linear_act(e, wl, b, act)
    assert out.shape == (2, 0, 96)
    gx, gw = torch.autograd.grad(out, (e, wl), torch.zeros_like(out))
    assert gx.shape == e.shape and not gw.any()


def test_linear_act_infinities_nan_and_frozen_inputs():
    x = torch.zeros(4, 40, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(48, 40, device="cuda", dtype=torch.bfloat16)
    x[1, 39], x[2, 3], x[3, 0] = INF, NAN, -INF
    for act in ("none", "relu"):
        y = ho.linear_act(x, w, activation=act)
        assert not y[0].any() and (y[1] == INF).all() and y[2].isnan().all()
        assert (y[3] == (-INF if act == "none" else 0)).all()
    # only what needs a gradient is computed; nothing else is held
    b = torch.zeros(48, device="cuda", requires_grad=True)
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        y = ho.linear_act(x[:1], w, b, "relu")
    assert [t.dtype for t in held] == [torch.int16]
    y.sum().backward()
    assert b.grad.shape == (48,)
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(ho.linear_act(x[:1].float(), w.float(), b, "silu").sum(), b, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_linear_act_gradient_against_differences(act):
    """L(x) = sum(y dy) along a direction v: (L(x + e v) - L(x - e v)) / 2e.  Off by e^2 / 6 |L'''| (|act'''| <= 3 for these; e v w <=
    e |v w|) and by the forward's own rounding over e."""
    gen = torch.Generator().manual_seed(2)
    x, w, dy, v = rnd(gen, 20, 64), rnd(gen, 48, 64, scale=0.125), rnd(gen, 20, 48), rnd(gen, 20, 64)
    e = 2.0 ** -6
    x1, x2 = x + e * v, x - e * v
    loss = lambda t: (ho.linear_act(t, w, None, act).double() * dy.double()).sum()
    xl = x.clone().requires_grad_()
    g, = torch.autograd.grad(ho.linear_act(xl, w, None, act), xl, dy)
    step = (x1.double() - x2.double()) / 2                                   # the step that was taken, exactly
    zw = (step @ w.double().t()).abs()
    round_off = ((64 + 16) * U * (x1.abs().double() @ w.abs().double().t() + 1) * dy.double().abs()).sum() * 2 / (2 * e)
    cut = (3 * zw ** 3 / 6 * dy.double().abs()).sum() / e
    got = (g.double() * step).sum() / e
    assert abs(float(got - (loss(x1) - loss(x2)) / (2 * e))) <= float(round_off + cut)


# ------------------------------------------------------------------------------------------------------------ labels
def _row_bounds(x, c=1.0):
    """Exact (log p, p, H) of rows and a bound on the log-sum-exp and entropy of the kernels.
    A term 2^t has argument error 2 u (1 + |t|) (one FMA, the rounded log2 e) and 1 ulp of its own; weighted by p, sum p |t| <= H' =
    (H + log s) / ln 2 + 1.  Summation: at most V / 512 + 32 additions deep, each u.  log2 and the last subtractions: 4 u of their size."""
    x = x.double().cpu() * c
    lp = torch.log_softmax(x, 1)
    p = lp.exp()
    H = -torch.where(p > 0, p * lp, 0.0).sum(1)
    V = x.size(1)
    big = H / math.log(2) + math.log2(V) + 1
    e_lse = U * (V / 512 + 40 + 4 * big + 4 * big)
    e_H = U * (V / 512 + 48 + 8 * big) * (1 + big) * 2
    return lp, p, H, e_lse, e_H


def label_case(x, y, top, ignore=-100, g=None, h=None):
    dt = x.dtype
    xd = x.detach().double().cpu()
    lp, p, H, e_lse, e_H = _row_bounds(xd)
    empty = (xd == -INF).all(1)
    nan = (xd.isnan() | (xd == INF)).any(1)
    T, V = xd.shape
    e_lp = lambda l, e: e + 4 * U * torch.where(l.isfinite(), l.abs(), 0.0)
    yc = y.cpu()
    inside = (yc >= 0) & (yc < V)
    lab = torch.where(inside, lp[torch.arange(T), yc.clamp(0, V - 1)], NAN)
    lab = torch.where(empty & inside, -INF, lab)
    lab = torch.where(nan & inside, NAN, lab)
    lab = torch.where(yc == ignore, 0.0, lab)
    ent = torch.where(empty, 0.0, torch.where(nan, NAN, H))
    out = dict(log_prob=(lab, e_lp(lab, e_lse)), entropy=(ent, e_H))
    if top:
        val, idx = torch.sort(xd, dim=1, descending=True, stable=True)
        idx = idx[:, :top].masked_fill((val[:, :top] == -INF) | nan[:, None], -1)
        tl = lp.gather(1, idx.clamp_min(0)).masked_fill(idx < 0, -INF)
        tl = tl.masked_fill(nan[:, None], NAN)
        out["top_index"] = idx
        # (lowest - highest passes the range of fp32, the outputs' type: the nearest fp32 value of -6.8e38 is -inf)
        tl = torch.where(tl < -2.0 ** 128, -INF, tl)
        out["top_log_prob"] = (tl, e_lp(tl, e_lse[:, None]))
    if g is not None:
        g, h = g.detach().double().cpu()[:, None], h.detach().double().cpu()[:, None]
        skip = (yc == ignore)[:, None]
        g = torch.where(skip, 0.0, g)
        plp = torch.where(p > 0, p * (lp + H[:, None]), 0.0)
        d = -g * p - h * plp
        on = torch.zeros_like(xd).scatter_(1, yc.clamp(0, V - 1)[:, None], 1.0)
        d = d + g * on * inside[:, None] * ~skip
        d = torch.where(empty[:, None], 0.0, d)
        fin = torch.where(lp.isfinite(), lp.abs(), 0.0)
        rel = e_lse[:, None] + 8 * U * (2 + fin)                              # of p
        e = p * rel * (g.abs() + h.abs() * (fin + H[:, None])) + p * h.abs() * (e_H[:, None] + e_lse[:, None] + 8 * U * fin) + 4 * U * d.abs()
        dead = (g == 0) & (h == 0)
        d = torch.where(dead, 0.0, torch.where(nan[:, None] | (~inside[:, None] & ~skip), NAN, d))
        out["d_logits"] = (d, e + half(dt) * (d.abs() + e) + tiny(dt))
    return out


def run_labels(x, y, top, ignore=-100, grads=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    T = x.size(0)
    g, h = rnd(gen, T), rnd(gen, T, scale=0.3)
    want = label_case(x, y, top, ignore, g, h)
    leaf = x.detach().requires_grad_()
    r = ho.label_log_probs(leaf, y, top=top, ignore_index=ignore)
    check(r.log_prob, *want["log_prob"], what="log_prob")
    check(r.entropy, *want["entropy"], what="entropy")
    if top:
        assert torch.equal(r.top_index.cpu(), want["top_index"])
        check(r.top_log_prob, *want["top_log_prob"], what="top")
        assert not r.top_index.requires_grad and not r.top_log_prob.requires_grad
    else:
        assert r.top_index is None and r.top_log_prob is None
    if grads:
        d, = torch.autograd.grad((r.log_prob, r.entropy), leaf, (g, h))
        assert d.dtype == x.dtype
        check(d, *want["d_logits"], what="d_logits")
    return r


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [1, 2, 15, 63, 64, 65, 200, 256, 257, 1000, 1024, 1025, 4096, 4099, 16384 + 5, 32003, 70001])
def test_label_log_probs(V, dtype):
    gen = torch.Generator().manual_seed(V)
    T = 5
    x = rnd(gen, T, V, scale=3.0, dtype=dtype)
    x[1, torch.rand(V, generator=gen).cuda() < 0.6] = -INF
    y = torch.randint(V, (T,), generator=gen).cuda()
    y[4] = -100
    for top in sorted({0, 1, min(V, 7), min(V, 64)}):
        run_labels(x, y, top, seed=top)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [40, 600, 5000, 40000])
def test_label_log_probs_hard_rows(V, dtype):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    gen = torch.Generator().manual_seed(V)
    rows, labels = [], []

    def add(r, y=0):
        rows.append(r)
        labels.append(y)
    add(torch.full((V,), -INF))                                     # nothing left
    one = torch.full((V,), -INF); one[V - 2] = 1.5
    add(one, V - 2)                                                 # one entry left
    add(one.clone(), 3)                                             # ... and the label masked
    add(torch.full((V,), low), V - 1)                               # the lowest value everywhere: uniform
    m = torch.full((V,), low); m[V // 3:V // 3 + 9] = torch.linspace(-1, 1, 9)
    add(m, V // 3 + 2)                                              # masked by the lowest value
    add(torch.full((V,), 0.25), 1)                                  # all equal: the first indices win
    add(torch.linspace(-4, 4, V), V - 1)                            # ascending
    add(torch.linspace(4, -4, V), 0)
    t = torch.zeros(V); t[::8] = 7.0
    add(t, 8)                                                       # ties in every vector
    s = torch.randn(V, generator=gen); s[torch.arange(0, V, 512 * 8) % V] = 9.0
    add(s, 2)
    z = torch.zeros(V); z[1::2] = -0.0
    add(z, 5)                                                       # +0 and -0 are equal
    add(torch.full((V,), high), 7)
    h = torch.randn(V, generator=gen); h[11] = high
    add(h, 11)
    nanrow = torch.randn(V, generator=gen); nanrow[V - 1] = NAN
    add(nanrow)
    infrow = torch.randn(V, generator=gen); infrow[5] = INF
    add(infrow, 5)
    infrow2 = torch.full((V,), -INF); infrow2[V - 1] = INF
    add(infrow2, 0)
    add(torch.full((V,), NAN))
    add(torch.randn(V, generator=gen), V)                           # labels outside
    add(torch.randn(V, generator=gen), -7)
    add(torch.randn(V, generator=gen), -100)                        # ignored
    mix = torch.full((V,), low); mix[0] = high
    add(mix, 0)
    x = torch.stack(rows).to(dtype).cuda()
    y = torch.tensor(labels).cuda()
    for top in (0, 5, 40):
        run_labels(x, y, top, seed=top)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [130, 3000])
def test_label_log_probs_best_entries_in_one_share(V, dtype):
    """The best entries all in vectors that one thread reads, in vectors of two threads, and at the row's end."""
    per = 128 // torch.finfo(dtype).bits                            # elements of 16 bytes
    V = V * per
    x = torch.zeros(3, V)
    share = (torch.arange(0, V, 512 * per)[:, None] + torch.arange(per)).flatten()
    share = share[share < V]
    x[0, share] = 2.0 + torch.arange(share.numel()) % 5
    x[1, (share + 3 * per) % V] = 1.0
    x[1, share] = 1.0
    x[2, -50:] = 3.0
    run_labels(x.to(dtype).cuda(), torch.tensor([0, 1, V - 1]).cuda(), 40)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_label_log_probs_strides_and_shapes(dtype):
    gen = torch.Generator().manual_seed(8)
    for V in (300, 2000):
        big = rnd(gen, 6, V + 77, dtype=dtype)
        y = torch.randint(V, (6,), generator=gen).cuda()
        run_labels(big[:, 5:5 + V], y, 3)                           # unaligned rows of another stride
        run_labels(big[2:3, :V].expand(6, V), y, 3)                 # row stride 0
        x = big[:, :V].reshape(2, 3, V)
        r = ho.label_log_probs(x, y.reshape(2, 3), top=4)
        s = ho.label_log_probs(big[:, :V], y, top=4)
        assert r.log_prob.shape == (2, 3) and r.top_index.shape == (2, 3, 4)
        assert torch.equal(r.entropy.flatten(), s.entropy) and torch.equal(r.top_index.reshape(6, 4), s.top_index)
        c = big[:, :V].t().contiguous().t()                         # columns first: copied
        assert torch.equal(ho.label_log_probs(c, y).log_prob, s.log_prob)
        one = ho.label_log_probs(big[0, :V], y[0])
        assert one.log_prob.shape == () and torch.equal(one.log_prob, s.log_prob[0])
        none = ho.label_log_probs(big[:0, :V].detach().requires_grad_(), y[:0], top=2)
        assert none.log_prob.shape == (0,) and none.top_index.shape == (0, 2)
        # one of the two gradients alone; labels that are a strided view
        leaf = big[:, :V].detach().requires_grad_()
        lab = torch.stack([y, y], 1)[:, 0]
        ga, = torch.autograd.grad(ho.label_log_probs(leaf, lab).log_prob.sum(), leaf)
        gb, = torch.autograd.grad(ho.label_log_probs(leaf, lab).entropy.sum(), leaf)
        one, nil = torch.ones(6), torch.zeros(6)
        check(ga, *label_case(big[:, :V], y, 0, g=one, h=nil)["d_logits"], what="log_prob alone")
        check(gb, *label_case(big[:, :V], y, 0, g=nil, h=one)["d_logits"], what="entropy alone")


# ----------------------------------------------------------------------------------------------------------- distill
def distill_case(x, idx, val, tau, g):
    dt = x.dtype
    xd, vd, ix = x.detach().double().cpu(), val.detach().double().cpu(), idx.cpu()
    lp, p, H, e_lse, _ = _row_bounds(xd, 1 / tau)
    T, V = xd.shape
    used = (ix >= 0) & (vd != -INF)
    some = used.any(1)
    lq = torch.log_softmax(torch.where(used, vd, -INF) / tau, 1)
    q = torch.where(used, lq.exp(), 0.0)
    lpi = lp.gather(1, ix.clamp(0, V - 1))
    empty = (xd == -INF).all(1)
    lpi = torch.where(empty[:, None], -INF, lpi)
    term = torch.where(q > 0, q * (lq - lpi), 0.0)
    loss = torch.where(some, tau * tau * term.sum(1), 0.0)
    fin = torch.where(lpi.isfinite(), lpi.abs(), 0.0) + torch.where(lq.isfinite(), lq.abs(), 0.0)
    k = ix.size(1)
    # q: its exponent's argument and its own normalisation; the terms add up k deep
    rq = U * (k + 16 + 4 * fin)
    e = tau * tau * ((q * (e_lse[:, None] + 8 * U * fin)).sum(1) + (q * rq * fin).sum(1) + (k + 8) * U * (q * fin).sum(1))
    out = dict(loss=(loss, torch.where(some, e, 0.0)))
    gt = g.detach().double().cpu()[:, None] * tau
    d = p - torch.zeros_like(p).scatter_add_(1, ix.clamp(0, V - 1), q)
    ed = p * (e_lse[:, None] + 8 * U * (2 + torch.where(lp.isfinite(), lp.abs(), 0.0)))
    ed = ed + torch.zeros_like(p).scatter_add_(1, ix.clamp(0, V - 1), q * rq)
    d, ed = torch.where((some & ~empty)[:, None], gt * d, 0.0), (gt.abs() * (ed + 2 * U * d.abs()))
    out["d_logits"] = (d, ed + half(dt) * (d.abs() + ed) + tiny(dt))
    return out


def run_distill(x, idx, val, tau, seed=0):
    gen = torch.Generator().manual_seed(seed)
    g = rnd(gen, x.size(0))
    want = distill_case(x, idx, val, tau, g)
    with torch.no_grad():
        check(ho.distill_top_k(x, idx, val, tau), *want["loss"], what="loss")
    leaf = x.detach().requires_grad_()
    loss = ho.distill_top_k(leaf, idx, val, tau)
    d, = torch.autograd.grad(loss, leaf, g)
    check(loss, *want["loss"], what="loss")
    check(d, *want["d_logits"], what="d_logits")
    return loss, d


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V,k", [(1, 1), (2, 2), (15, 5), (64, 64), (300, 7), (1025, 64), (4099, 1), (32003, 33), (70001, 100)])
def test_distill_top_k(V, k, dtype):
    gen = torch.Generator().manual_seed(V)
    T = 5
    x = rnd(gen, T, V, scale=3.0, dtype=dtype)
    idx = torch.stack([torch.randperm(V, generator=gen)[:min(k, V)] for _ in range(T)]).cuda()
    val = rnd(gen, T, idx.size(1), scale=2.0, dtype=TYPES[V % 3])
    for tau in (1.0, 2.5, 0.5):
        run_distill(x, idx, val, tau)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [40, 5000])
def test_distill_top_k_unused_slots_repeats_and_masks(V, dtype):
    gen = torch.Generator().manual_seed(V)
    T, k = 8, 70
    x = rnd(gen, T, V, dtype=dtype)
    idx = torch.randint(V, (T, k), generator=gen).cuda()            # indices repeat within a row
    val = rnd(gen, T, k, scale=2.0)
    idx[0, 3:] = -1                                                 # unused slots by index, by value, both, all
    val[1, ::2] = -INF
    idx[2, :5], val[2, 4:9] = -5, -INF
    idx[3] = -1
    val[4] = -INF
    idx[5] = 7                                                      # one index only: q = 1 there
    x[6] = -INF                                                     # a student row without an entry
    x[7, V // 2:] = -INF                                            # entries masked for the student (loss +inf where the teacher has one)
    idx[7] = idx[7] % (V // 2)
    loss, d = run_distill(x, idx, val, 1.5)
    assert loss[3] == 0 and loss[4] == 0 and not d[3].any() and not d[4].any()
    assert loss[6] == INF and not d[6].any()
    idx[7, 0] = V - 1
    loss, d = run_distill(x, idx, val, 1.5)
    assert loss[7] == INF and d[7].isfinite().all()
    # an index outside [0, V): the row says so, its neighbours do not
    idx[1, 1] = V
    leaf = x.detach().requires_grad_()
    bad = ho.distill_top_k(leaf, idx, val, 1.5)
    d2, = torch.autograd.grad(bad, leaf, torch.ones_like(bad))
    assert bad[1].isnan() and d2[1].isnan().all() and bad[0].isfinite() and d2[0].isfinite().all()
    # leading axes, strided index and values, an empty batch
    two = ho.distill_top_k(x.reshape(2, 4, V), idx.reshape(2, 4, k), val.reshape(2, 4, k), 1.5)
    assert two.shape == (2, 4) and torch.equal(two.flatten().nan_to_num(), bad.detach().nan_to_num())
    assert torch.equal(ho.distill_top_k(x, idx[:, ::2], val[:, ::2], 1.5).nan_to_num(),
                       ho.distill_top_k(x, idx[:, ::2].contiguous(), val[:, ::2].contiguous(), 1.5).nan_to_num())
    assert ho.distill_top_k(x[:0], idx[:0], val[:0]).shape == (0,)


# few long rows: in segments, joined by a second launch
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [131072, 131077, 270001, 600011])
def test_few_long_rows(V, dtype):
    gen = torch.Generator().manual_seed(V)
    x = rnd(gen, 3, V, scale=3.0, dtype=dtype)
    x[1, torch.rand(V, generator=gen).cuda() < 0.6] = -INF
    x[2, :V - 40000] = -INF                                         # whole segments without an entry
    y = torch.tensor([V - 1, 3, V - 7]).cuda()
    for top in (0, 1, 20, 64):
        run_labels(x, y, top, seed=top)
    idx = torch.randint(V, (3, 64), generator=gen).cuda()
    idx[2] = V - 1 - torch.arange(64).cuda()
    idx[1, :60] = -1
    x[1, idx[1, 60:]] = 1.0
    run_distill(x, idx, rnd(gen, 3, 64, scale=2.0), 1.5)
    # a row alone, and out of a wider matrix
    a, b = ho.label_log_probs(x[1:2], y[1:2], top=20), ho.label_log_probs(x, y, top=20)
    assert all(torch.equal(p[0], q[1]) for p, q in zip(a, b))
    wide = torch.full((3, V + 3), 50.0, device="cuda", dtype=dtype)
    wide[:, 1:V + 1] = x
    c = ho.label_log_probs(wide[:, 1:V + 1], y, top=20)
    assert all(torch.equal(p, q) for p, q in zip(b, c))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [131077, 262144 + 5])
def test_few_long_hard_rows(V, dtype):
    test_label_log_probs_hard_rows(V, dtype)
    test_distill_top_k_unused_slots_repeats_and_masks(V, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_few_long_rows_best_entries_in_one_share(dtype):
    """Every thread's share of the segments in turn holds the best entries: those of one thread, neighbours', the row's ends."""
    per = 128 // torch.finfo(dtype).bits
    V = 16384 * per + 3
    x = torch.zeros(4, V)
    share = (torch.arange(0, 1024 * per, 256 * per)[:, None] + torch.arange(per)).flatten()
    x[0, share] = 2.0 + torch.arange(share.numel()) % 5
    x[1, share + 7 * 1024 * per] = 1.0
    x[1, share + 7 * 1024 * per + 3 * per] = 1.0
    x[2, -50:] = 3.0
    x[3, ::1024] = 4.0
    run_labels(x.to(dtype).cuda(), torch.tensor([0, 1, V - 1, 1024]).cuda(), 40)


def test_few_long_rows_in_two_graphs_and_on_two_streams():
    """Segments' workspaces belong to their call: two captured graphs replayed in turn with eager work between, two streams at once."""
    gen = torch.Generator().manual_seed(9)
    V = 140001
    x, y = rnd(gen, 2, V, dtype=torch.bfloat16), torch.tensor([5, V - 1]).cuda()
    idx, val = torch.randint(V, (2, 20), generator=gen).cuda(), rnd(gen, 2, 20)

    def step():
        r = ho.label_log_probs(x, y, top=20)
        return [*r, ho.distill_top_k(x, idx, val)]
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for n in range(4):
        x.copy_(rnd(torch.Generator().manual_seed(70 + n), 2, V, dtype=torch.bfloat16))
        g, out = graphs[n % 2]
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, e) for a, e in zip(got, step()))
    want = step()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        both = []
        for s in streams:
            with torch.cuda.stream(s):
                both.append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for out in both for a, b in zip(out, want))


def test_gradients_against_differences():
    """Directional derivatives of the row statistics in fp32: cut-off e^2 / 6 times a third derivative bounded by 6 |v|^3 for the
    log-sum-exp (twice that times 1 + log V for the entropy), rounding of the two forward values over e."""
    gen = torch.Generator().manual_seed(3)
    T, V, e = 6, 1500, 2.0 ** -5
    x, v = rnd(gen, T, V, scale=2.0), torch.sign(rnd(gen, T, V))
    y = torch.randint(V, (T,), generator=gen).cuda()
    idx, val = torch.randint(V, (T, 9), generator=gen).cuda(), rnd(gen, T, 9)
    x1, x2 = x + e * v, x - e * v
    step = (x1.double() - x2.double()) / 2
    for name, f, size in (("log_prob", lambda t: ho.label_log_probs(t, y).log_prob, 1), ("entropy", lambda t: ho.label_log_probs(t, y).entropy, 20),
                          ("loss", lambda t: ho.distill_top_k(t, idx, val, 2.0), 4)):
        leaf = x.clone().requires_grad_()
        d, = torch.autograd.grad(f(leaf).sum(), leaf)
        want = (f(x1).double() - f(x2).double()) / (2 * e)
        got = (d.double() * step).sum(1) / e
        tol = size * (e * e + (V / 512 + 200) * U * 20 / e)
        assert float((got - want).abs().max()) <= tol, name


# ------------------------------------------------------------------------------------------------- used as a program does
def _program(x, w1, b1, w2, b2, y, teacher):
    """One training step of a head: two layers, the label's log probability, the teacher's alternatives."""
    h = ho.linear_act(x, w1, b1, "gelu")
    logits = ho.linear_act(h, w2, b2)
    r = ho.label_log_probs(logits, y, top=3)
    loss = -r.log_prob.mean() - 0.01 * r.entropy.mean() + ho.distill_top_k(logits, teacher[0], teacher[1], 2.0).mean()
    return loss, r


def _program_inputs(gen, dtype, T=72, F=96, H=160, V=1200):
    x = rnd(gen, T, F, dtype=dtype)
    params = [rnd(gen, H, F, scale=F ** -0.5, dtype=dtype), rnd(gen, H, scale=0.1, dtype=dtype),
              rnd(gen, V, H, scale=H ** -0.5, dtype=dtype), rnd(gen, V, scale=0.1, dtype=dtype)]
    y = torch.randint(V, (T,), generator=gen).cuda()
    t = ho.label_log_probs(rnd(gen, T, V, scale=2.0, dtype=dtype), y, top=5)          # the teacher's own answer
    return x, params, y, (t.top_index, t.top_log_prob)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_a_head_trained_from_a_teacher(dtype):
    """The operators together, as a head uses them; values and gradients against torch in 64 bits.  The chain's tolerance: each of
    the five roundings of 16-bit tensors along a path (h, logits, d logits, dz, the result) is off by half a step of relative size,
    taken against the root mean square of the result."""
    gen = torch.Generator().manual_seed(4)
    x, params, y, teacher = _program_inputs(gen, dtype)
    leaves = [p.detach().requires_grad_() for p in params]
    loss, r = _program(x, *leaves, y, teacher)
    grads = torch.autograd.grad(loss, leaves)
    ref = [p.detach().double().requires_grad_() for p in params]
    h = torch.nn.functional.gelu(x.double() @ ref[0].t() + ref[1])
    logits = h @ ref[2].t() + ref[3]
    lp = torch.log_softmax(logits, 1)
    want = -lp.gather(1, y[:, None]).mean() + 0.01 * (lp.exp() * lp).sum(1).mean()
    q = torch.softmax(teacher[1].double() / 2, 1)
    l2 = torch.log_softmax(logits / 2, 1)
    want = want + 4 * (q * (q.log() - l2.gather(1, teacher[0]))).sum(1).mean()
    wg = torch.autograd.grad(want, ref)
    tol = 5 * max(half(dtype), 64 * U)
    assert abs(float((loss - want).detach())) <= tol * float(want.detach().abs())
    for g, e in zip(grads, wg):
        assert g.dtype == dtype
        rms = float(e.pow(2).mean().sqrt())
        assert float((g.double() - e).pow(2).mean().sqrt()) <= tol * rms
        assert float((g.double() - e).abs().max()) <= 8 * tol * max(rms, float(e.abs().max()) / 4)


def test_captured_step_replays_with_new_inputs():
    gen = torch.Generator().manual_seed(6)
    x, params, y, teacher = _program_inputs(gen, torch.bfloat16)

    def step():
        leaves = [p.detach().requires_grad_() for p in params]
        loss, r = _program(x, *leaves, y, teacher)
        return [loss.detach(), r.top_index, *torch.autograd.grad(loss, leaves)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(4):
        fresh, p2, y2, t2 = _program_inputs(torch.Generator().manual_seed(10 + n), torch.bfloat16)
        x.copy_(fresh), y.copy_(y2), teacher[0].copy_(t2[0]), teacher[1].copy_(t2[1])
        for a, b in zip(params, p2):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            # (mean() of the loss is torch's; everything else is bit-identical between eager and replay)
            assert torch.equal(a, b) if a.dtype != torch.float32 else torch.allclose(a, b, rtol=1e-6)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1003, 777, 1001), (300, 200, 9000), (4096, 96, 64)], ids=lambda s: "x".join(map(str, s)))
def test_captured_layer_with_copies_and_split_sums(shape, dtype):
    """Workspaces inside a graph: padded copies, dz, strips of db, partial sums; two graphs of the same layer replayed in turn."""
    M, N, K = shape
    gen = torch.Generator().manual_seed(M)
    x, w, dy = rnd(gen, M, K, dtype=dtype), rnd(gen, N, K, scale=K ** -0.5, dtype=dtype), rnd(gen, M, N, dtype=dtype)
    b = rnd(gen, N, dtype=dtype)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = ho.linear_act(*leaves, "gelu")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for n in range(4):
        x.copy_(rnd(torch.Generator().manual_seed(50 + n), M, K, dtype=dtype))
        dy.copy_(rnd(torch.Generator().manual_seed(60 + n), M, N, dtype=dtype))
        g, out = graphs[n % 2]
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, e) for a, e in zip(got, step()))


def test_two_streams_at_once_and_record_of_inputs():
    gen = torch.Generator().manual_seed(7)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    x1, x2 = rnd(gen, 64, 2048, dtype=torch.float16), rnd(gen, 64, 2048, dtype=torch.float16)
    w = rnd(gen, 96, 2048, scale=0.02, dtype=torch.float16)
    y = torch.randint(2048, (64,), generator=gen).cuda()
    w1 = [ho.linear_act(x, w, None, "silu") for x in (x1, x2)]
    l1 = [ho.label_log_probs(x, y, top=9) for x in (x1, x2)]
    torch.cuda.synchronize()
    got = {}
    for n in range(3):
        for s, i, x in ((a, 0, x1), (b, 1, x2)):
            with torch.cuda.stream(s):
                got[i] = (ho.linear_act(x, w, None, "silu"), ho.label_log_probs(x, y, top=9))
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(got[i][0], w1[i])
            assert all(torch.equal(p, q) for p, q in zip(got[i][1], l1[i]))


def test_rows_past_two_to_the_32_elements():
    """Row offsets that pass 32 bits: 140 000 rows at a stride of 32 768 elements (9.2 GB), first, middle and last rows looked at."""
    T, V = 140000, 32768
    x = torch.zeros(T, V, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 65535, 65536, 131072, T - 1])
    gen = torch.Generator().manual_seed(9)
    x[rows.cuda()] = rnd(gen, 5, V, scale=2.0, dtype=torch.bfloat16)
    y = (torch.arange(T) % V).cuda()
    r = ho.label_log_probs(x, y, top=3)
    part = x[rows.cuda()]
    want = label_case(part, y[rows.cuda()], 3)
    check(r.log_prob[rows.cuda()], *want["log_prob"])
    assert torch.equal(r.top_index[rows.cuda()].cpu(), want["top_index"])
    assert float((r.entropy[1:1000] - math.log(V)).abs().max()) < 1e-5


def test_kernel_timer_records_the_heads_and_their_gradients(monkeypatch):
    """Under the timer every launch is one record with its bytes and operations; results stay what they are without it."""
    gen = torch.Generator().manual_seed(3)
    x, w = rnd(gen, 72, 256).requires_grad_(), rnd(gen, 15, 256).requires_grad_()
    y, best, val = torch.arange(72).cuda() % 15, torch.arange(72 * 5).view(72, 5).cuda() % 15, rnd(gen, 72, 5)

    def step():
        z = ho.linear_act(x, w)
        r = ho.label_log_probs(z, y, top=3)
        loss = ho.distill_top_k(z, best, val)
        return (r.log_prob, r.top_index, loss, *torch.autograd.grad(loss.sum() - r.log_prob.sum() - r.entropy.sum(), (x, w)))
    want = step()
    timer = _ext.KernelTimer(pool=16)
    monkeypatch.setattr(_ext, "TIMER", timer)
    got = step()
    monkeypatch.setattr(_ext, "TIMER", None)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    names = ["linear_act", "linear_act_grad", "label_logprobs", "label_logprobs_grad", "distill_topk", "distill_topk_grad"]
    rows = timer.summary()
    assert sorted(rows) == sorted("pn2_" + n for n in names) and all(r["calls"] == 1 and r["ms"] > 0 for r in rows.values())
    assert rows["pn2_linear_act"]["alg_flops"] * 2 == rows["pn2_linear_act_grad"]["alg_flops"] == 4 * 72 * 15 * 256
    assert rows["pn2_distill_topk"]["alg_bytes"] == 72 * 15 * 4


@pytest.mark.parametrize("frozen", range(16))
def test_linear_act_any_inputs_frozen(frozen):
    """Each set of inputs that need a gradient: the gradients of all of them up to the order of their sums (which kernels run depends
    on what is wanted), none for the others.  Both sides hold the same fp32 slopes and sum n <= 33 products of fp32: either is off by
    at most n + 2 roundings of sum |term|, and |silu'| < 1.1."""
    gen = torch.Generator().manual_seed(4)
    ts = [rnd(gen, 33, 40), rnd(gen, 24, 40), rnd(gen, 24), rnd(gen, 33, 24)]
    dy = rnd(gen, 33, 24)

    def grads(off):
        leaves = [t.clone().requires_grad_(not off >> i & 1) for i, t in enumerate(ts)]
        y = ho.linear_act(leaves[0], leaves[1], leaves[2], "silu", leaves[3])
        assert y.requires_grad == (off != 15)
        if y.requires_grad:
            y.backward(dy)
        return [t.grad for t in leaves]
    d = 1.1 * dy.abs()
    terms = [d @ ts[1].abs(), d.t() @ ts[0].abs(), d.sum(0), torch.zeros_like(dy)]
    for i, (a, b, t) in enumerate(zip(grads(0), grads(frozen), terms)):
        assert b is None if frozen >> i & 1 else bool(((a - b).abs() <= 2 * 35 * U * t).all())


@pytest.mark.parametrize("frozen", [1, 2, 3, 4, 5, 6])
@pytest.mark.parametrize("M,N,K", [(300, 136, 520), (2051, 72, 190), (4100, 264, 33)])
def test_linear_act_products_at_once_and_alone(M, N, K, frozen):
    """fp16 layers of the general route: with everything wanted dx, dW and db are one launch, otherwise each has its own.  The same dz
    and n products on both sides: sums off by n + 2 roundings of sum |term| each, results by one more rounding each."""
    gen = torch.Generator().manual_seed(7)
    ts = [rnd(gen, M, K, dtype=torch.float16), rnd(gen, N, K, scale=0.1, dtype=torch.float16), rnd(gen, N)]
    dy = rnd(gen, M, N, dtype=torch.float16)

    def grads(off):
        leaves = [t.clone().requires_grad_(not off >> i & 1) for i, t in enumerate(ts)]
        ho.linear_act(*leaves, "gelu").backward(dy)
        return [t.grad for t in leaves]
    d, x, w = 1.2 * dy.float().abs(), ts[0].float().abs(), ts[1].float().abs()
    terms = [((N + 2) * U, d @ w), ((M + 2) * U, d.t() @ x), ((M + 2) * U, d.sum(0))]
    for i, (a, b, (u, t)) in enumerate(zip(grads(0), grads(frozen), terms)):
        assert (b is None) == bool(frozen >> i & 1)
        if b is not None:
            tol = 2 * u * t + 2 * half(a.dtype) * (a.float().abs() + u * t) + tiny(a.dtype)
            assert bool(((a.float() - b.float()).abs() <= tol).all())


def test_views_with_the_negative_bit():
    gen = torch.Generator().manual_seed(8)
    z = torch.complex(rnd(gen, 9, 1), rnd(gen, 9, 1))
    x, w = z.conj().imag, rnd(gen, 5, 1)
    assert x.is_neg()
    assert torch.equal(ho.linear_act(x, w), ho.linear_act(x.clone().resolve_neg(), w))
    b = torch.complex(rnd(gen, 1), rnd(gen, 1)).conj().imag
    assert b.is_neg() and b.is_contiguous()
    want = ho.linear_act(w, w[:1], b.resolve_neg())
    assert torch.equal(ho.linear_act(w, w[:1], b), want)
    assert torch.equal(ho.linear_act(w.clone().requires_grad_(), w[:1], b), want)
    z = torch.complex(rnd(gen, 4, 6), rnd(gen, 4, 6))
    x, y, best = z.conj().imag, torch.arange(4).cuda(), torch.arange(8).view(4, 2).cuda()
    assert torch.equal(ho.label_log_probs(x, y).log_prob, ho.label_log_probs(-z.imag.contiguous(), y).log_prob)
    v = torch.complex(rnd(gen, 4, 2), rnd(gen, 4, 2))
    # (the last row's indices lie outside the columns: NaN on both sides)
    torch.testing.assert_close(ho.distill_top_k(x, best, v.conj().imag),
                               ho.distill_top_k(-z.imag.contiguous(), best, -v.imag.contiguous()), rtol=0, atol=0, equal_nan=True)


def test_each_operator_is_differentiable_once():
    gen = torch.Generator().manual_seed(6)
    x, w, r = (t.requires_grad_() for t in (rnd(gen, 4, 8), rnd(gen, 8, 8), rnd(gen, 4, 8)))
    y, best, val = torch.arange(4).cuda(), torch.arange(8).view(4, 2).cuda(), rnd(gen, 4, 2)
    for out, leaf in ((ho.linear_act(x, w, None, "gelu", r), x), (ho.linear_act(x, w, None, "none", r), r),
                      (ho.label_log_probs(x, y).log_prob, x), (ho.distill_top_k(x, best, val), x)):
        g, = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):
            g.sum().backward()


# ------------------------------------------------------------------------------------------------- the model's own paths
@pytest.mark.parametrize("train", [False, True])
def test_fused_heads_equal_the_library_heads(train, monkeypatch):
    """Both classification heads with the trunk's layers as linear_act: outputs and gradients of the library route within fp32
    rounding of a 512-term product per layer (three layers, gradients relative to their largest entry)."""
    from scene_graph_prediction.scene_graph_helpers.model.pointnets import network_PointNet as npn
    torch.manual_seed(0)
    obj = npn.PointNetCls(12, in_size=256, batch_norm=False, drop_out=True).cuda().train(train)
    rel = npn.PointNetRelCls(15, in_size=256, batch_norm=False, drop_out=True, n_object_types=6).cuda().train(train)
    x, e, hot = torch.randn(9, 256).cuda(), torch.randn(72, 256).cuda(), torch.zeros(72, 12).cuda()
    hot[torch.arange(72), torch.arange(72) % 12] = 1

    def run(fused):
        monkeypatch.setattr(npn._Head, "fused_linear", fused)
        torch.manual_seed(5)                                        # the same dropout masks
        xs, es = x.clone().requires_grad_(), e.clone().requires_grad_()
        a, b = obj(xs), rel(es, relation_objects_one_hot=hot)
        params = [*obj.parameters(), *rel.parameters()]
        return [a, b], torch.autograd.grad(a[:, 3].sum() + b[:, 5].sum(), [xs, es, *params])
    out, grads = run(False)
    out2, grads2 = run(True)
    for a, b in zip(out, out2):
        torch.testing.assert_close(a, b, atol=3 * 512 * U * float(a.abs().max()), rtol=0)
    for a, b in zip(grads, grads2):
        torch.testing.assert_close(a, b, atol=3 * 512 * U * float(a.abs().max()), rtol=0)


def test_fused_heads_leave_autocast_to_the_library(monkeypatch):
    from scene_graph_prediction.scene_graph_helpers.model.pointnets import network_PointNet as npn
    torch.manual_seed(0)
    head = npn.PointNetCls(12, in_size=256, batch_norm=False, drop_out=False).cuda().eval()
    x = torch.randn(9, 256).cuda().bfloat16()
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        want = head(x)
        monkeypatch.setattr(npn._Head, "fused_linear", True)
        assert torch.equal(head(x), want)


def test_model_alternatives_and_learning_from_a_teacher(tmp_path):
    import json
    from scene_graph_prediction import main as runner
    out = tmp_path / "rels.json"
    runner.main(["--mode", "infer", "--scans", "1", "--objects", "4", "--out", str(out), "--alternatives", "3"])
    rels = json.load(open(out))
    more = json.load(open(str(out) + ".alternatives.json"))
    assert rels.keys() == more.keys()
    (scan, edges), = more.items()
    assert len(edges) == 12
    best = {(a, b): alt for a, b, _, alt in edges}
    for a, b, entropy, alt in edges:
        assert len(alt) == 3 and 0 <= entropy <= math.log(15) + 1e-5
        assert all(p >= q for (_, p), (_, q) in zip(alt, alt[1:])) and sum(math.exp(p) for _, p in alt) <= 1 + 1e-5
    for sub, pred, ob in rels[scan]:
        assert best[(sub, ob)][0][0] == pred                        # the best alternative is predict_step's answer
    # a student's loss with a teacher's alternatives in its batch
    config = runner.config_loader("no_gt.json")
    torch.manual_seed(1)
    model = runner.SGPNModelWrapper(config, 12, 15, torch.ones(12), torch.ones(15), runner.RELATION_NAMES).cuda()
    gen = torch.Generator().manual_seed(2)
    rel_pred = torch.log_softmax(rnd(gen, 20, 15), 1).requires_grad_()
    obj_pred = torch.log_softmax(rnd(gen, 5, 12), 1)
    teacher = model.relation_alternatives(rnd(gen, 20, 15, scale=2.0), 5)
    batch = dict(gt_class=torch.zeros(5, dtype=torch.int64).cuda(), gt_rels=torch.zeros(20, dtype=torch.int64).cuda())
    plain = model.loss(obj_pred, rel_pred, batch)
    taught = model.loss(obj_pred, rel_pred, dict(batch, teacher_rels=(teacher.top_index, teacher.top_log_prob)))
    q = torch.softmax(teacher.top_log_prob.double(), 1)
    want = (q * (q.log() - torch.log_softmax(rel_pred.double(), 1).gather(1, teacher.top_index))).sum(1).mean()
    assert abs(float(taught - plain) - float(want)) <= 64 * U * (abs(float(want)) + abs(float(taught)))
    g, = torch.autograd.grad(taught - plain, rel_pred)
    wg, = torch.autograd.grad(want, rel_pred)
    torch.testing.assert_close(g.double(), wg.double(), atol=64 * U, rtol=64 * U)
