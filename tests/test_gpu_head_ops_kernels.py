"""Every kernel of the dense heads at the work it is meant for: contractions of many tiles with a remainder, rows that fill a workgroup
several times over.  Which kernel a shape takes is asserted from a profile, so that a change of the rules cannot drop one from here
unnoticed.  Bounds: test_gpu_head_ops; the linear oracle is the same, in 64 bits, on the GPU (products of 3400^3)."""
import math
import re

import pytest
import torch

from pointnet2_ops import head_ops as ho
from test_gpu_head_ops import IDS, INF, NAN, TYPES, U, act64, check, half, rnd, run_distill, run_labels, tiny

pytestmark = pytest.mark.gpu
NAMES = {torch.float32: "HdF32", torch.bfloat16: "HdBF16", torch.float16: "HdF16"}


def launched(f):
    """The names of the heads' kernels that f() launches, without namespaces and arguments: la_tile_kernel<HdF16, false, ...>."""
    from torch.profiler import ProfilerActivity, profile
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        f()
        torch.cuda.synchronize()
    names = [e.name.replace("(anonymous namespace)::", "") for e in p.events()]
    return [m.group(1) for m in (re.match(r"void ((?:la|lp)_\w+<[^()]*>)", n) for n in names) if m]


def linear_exact(x, w, b, act, r, dy):
    """linear_case of test_gpu_head_ops, where the tensors are."""
    dt, (M, K), N = x.dtype, x.shape, w.size(0)
    x, w, dy = x.double(), w.double(), dy.double()
    z, size = x @ w.t().contiguous(), x.abs() @ w.abs().t().contiguous()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    ez = (K + 4) * U * size
    y, d = act64(z, act)
    ey = 1.2 * ez + (0 if act in ("none", "relu") else 8 * U * (1 + z.abs()))
    if r is not None:
        y, ey = y + r.double(), ey + 2 * U * (y.abs() + r.double().abs())
    ey = ey + half(dt) * (y.abs() + ey) + tiny(dt)
    ed = torch.zeros_like(z) if act == "none" else ((z.abs() <= ez).double() if act == "relu" else
                                                   1.2 * ez + 16 * U * (1 + z.abs()) + (U * d.abs() if dt == torch.float32 else 2.0 ** -15 + 2 * U * d.abs()))
    dz = dy * d
    edz0 = dy.abs() * ed + U * dz.abs()
    edz = edz0 + (0 if act == "none" else half(dt) * (dz.abs() + edz0) + tiny(dt))
    adz = dz.abs() + edz
    edx = edz @ w.abs() + (N + 4) * U * (adz @ w.abs())
    edw = edz.t().contiguous() @ x.abs() + (M + 4) * U * (adz.t().contiguous() @ x.abs())
    edb = edz0.sum(0) + (M + 4) * U * adz.sum(0)
    out = lambda v, e: (v, e + half(dt) * (v.abs() + e) + tiny(dt))
    return dict(y=(y, ey), dx=out(dz @ w, edx), dw=out(dz.t().contiguous() @ x, edw), db=out(dz.sum(0), edb))


# M, N, K; the tile of the forward product, of dx and of dW: (waves, fragments) of both directions.  Remainders in every contraction, and
# the second of each pair with operands that are copied
BIG = {torch.float32: "2, 2, 4, 4", torch.bfloat16: "2, 4, 8, 4", torch.float16: "2, 4, 8, 4"}
LAYERS = [((3401, 3336, 3368), None), ((3401, 3337, 3371), None), ((2100, 2104, 1096), "2, 2, 4, 2"), ((2100, 2105, 1101), "2, 2, 4, 2")]


def layer(shape, dtype, act, seed):
    M, N, K = shape
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s, scale=1.0: (torch.randn(*s, generator=gen, device="cuda") * scale).to(dtype)
    return new(M, K), new(N, K, scale=K ** -0.5), new(N, scale=0.3), new(M, N) if seed % 2 else None, new(M, N)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape,tile", LAYERS, ids=["x".join(map(str, s)) for s, _ in LAYERS])
def test_layers_take_the_kernels_that_are_tested_below(shape, tile, dtype):
    x, w, b, r, dy = layer(shape, dtype, "gelu", 0)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    names = launched(lambda: torch.autograd.grad(ho.linear_act(*leaves, "gelu"), leaves, dy))
    tile = tile or BIG[dtype]
    act = ho.ACTIVATIONS.index("gelu")
    assert [n for n in names if n.startswith("la_tile")] == [f"la_tile_kernel<{NAMES[dtype]}, {p}, {q}, {tile}, {a}>" for p, q, a in
                                                             (("false", "false", act), ("false", "true", 0), ("true", "true", 0))], names
    assert any(n.startswith("la_pad") for n in names) == (shape[2] % 4 != 0)


@pytest.mark.parametrize("act", ho.ACTIVATIONS)
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [s for s, _ in LAYERS], ids=lambda s: "x".join(map(str, s)))
def test_linear_act_on_its_largest_tiles(shape, dtype, act):
    x, w, b, r, dy = layer(shape, dtype, act, ho.ACTIVATIONS.index(act) + len(shape))
    want = linear_exact(x, w, b, act, r, dy)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def run():
        y = ho.linear_act(*leaves, act, r)
        return dict(zip(("y", "dx", "dw", "db"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))
    got = run()
    for k, v in got.items():
        value, tol = want[k]
        off = (v.double() - value).abs() - tol
        bad = ~(off <= 0)
        assert not bad.any(), (k, int(bad.sum()), bad.nonzero()[:4].tolist(), v[bad][:4].tolist(), value[bad][:4].tolist(), tol[bad][:4].tolist())
    again = run()
    assert all(torch.equal(got[k], again[k]) for k in got)


# ------------------------------------------------------------------------------------------------ rows of several hundred workgroups
# V, threads of a workgroup by type: more than 256 rows, up to 4096 vectors of 16 bytes or more
ROWS = [(9001, 256, 256), (40003, 512, 512), (17001, 512, 256)]


def rows_of(V, dtype, T=280):
    """Random rows with the hard ones among them, and their labels."""
    low = torch.finfo(dtype).min
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(T, V, generator=gen) * 3
    x[1] = -INF
    x[2] = -INF
    x[2, V - 2] = 1.5
    x[3] = low
    x[4] = low
    x[4, V // 3:V // 3 + 9] = torch.linspace(-1, 1, 9)
    x[5] = 0.25
    x[6] = torch.linspace(-4, 4, V)
    x[7] = torch.linspace(4, -4, V)
    x[8] = 0
    x[8, ::8] = 7.0
    x[9, V - 1] = NAN
    x[10, 5] = INF
    x[11, torch.rand(V, generator=gen) < 0.9] = -INF
    per = 128 // torch.finfo(dtype).bits                             # the best entries in the vectors of one thread, and its neighbour's
    for row, threads in ((12, 256), (13, 512)):
        share = (torch.arange(0, V, threads * per)[:, None] + torch.arange(per)).flatten()
        x[row] = 0
        x[row, share[share < V]] = 2.0 + torch.arange(int((share < V).sum())) % 5
        x[row + 2] = 0
        x[row + 2, (share + 3 * per) % V] = 1.0
        x[row + 2, share[share < V]] = 1.0
    x[16] = 0
    x[16, -50:] = 3.0
    y = torch.randint(V, (T,), generator=gen)
    y[20], y[21], y[22] = -100, V, -7
    y[2] = V - 2
    return x.to(dtype).cuda(), y.cuda()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V,f32,f16", ROWS)
def test_many_long_rows_take_the_kernels_that_are_tested_below(V, f32, f16, dtype):
    x, y = rows_of(V, dtype)
    threads = f32 if dtype == torch.float32 else f16
    index, value = torch.zeros(280, 3, dtype=torch.int64, device="cuda"), torch.zeros(280, 3, device="cuda")
    for call, mode, top in ((lambda: ho.label_log_probs(x, y), 0, "false"), (lambda: ho.label_log_probs(x, y, top=20), 0, "true"),
                            (lambda: ho.distill_top_k(x, index, value), 1, "false")):
        assert launched(call) == [f"lp_row_kernel<{NAMES[dtype]}, {mode}, {top}, {threads}, 4, false>"]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [v for v, _, _ in ROWS])
def test_label_log_probs_of_many_long_rows(V, dtype):
    x, y = rows_of(V, dtype)
    for top in (0, 5, 64):
        run_labels(x, y, top, seed=top)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [v for v, _, _ in ROWS])
def test_distill_top_k_of_many_long_rows(V, dtype):
    x, _ = rows_of(V, dtype)
    x[[3, 4, 9, 10]] = x[[30, 31, 32, 33]]                           # (its oracle takes rows of ordinary logits)
    gen = torch.Generator().manual_seed(V + 1)
    index = torch.randint(V, (280, 70), generator=gen).cuda()         # indices repeat within a row
    index[11] = x[11].argmax()
    index[2] = V - 2
    index[5, 3:], index[6] = -1, -1
    value = rnd(gen, 280, 70, scale=2.0)
    value[7, ::2] = -INF
    run_distill(x, index, value, 1.5)


# ---------------------------------------------------------------------------------- rows around the length from which they are segments
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T,V,segments", [(1, 65536, False), (2, 65537, True), (64, 65544, True), (65, 65544, False), (3, 70001, True), (2, 100003, True)])
def test_rows_around_the_length_of_segments(T, V, segments, dtype):
    gen = torch.Generator().manual_seed(V + T)
    x = rnd(gen, T, V, scale=3.0, dtype=dtype)
    x[T // 2, torch.rand(V, generator=gen).cuda() < 0.6] = -INF
    y = torch.randint(V, (T,), generator=gen).cuda()
    y[T // 2] = x[T // 2].argmax()
    y[-1], x[-1, V - 1] = V - 1, 9.0                                  # the row's last entry, in a partial vector or a segment of its own
    joined = [n.startswith("lp_join") for n in launched(lambda: ho.label_log_probs(x, y, top=3))]
    assert joined == ([False, True] if segments else [False])
    for top in (0, 20) if T < 10 else (20,):
        run_labels(x, y, top, seed=top)
    index = torch.randint(V, (T, 30), generator=gen).cuda()
    index[T // 2], index[-1] = y[T // 2], V - 1
    run_distill(x, index, rnd(gen, T, 30, scale=2.0), 1.5)
