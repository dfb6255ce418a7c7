"""Dense-head operators where the documentation allows a call that small sizes do not reach: launches past 2^32 threads, NaN before
every activation, slots that are unused in two ways, the kernels of the largest tiles and rows.  Oracles and bounds: test_gpu_head_ops."""
import math

import pytest
import torch
import torch.utils.checkpoint

from pointnet2_ops import head_ops as ho

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------- more threads than 32 bits count
def test_label_rows_past_two_to_the_32_threads():
    """2^26 + 5 rows of two columns: 64 threads a row.  Every row by its formula; expm1 and log1p of the difference in fp32 are good
    to a few u, the kernels' sums of two terms to less than 16 u of 1 + |difference|."""
    T = 2 ** 26 + 5
    x = torch.zeros(T, 2, dtype=torch.bfloat16, device="cuda")
    x[:, 1] = (torch.arange(T, device="cuda") % 7).to(torch.bfloat16)
    y = torch.arange(T, device="cuda") % 2
    leaf = x.requires_grad_()
    r = ho.label_log_probs(leaf, y, top=1)
    d = x.detach()[:, 1].float()
    tol = 16 * 2.0 ** -24 * (1 + d)
    lse = d + torch.log1p(torch.exp(-d))
    assert bool(((r.log_prob - (torch.where(y == 1, d, 0.0) - lse)).abs() <= tol).all())
    assert torch.equal(r.top_index[:, 0], (d > 0).long())
    g, = torch.autograd.grad(r.log_prob, leaf, torch.ones(T, device="cuda"))
    p1 = torch.sigmoid(d)
    want = torch.where(y == 1, 1 - p1, -p1)                         # d log p_y / d x_1
    assert bool(((g[:, 1].float() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * tol).all())
    assert bool(((g[:, 0].float() + want).abs() <= 2.0 ** -8 * want.abs() + 4 * tol).all())


def test_distillation_rows_past_two_to_the_32_threads():
    """One entry of the teacher: q = 1, loss = -log p of it."""
    T = 2 ** 26 + 5
    x = torch.zeros(T, 2, dtype=torch.bfloat16, device="cuda")
    x[:, 1] = (torch.arange(T, device="cuda") % 7).to(torch.bfloat16)
    index, value = (torch.arange(T, device="cuda") % 2)[:, None], torch.zeros(T, 1, device="cuda")
    leaf = x.requires_grad_()
    loss = ho.distill_top_k(leaf, index, value)
    d = x.detach()[:, 1].float()
    tol = 16 * 2.0 ** -24 * (1 + d)
    on = index[:, 0] == 1
    assert bool(((loss - (d + torch.log1p(torch.exp(-d)) - torch.where(on, d, 0.0))).abs() <= tol).all())
    g, = torch.autograd.grad(loss, leaf, torch.ones(T, device="cuda"))
    p1 = torch.sigmoid(d)
    want = torch.where(on, p1 - 1, p1)
    assert bool(((g[:, 1].float() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * tol).all())


def test_long_label_rows_past_two_to_the_32_threads():
    """A workgroup per row: 2^24 + 3 rows that are one row of 2056 columns (row stride 0)."""
    T, V = 2 ** 24 + 3, 2056
    row = torch.randn(1, V, generator=torch.Generator().manual_seed(0)).to(torch.float16).cuda()
    y = torch.arange(T, device="cuda") % V
    r = ho.label_log_probs(row.expand(T, V), y)
    want = ho.label_log_probs(row.expand(V, V), torch.arange(V, device="cuda"))
    assert torch.equal(r.log_prob, want.log_prob[y]) and bool((r.entropy == want.entropy[0]).all())


def test_linear_rows_past_two_to_the_32_threads():
    """One column to one column: M results in M / 32 workgroups of the small kernel (products of small whole numbers: exact)."""
    M = 2 ** 29 + 37
    x = (torch.arange(M, device="cuda") % 5).to(torch.bfloat16)[:, None]
    y = ho.linear_act(x, torch.full((1, 1), 3.0, dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(y, x * 3)


def test_linear_gradient_rows_past_two_to_the_32_threads():
    """dx of 2^31 - 1 rows: M / 128 tiles of 256 threads."""
    M = 2 ** 31 - 1
    leaf = torch.zeros(1, 1, dtype=torch.bfloat16, device="cuda").expand(M, 1).requires_grad_()
    y = ho.linear_act(leaf, torch.full((1, 8), 3.0, dtype=torch.bfloat16, device="cuda")[:, :1])
    dy = torch.zeros(M, 8, dtype=torch.bfloat16, device="cuda")[:, :1]          # (rows at whole 16 bytes: no copies)
    dy[-200:, 0] = torch.arange(200, device="cuda").to(torch.bfloat16)
    dy[:200, 0] = 1.0
    dx, = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(dx[-200:], 3 * dy[-200:]) and bool((dx[:200] == 3).all()) and not dx[200:-200].any()


# -------------------------------------------------------------------------------------- what goes around torch's dispatcher
@pytest.mark.filterwarnings("ignore")
def test_forward_mode_and_recording_are_refused_and_onlookers_are_not():
    import torch.autograd.forward_ad as fwd
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn(6, 40, generator=gen).cuda(), torch.randn(9, 40, generator=gen).cuda()
    y, index, value = torch.arange(6).cuda(), torch.arange(12).view(6, 2).cuda() % 9, torch.randn(6, 2, generator=gen).cuda()
    calls = [lambda t: ho.linear_act(t, w, None, "silu"), lambda t: ho.label_log_probs(t, y, top=2).log_prob,
             lambda t: ho.distill_top_k(t, index, value)]
    for call in calls:
        with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call(fwd.make_dual(x, x))
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            torch.jit.trace(call, (x,))
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            make_fx(call)(x)
        with pytest.raises(RuntimeError, match="memory of its own"):
            torch.func.functionalize(call)(x)

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    def step(call):
        leaf = x.clone().requires_grad_()
        out = torch.utils.checkpoint.checkpoint(call, leaf, use_reentrant=False)
        return out, torch.autograd.grad(out.sum(), leaf)[0]
    for call in calls:
        want = step(call)
        with Watch():
            got = step(call)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert torch.equal(torch.compile(call, backend="eager")(x), want[0])      # (compiled around the call, not through it)


# ------------------------------------------------------------------------------------------- NaN and infinities before an activation
@pytest.mark.parametrize("act", ho.ACTIVATIONS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N", [(3, 8), (70, 130), (2100, 1040)], ids=["few", "small", "tiles"])
def test_linear_act_nan_reaches_every_gradient(M, N, dtype, act):
    """Row 2 of x is NaN in one place: y's row, d x's row through the slope and every entry of d bias are NaN; where the activation has
    no slope of its own at NaN (none: 1, relu: 1, as torch's) d x stays that of a slope of 1.  The other rows are untouched."""
    gen = torch.Generator().manual_seed(3)
    x, w = torch.randn(M, 40, generator=gen).to(dtype).cuda(), (torch.randn(N, 40, generator=gen) / 6).to(dtype).cuda()
    b, dy = torch.zeros(N, device="cuda", dtype=dtype), torch.randn(M, N, generator=gen).to(dtype).cuda()

    def run(x):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = ho.linear_act(*leaves, act)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    clean = run(x)
    x[2, 3] = float("nan")
    y, dx, dw, db = run(x)
    rest = torch.arange(M, device="cuda") != 2
    assert torch.equal(y[rest], clean[0][rest]) and torch.equal(dx[rest], clean[1][rest])
    assert y[2].isnan().all()
    if act in ("none", "relu"):
        assert dx[2].isfinite().all() and db.isfinite().all()
    else:
        assert dx[2].isnan().all() and db.isnan().all() and dw.isnan().all()
    assert dw[:, 3].isnan().all()                                   # d w = d z^T x: x itself is NaN there
    assert torch.equal(dw.isnan().all(1), torch.ones(N, dtype=torch.bool, device="cuda")) == (act not in ("none", "relu"))


@pytest.mark.parametrize("act", ho.ACTIVATIONS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_linear_act_far_and_infinite_arguments(act, dtype):
    """z from the bias: large finite values are exact (z or 0, slope 1 or 0), +inf stays +inf."""
    big = 3e4 if dtype == torch.float16 else 1e30
    b = torch.tensor([-big, -200.0, 200.0, big], device="cuda", dtype=dtype)
    x, w = torch.zeros(3, 16, device="cuda", dtype=dtype), torch.ones(4, 16, device="cuda", dtype=dtype)
    leaf = x.clone().requires_grad_()
    y = ho.linear_act(leaf, w, b, act)
    assert torch.equal(y, (b if act == "none" else b.clamp_min(0)).expand(3, 4))
    g, = torch.autograd.grad(y, leaf, torch.ones(3, 4, device="cuda", dtype=dtype))
    assert torch.equal(g, torch.full_like(g, 4.0 if act == "none" else 2.0))
    assert (ho.linear_act(x, w, b.new_full((4,), math.inf), act) == math.inf).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [15, 700, 5000, 140000])
def test_distillation_slots_unused_by_value_at_any_index(V, dtype):
    """A slot of value -inf is unused whatever its index, past the columns too: losses and gradients of the row without it."""
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(3, V, generator=gen).to(dtype).cuda()
    index = torch.tensor([[3, 7, V, V + 9, 2 ** 40], [V - 1, V, V, V, V], [V, V, V, V, V]]).cuda()
    value = torch.tensor([[0.5, -1.0] + [-math.inf] * 3, [2.0] + [-math.inf] * 4, [-math.inf] * 5]).cuda()
    as_padding = torch.where(value == -math.inf, -1, index)

    def run(index, value):
        leaf = x.clone().requires_grad_()
        loss = ho.distill_top_k(leaf, index, value, 1.5)
        return loss.detach(), torch.autograd.grad(loss, leaf, torch.ones(3, device="cuda"))[0]
    got, want = run(index, value), run(as_padding, value)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0].isfinite().all()
    # a used slot past the columns still says so
    bad = run(torch.where(index == V + 9, V, index), torch.where(index == V + 9, 0.0, value))
    assert bad[0][0].isnan() and bad[1][0].isnan().all() and torch.equal(bad[0][1:], want[0][1:])


# ------------------------------------------------------------------------------------------------- the heads' opt-in route
def _heads(monkeypatch, drop_out=False):
    """(head, library's answer, fused answer) for heads on 9 and 72 rows; the fused one under the class's switch."""
    from scene_graph_prediction.scene_graph_helpers.model.pointnets import network_PointNet as npn
    torch.manual_seed(0)
    head = npn.PointNetCls(12, in_size=256, batch_norm=False, drop_out=drop_out).cuda().eval()
    x = torch.randn(9, 256).cuda()

    def run(fused, x=x):
        monkeypatch.setattr(npn._Head, "fused_linear", fused)
        with torch.no_grad():
            return head(x)
    return head, x, run


def test_fused_heads_leave_fp32_inputs_under_autocast_to_the_library(monkeypatch):
    head, x, run = _heads(monkeypatch)
    exact = run(True)
    for dtype in (torch.bfloat16, torch.float16):
        with torch.autocast("cuda", dtype):
            assert torch.equal(run(True), run(False)) and not torch.equal(run(True), exact)
    assert torch.equal(run(True), exact)                              # (outside: the kernel again)


@pytest.mark.parametrize("how", ["hook", "pre-hook", "global hook", "weight_norm", "parametrised", "spectral_norm", "replaced", "own forward",
                                 "other activation", "float64"])
def test_fused_heads_leave_layers_that_are_more_than_a_product_to_torch(how, monkeypatch):
    """Whatever a program hung onto fc1, fc2 or their activation takes part on both routes: equal bit for bit, one route by then."""
    import torch.nn as nn
    head, x, run = _heads(monkeypatch)
    before, handle = run(True), None
    if how == "hook":
        head.fc2.register_forward_hook(lambda m, a, out: out * 2)
    elif how == "pre-hook":
        head.fc1.register_forward_pre_hook(lambda m, a: (a[0] + 1,))
    elif how == "global hook":
        handle = nn.modules.module.register_module_forward_hook(lambda m, a, out: out + 1 if m is head.fc1 else None)
    elif how == "weight_norm":
        nn.utils.weight_norm(head.fc1)
        head.fc1.weight_g.data.mul_(3)                                # (the hook forms the weight anew at the next call)
    elif how == "parametrised":
        class Twice(nn.Module):
            def forward(self, w):
                return 2 * w
        nn.utils.parametrize.register_parametrization(head.fc2, "weight", Twice())
    elif how == "spectral_norm":
        nn.utils.spectral_norm(head.fc2)
    elif how == "replaced":
        head.fc1 = nn.Sequential(nn.Linear(256, 256), nn.Linear(256, 512)).cuda()
    elif how == "own forward":
        head.fc1.forward = lambda t: nn.functional.linear(t, head.fc1.weight) * 2
    elif how == "other activation":
        head.relu = nn.Tanh()
    else:
        head.double()
        x = x.double()
    try:
        got = run(True, x)
        assert torch.equal(got, run(False, x))
        assert how == "float64" or not torch.allclose(got, before, atol=1e-4)
    finally:
        if handle is not None:
            handle.remove()


def test_alternatives_come_from_the_pass_that_made_the_triples(tmp_path, monkeypatch):
    """One forward pass per scan with --alternatives too, and the answers of the two methods on their own."""
    import json
    from scene_graph_prediction import main as runner
    calls, models = [], []
    forward = runner.SGPNModelWrapper.forward

    def counted(self, batch, **kw):
        calls.append(batch["scan_id"])
        models.append(self)
        return forward(self, batch, **kw)
    monkeypatch.setattr(runner.SGPNModelWrapper, "forward", counted)
    out = tmp_path / "rels.json"
    runner.main(["--mode", "infer", "--scans", "2", "--objects", "3", "--out", str(out), "--alternatives", "2"])
    assert calls == ["synthetic_000000", "synthetic_000001"]
    model = models[0]
    d = runner.config_loader("no_gt.json")["dataset"]
    rels, more = json.load(open(out)), json.load(open(str(out) + ".alternatives.json"))
    for i, name in enumerate(calls[:2]):
        batch = runner.to_device(runner.synthetic_scan(3, d["num_points_objects"], d["num_points_relation"], seed=i, scan_id=name), "cuda")
        with torch.no_grad():
            assert json.loads(json.dumps(model.predict_step(batch)[1])) == rels[name]
            assert json.loads(json.dumps(model.predict_alternatives(batch, 2)[1])) == more[name]


# ------------------------------------------------------------------------- captured backward passes and what is alive outside of them
CAPTURED = ["linear_act", "linear_act behind another node", "label_log_probs", "distill_top_k"]


def _captured_calls():
    gen = torch.Generator().manual_seed(5)
    x, w = torch.randn(30, 40, generator=gen).cuda(), torch.randn(20, 40, generator=gen).cuda()
    logits, y = torch.randn(30, 20, generator=gen).cuda(), torch.arange(30).cuda() % 20
    index, value = torch.arange(60).view(30, 2).cuda() % 20, torch.randn(30, 2, generator=gen).cuda()
    return {"linear_act": (w, lambda t: ho.linear_act(x, t, None, "silu")), "linear_act behind another node": (w, lambda t: ho.linear_act(x, t * 2)),
            "label_log_probs": (logits, lambda t: ho.label_log_probs(t, y, top=2).log_prob), "distill_top_k": (logits, lambda t: ho.distill_top_k(t, index, value))}


@pytest.mark.parametrize("name", CAPTURED)
def test_a_captured_backward_pass_beside_an_eager_graph_of_the_same_leaves_is_refused(name):
    """... before torch makes the eager graph's stream wait for the captured one; the capture goes on, and without that graph, or with
    leaves of its own, the pass is captured and replays."""
    data, call = _captured_calls()[name]
    leaf = data.requires_grad_()
    alive = call(leaf)
    want, = torch.autograd.grad(call(leaf).sum(), leaf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(leaf)
        with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
            torch.autograd.grad(out.sum(), leaf)
        own = leaf.detach().requires_grad_()
        got, = torch.autograd.grad(call(own).sum(), own)
    for _ in range(2):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    del alive, out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(call(leaf).sum(), leaf)
    for _ in range(2):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("name", CAPTURED)
def test_a_captured_backward_pass_over_two_streams(name):
    """A stream that has joined the capture is part of it."""
    data, call = _captured_calls()[name]
    leaf = data.requires_grad_()
    want, = torch.autograd.grad((call(leaf * 1) + call(leaf * 1)).sum(), leaf)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        a, b = leaf * 1, leaf * 1
        side.wait_stream(main)
        with torch.cuda.stream(side):
            one = call(b)
        two = call(a)
        main.wait_stream(side)
        got, = torch.autograd.grad((one + two).sum(), leaf)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        torch.testing.assert_close(got, want, rtol=4 * 2.0 ** -24, atol=4 * 2.0 ** -24 * float(want.abs().max()))
