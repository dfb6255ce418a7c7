"""Dense-head operators (pointnet2_ops.head_ops) without a GPU: every refusal comes before any launch, with its reason."""
import ctypes

import pytest
import torch

from pointnet2_ops import _ext, head_ops as ho


def f(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


REFUSALS = [
    ("CPU not supported", lambda: ho.linear_act(f(2, 3), f(4, 3))),
    ("CPU not supported", lambda: ho.label_log_probs(f(2, 3), torch.zeros(2, dtype=torch.int64))),
    ("CPU not supported", lambda: ho.distill_top_k(f(2, 3), torch.zeros(2, 1, dtype=torch.int64), f(2, 1))),
    # linear_act
    ("weight must have shape", lambda: ho.linear_act(f(2, 3), f(4, 5))),
    ("weight must have shape", lambda: ho.linear_act(f(2, 3), f(3))),
    ("weight must have the type of x", lambda: ho.linear_act(f(2, 3), f(4, 3, dtype=torch.bfloat16))),
    ("at least one row", lambda: ho.linear_act(f(2, 3), f(0, 3))),
    ("at least one column", lambda: ho.linear_act(f(2, 0), f(4, 0))),
    ("activation must be one of", lambda: ho.linear_act(f(2, 3), f(4, 3), activation="tanh")),
    ("bias must be", lambda: ho.linear_act(f(2, 3), f(4, 3), f(3))),
    ("bias must have the type", lambda: ho.linear_act(f(2, 3), f(4, 3), f(4, dtype=torch.float16))),
    ("residual must broadcast", lambda: ho.linear_act(f(2, 3), f(4, 3), residual=f(2, 5))),
    ("residual must have the type", lambda: ho.linear_act(f(2, 3), f(4, 3), residual=f(2, 4, dtype=torch.float16))),
    ("float32, bfloat16 or float16", lambda: ho.linear_act(f(2, 3, dtype=torch.float64), f(4, 3, dtype=torch.float64))),
    ("at least one axis", lambda: ho.linear_act(torch.tensor(1.0), f(4, 3))),
    # label_log_probs
    ("labels must be a long", lambda: ho.label_log_probs(f(2, 3), torch.zeros(2, dtype=torch.int32))),
    ("labels must be a tensor of shape", lambda: ho.label_log_probs(f(2, 3), torch.zeros(3, dtype=torch.int64))),
    ("top must lie in", lambda: ho.label_log_probs(f(2, 3), torch.zeros(2, dtype=torch.int64), top=4)),
    ("top must lie in", lambda: ho.label_log_probs(f(2, 300), torch.zeros(2, dtype=torch.int64), top=65)),
    ("top must lie in", lambda: ho.label_log_probs(f(2, 3), torch.zeros(2, dtype=torch.int64), top=-1)),
    ("at least one column", lambda: ho.label_log_probs(f(2, 0), torch.zeros(2, dtype=torch.int64))),
    # distill_top_k
    ("teacher_index must be a long", lambda: ho.distill_top_k(f(2, 3), torch.zeros(2, 1, dtype=torch.int32), f(2, 1))),
    ("must have shape", lambda: ho.distill_top_k(f(2, 3), torch.zeros(2, 2, dtype=torch.int64), f(2, 1))),
    ("teacher_index must be a tensor of shape", lambda: ho.distill_top_k(f(2, 3), torch.zeros(3, 1, dtype=torch.int64), f(2, 1))),
    ("k >= 1", lambda: ho.distill_top_k(f(2, 3), torch.zeros(2, 0, dtype=torch.int64), f(2, 0))),
    ("temperature", lambda: ho.distill_top_k(f(2, 3), torch.zeros(2, 1, dtype=torch.int64), f(2, 1), temperature=0.0)),
    ("temperature", lambda: ho.distill_top_k(f(2, 3), torch.zeros(2, 1, dtype=torch.int64), f(2, 1), temperature=float("inf"))),
    ("temperature", lambda: ho.distill_top_k(f(2, 3), torch.zeros(2, 1, dtype=torch.int64), f(2, 1), temperature=float("nan"))),
    ("must not require a gradient",
     lambda: ho.distill_top_k(f(2, 3), torch.zeros(2, 1, dtype=torch.int64), f(2, 1).requires_grad_())),
]


@pytest.mark.parametrize("match,call", REFUSALS, ids=[f"{i}" for i in range(len(REFUSALS))])
def test_refusals(match, call):
    with pytest.raises(RuntimeError, match=match):
        call()


@pytest.mark.parametrize("match,call", [
    ("x must be a torch.Tensor", lambda: ho.linear_act([1.0], f(4, 3))),
    ("weight must be a torch.Tensor", lambda: ho.linear_act(f(2, 3), None)),
    ("bias must be a torch.Tensor", lambda: ho.linear_act(f(2, 3), f(4, 3), 1.0)),
    ("residual must be a torch.Tensor", lambda: ho.linear_act(f(2, 3), f(4, 3), residual=0)),
    ("activation must be one of", lambda: ho.linear_act(f(2, 3), f(4, 3), activation=["relu"])),
    ("activation must be one of", lambda: ho.linear_act(f(2, 3), f(4, 3), activation=None)),
    ("labels must be a torch.Tensor", lambda: ho.label_log_probs(f(2, 3), [0, 1])),
    ("teacher_logits must be a torch.Tensor", lambda: ho.distill_top_k(f(2, 3), torch.zeros(2, 1, dtype=torch.int64), None)),
    ("teacher_index must be a tensor of shape", lambda: ho.distill_top_k(f(3), torch.zeros(2, 2, dtype=torch.int64), f(2, 2))),
    ("at most 4194304", lambda: ho.linear_act(f(1, 1).expand(1, 2 ** 22 + 1), f(1, 1).expand(1, 2 ** 22 + 1))),
    ("residual must broadcast", lambda: ho.linear_act(f(2, 3), f(4, 3), residual=f(1, 2, 4))),
])
def test_refusals_of_other_objects_and_shapes(match, call):
    with pytest.raises(RuntimeError, match=match):
        call()


def test_entry_points_refuse_bad_arguments_before_any_launch():
    """Every argument check of the C entry points returns its code on the host (the pointers are never followed)."""
    lib = _ext._lib
    some, big = ctypes.c_void_p(16), 1 << 40
    EINVAL, ENULL, ENOSPC = -1, -2, -4

    def linear(M=4, N=4, K=4, dt=0, x=some, w=some, b=None, bdt=0, act=0, y=some, ws=None, nb=0):
        return lib.pn2_linear_act(M, N, K, dt, x, K, w, K, b, bdt, act, None, 0, y, None, ws, nb, None)
    assert linear(M=-1) == linear(N=0) == linear(K=0) == linear(dt=3) == linear(dt=-1) == linear(act=5) == linear(act=-1) == EINVAL
    assert linear(dt=1, b=some, bdt=2) == linear(M=big) == linear(N=(1 << 22) + 1) == EINVAL
    assert linear(x=None) == linear(w=None) == linear(y=None) == ENULL
    assert linear(M=0, x=None) == 0
    # a product whose contraction is split needs its workspace
    assert lib.pn2_linear_act_workspace_bytes(64, 64, 32768, 0, some, 32768, some, 32768) > 0
    assert linear(M=64, N=64, K=32768) == ENOSPC
    assert linear(M=64, N=64, K=32768, nb=big) == ENULL
    # ... and one whose operands have to be padded (a row stride of no whole 16 bytes)
    assert lib.pn2_linear_act_workspace_bytes(2048, 2048, 512, 1, some, 512, some, 512) == 0
    assert lib.pn2_linear_act_workspace_bytes(2048, 2048, 512, 1, some, 513, some, 512) >= 2048 * 512 * 2

    def grad(M=4, dy=some, x=some, w=some, dx=some, dw=some, db=None, bdt=0, nb=big, ws=some):
        return lib.pn2_linear_act_grad(M, 4, 4, 0, dy, 4, None, x, 4, w, 4, dx, dw, db, bdt, ws, nb, None)
    assert grad(M=0) == grad(db=some, bdt=1) == EINVAL
    assert grad(dy=None) == grad(x=None) == grad(w=None) == ENULL
    assert lib.pn2_linear_act_grad_workspace_bytes(4096, 512, 512, 0, some, 512, 1, some, 512, some, 512, 7) >= 4096 * 512 * 4

    def labels(T=4, V=8, dt=0, x=some, y=some, top=0, lp=some, tl=None, ws=None, nb=0):
        return lib.pn2_label_logprobs(T, V, V, dt, x, y, -100, top, lp, some, None, tl, tl, ws, nb, None)
    assert labels(T=-1) == labels(V=0) == labels(dt=7) == labels(top=9) == labels(top=-1) == labels(V=100, top=65) == EINVAL
    assert labels(x=None) == labels(y=None) == labels(lp=None) == labels(top=1) == ENULL
    assert labels(T=0, x=None) == 0
    # few long rows are summed in segments, whose results meet in a workspace
    need = lib.pn2_label_logprobs_workspace_bytes(1, 131072, 1, 20)
    assert need > 0 and lib.pn2_label_logprobs_workspace_bytes(1000, 131072, 1, 20) == 0
    assert lib.pn2_label_logprobs_workspace_bytes(-1, 131072, 1, 20) == lib.pn2_label_logprobs_workspace_bytes(1, 2048, 1, 20) == 0
    assert labels(T=1, V=131072, dt=1, top=20, tl=some, nb=need - 1) == ENOSPC
    assert labels(T=1, V=131072, dt=1, top=20, tl=some, nb=need) == ENULL

    def distill(k=2, t=1.0, tdt=0, x=some, T=4, V=8, nb=0):
        return lib.pn2_distill_topk(T, V, V, 0, x, k, some, tdt, some, t, some, None, None, nb, None)
    assert distill(k=0) == distill(t=0.0) == distill(t=-1.0) == distill(t=float("nan")) == distill(t=float("inf")) == EINVAL
    assert distill(tdt=3) == EINVAL and distill(x=None) == ENULL


# ------------------------------------------- what torch's dispatcher would do beside the launch is refused before the device is looked at
def _calls():
    y, i = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 1, dtype=torch.int64)
    return {"linear_act x": lambda t: ho.linear_act(t, f(4, 3)), "linear_act weight": lambda t: ho.linear_act(f(2, 3), t),
            "linear_act residual": lambda t: ho.linear_act(f(2, 3), f(3, 3), residual=t),
            "linear_act bias": lambda t: ho.linear_act(f(2, 3), f(3, 3), t[0]), "linear_act grad": lambda t: ho.linear_act(t, f(4, 3).requires_grad_()),
            "label_log_probs logits": lambda t: ho.label_log_probs(t, y).log_prob,
            "distill_top_k logits": lambda t: ho.distill_top_k(t, i, f(2, 1)),
            "distill_top_k teacher_logits": lambda t: ho.distill_top_k(f(2, 3), torch.zeros(2, 3, dtype=torch.int64), t)}


@pytest.mark.parametrize("name", list(_calls()))
def test_forward_mode_is_refused(name):
    import torch.autograd.forward_ad as fwd
    call = _calls()[name]
    with fwd.dual_level():
        dual = fwd.make_dual(f(2, 3), torch.ones(2, 3))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            call(dual)
    with pytest.raises(RuntimeError, match="CPU not supported"):      # (the same call without a tangent gets as far as the device)
        call(f(2, 3))


@pytest.mark.parametrize("name", list(_calls()))
@pytest.mark.filterwarnings("ignore")
def test_recording_is_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    call = _calls()[name]
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        torch.jit.trace(call, (f(2, 3),))
    for mode in ("real", "symbolic"):
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            make_fx(call, tracing_mode=mode, _allow_non_fake_inputs=True)(f(2, 3))
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        make_fx(call, pre_dispatch=True)(f(2, 3))


@pytest.mark.parametrize("name", list(_calls()))
def test_tensors_that_are_not_plain_memory_are_refused(name):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Sub(torch.Tensor):
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return func(*[torch.Tensor(a) if isinstance(a, cls) else a for a in args], **(kwargs or {}))
    call = _calls()[name]
    if name != "linear_act bias":                                     # (whose row is a plain tensor by then)
        with pytest.raises(RuntimeError, match="plain tensor"):
            call(torch.Tensor._make_subclass(Sub, f(2, 3)))
    with pytest.raises(RuntimeError):
        torch.func.functionalize(call)(f(2, 3))
    with pytest.raises(RuntimeError, match="memory of its own"):
        call(torch._efficientzerotensor((3, 3))[1:])
    with pytest.raises(RuntimeError, match="memory of its own"):
        call(f(2, 3).to_sparse())
    for transform in (torch.vmap, torch.func.grad, lambda g: lambda t: torch.func.jvp(g, (t,), (t,))):
        with pytest.raises(RuntimeError):
            transform(call)(f(2, 2, 3) if transform is torch.vmap else f(2, 3))

    class Watch(TorchDispatchMode):                                   # a mode that only looks on is none of these
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    with Watch(), pytest.raises(RuntimeError, match="CPU not supported"):
        call(f(2, 3))


def test_objects_are_built_again_when_the_flags_change():
    """`make` with a newer Makefile names every source again (asked for, not run)."""
    import glob
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "4d-or_amd", "csrc")
    plan = subprocess.run(["make", "-n", "-W", "Makefile", "-C", csrc], capture_output=True, text=True, check=True).stdout
    sources = [os.path.basename(p) for p in glob.glob(os.path.join(csrc, "*.hip"))]
    assert len(sources) >= 15
    for name in sources:
        assert any(f"-c {name} " in line and "-packed-fp32-ops" in line for line in plan.splitlines()), name
    assert "head_binding.cpp" in plan
