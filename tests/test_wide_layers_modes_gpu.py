"""GPU: the wide layers beside torch's tracer, forward-mode derivatives and function transforms."""
import pytest
import torch

from triton_helpers_amd.layers.checkpointed_linear import checkpointed_linear
from triton_helpers_amd.layers.int8_linear import Int8Linear, int8_linear, quantize_rows
from triton_helpers_amd.layers.rms_norm import rms_norm, rms_norm_int8
from triton_helpers_amd.layers.wide_mlp import WideMLP

pytestmark = pytest.mark.gpu
DEV = "cuda"
M, K, N = 70, 96, 40

INFERENCE = ["quantize_rows", "int8_linear", "rms_norm_int8", "rms_norm_int8 residual"]
TRAINED = ["rms_norm", "rms_norm residual", "checkpointed_linear"]


def operator(name, seed=0):
    """(operator, its tensor arguments): the input in front."""
    g = torch.Generator(device=DEV).manual_seed(seed)

    def u(*s):
        return torch.randn(*s, generator=g, device=DEV)

    def bytes_of(*s):
        return torch.randint(-127, 128, s, generator=g, device=DEV, dtype=torch.int8)

    if name == "quantize_rows":
        return quantize_rows, [u(M, K)]
    if name == "int8_linear":
        return lambda s, t, b, q, w: int8_linear(q, s, w, t, b, "gelu"), [u(M).abs() * 0.01, u(N).abs() * 0.01, u(N), bytes_of(M, K), bytes_of(N, K)]
    if name.startswith("rms_norm"):
        f = rms_norm_int8 if name.startswith("rms_norm_int8") else rms_norm
        if name.endswith("residual"):
            return lambda x, w, r: f(x, w, 1e-6, r), [u(M, K).bfloat16(), u(K), u(M, K)]
        return f, [u(M, K).bfloat16(), u(K)]
    return lambda x, w, b: checkpointed_linear(x, w, b, "gelu"), [u(M, K).bfloat16(), u(N, K).bfloat16(), u(N)]


def several(out):
    return out if isinstance(out, tuple) else (out,)


@pytest.mark.parametrize("name,train", [(n, False) for n in INFERENCE + TRAINED] + [(n, True) for n in TRAINED])
def test_a_traced_function_runs_the_operator(name, train):
    fn, args = operator(name)
    _, others = operator(name, seed=1)
    if train:
        args[1] = args[1].requires_grad_()

    def doubled(*a):
        return tuple(t.float() * 2 for t in several(fn(*a)))

    traced = torch.jit.trace(doubled, tuple(args), check_trace=False)
    assert "PythonOp" in str(traced.graph) or "^" in str(traced.graph)
    for _ in range(3):
        junk = [torch.full((M, K), 77.0, device=DEV).to(t) for t in (torch.float32, torch.bfloat16, torch.int8)]  # what a fresh allocation may hold
        del junk
        for a, b in zip(traced(*others), doubled(*others)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("name", INFERENCE + TRAINED)
def test_a_traced_function_checks_its_arguments(name):
    """Tensors of another shape or type than at the tracing are held against the operator's conditions before anything is launched."""
    fn, args = operator(name)
    traced = torch.jit.trace(lambda *a: several(fn(*a)), tuple(args), check_trace=False)
    for i in range(1, len(args)):  # (torch's interpreter hands the error on as its own)
        with pytest.raises(RuntimeError, match="must|not implemented|runs on|NotImplemented|Assertion"):
            traced(*args[:i], args[i][:-1], *args[i + 1 :])
    with pytest.raises(RuntimeError):
        traced(args[0].double(), *args[1:])


def test_traced_modules():
    torch.manual_seed(0)
    linear = Int8Linear.from_linear(torch.nn.Linear(K, N).to(DEV, torch.bfloat16), "relu")
    block = WideMLP(K, N).to(DEV, torch.bfloat16).to_int8()
    x, other = torch.randn(M, K, device=DEV).bfloat16(), torch.randn(M, K, device=DEV).bfloat16()
    for m, args, others in ((linear, (x,), (other,)), (block, (x, other), (other, x))):
        traced = torch.jit.trace(m, args, check_trace=False)
        for a, b in zip(several(traced(*others)), several(m(*others))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("mode", ["plain", "no_grad", "train"])
@pytest.mark.parametrize("name,which", [(n, i) for n in INFERENCE + TRAINED for i in range({"quantize_rows": 1, "rms_norm": 2, "rms_norm_int8": 2}.get(n, 3))])
def test_forward_mode_derivatives_are_refused(name, which, mode):
    """A tangent that no kernel carries on raises instead of getting lost."""
    import torch.autograd.forward_ad as fw

    fn, args = operator(name)
    if mode == "train" and name in TRAINED:
        args[1].requires_grad_()
    with fw.dual_level(), torch.set_grad_enabled(mode != "no_grad"):
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            fn(*args)


@pytest.mark.parametrize("name", INFERENCE + TRAINED)
def test_function_transforms_are_refused(name):
    """Inside a transform the autograd Functions refuse, also where the operator's own arguments are plain tensors."""
    fn, args = operator(name)
    want = several(fn(*args))

    def total(s, *a):
        return sum((t.float() * s).sum() for t in several(fn(*a)))

    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda s: total(s, *args))(torch.ones(3, device=DEV))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda s: total(s, *args))(torch.ones((), device=DEV))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: total(1.0, x, *args[1:]))(torch.stack([args[0], args[0]]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: total(1.0, x, *args[1:]))(args[0])
    for a, b in zip(several(fn(*args)), want):
        assert torch.equal(a, b)
