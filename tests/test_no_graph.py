"""The adapter and head operators record no autograd graph, and refuse inputs whose derivatives would be lost: all four
functions, each differentiable operand, reverse and forward mode.  The refusal comes before the device is
looked at, so it is tested on the CPU; on the GPU inside autograd functions."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from test_adapters_gpu import _Plan, make, on_gpu


def lora_operands():
    T, n, r, K, N = 4, 2, 8, 32, 24
    return dict(y=torch.zeros(T, N), x=torch.zeros(T, K), A=torch.zeros(n, r, K), B=torch.zeros(n, N, r), plan=_Plan(T, n),
                scales=torch.ones(n))


def heads_operands():
    T, D = 4, 64
    return dict(q=torch.zeros(T, 2, D), k=torch.zeros(T, 1, D), q_weight=torch.ones(D), k_weight=torch.ones(D),
                positions=torch.zeros(T, dtype=torch.int32), inv_freq=torch.ones(D // 2))


def lora_backward(pkg, y, x, A, B, plan, scales, shrunk, dx):
    return pkg.lora_add_backward(y, x, A, B, plan, scales, shrunk=shrunk, dx=dx)


CALLS = {
    "lora_add": (lambda pkg, **o: pkg.lora_add(*o.values()), lora_operands),
    "lora_add_backward": (lora_backward, lambda: dict(lora_operands(), shrunk=torch.zeros(4, 8), dx=torch.zeros(4, 32))),
    "qk_norm_rope": (lambda pkg, **o: pkg.qk_norm_rope(*o.values()), heads_operands),
    "qk_norm_rope_backward": (lambda pkg, **o: pkg.qk_norm_rope_backward(*o.values()),
                              lambda: dict(q_grad=torch.zeros(4, 2, 64), k_grad=torch.zeros(4, 1, 64), **heads_operands())),
}
OPERANDS = [(call, name) for call, (_, operands) in CALLS.items() for name, t in operands().items()
            if torch.is_tensor(t) and t.is_floating_point()]


@pytest.mark.parametrize("call,name", OPERANDS)
def test_differentiable_operands_are_refused(pkg, call, name):
    run, operands = CALLS[call]
    o = operands()
    o[name].requires_grad_()
    with pytest.raises(RuntimeError, match=f"{call} records no autograd graph"):
        run(pkg, **o)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):  # the next check
        run(pkg, **o)


@pytest.mark.parametrize("call,name", OPERANDS)
def test_dual_operands_are_refused(pkg, call, name):
    run, operands = CALLS[call]
    o = operands()
    with forward_ad.dual_level():
        o[name] = forward_ad.make_dual(o[name], torch.ones_like(o[name]))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match=f"{call} records no autograd graph: forward-mode"):
                run(pkg, **o)
        o[name] = forward_ad.unpack_dual(o[name]).primal
        with pytest.raises(RuntimeError, match="GPU"):
            run(pkg, **o)


def functions(pkg, decorate):
    class Lora(torch.autograd.Function):
        @staticmethod
        def forward(ctx, y, x, A, B, plan, scales):
            out, u = pkg.lora_add(y, x, A, B, plan, scales, return_shrunk=True)
            ctx.save_for_backward(x, A, B, u)
            ctx.rest = plan, scales
            return out

        @staticmethod
        @decorate
        def backward(ctx, dy):
            x, A, B, u = ctx.saved_tensors
            return (dy, *pkg.lora_add_backward(dy, x, A, B, *ctx.rest, shrunk=u), None, None)

    class Heads(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, qw, kw, positions, inv_freq):
            ctx.save_for_backward(q, k, qw, kw, positions, inv_freq)
            return pkg.qk_norm_rope(q, k, qw, kw, positions, inv_freq)

        @staticmethod
        @decorate
        def backward(ctx, gq, gk):
            return (*pkg.qk_norm_rope_backward(gq, gk, *ctx.saved_tensors), None, None)

    return Lora, Heads


@pytest.mark.gpu
@pytest.mark.parametrize("once", [False, True])
def test_second_derivatives_are_refused(pkg, once):
    Lora, Heads = functions(pkg, once_differentiable if once else lambda f: f)
    T, n, r, K, N = 20, 2, 8, 64, 128
    d = on_gpu(make(T, n, r, K, N, "fp32", seed=1))
    plan = pkg.adapter_plan(d["ids"], n)
    A = d["A"].requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    freq, pos = torch.rand(32, device="cuda"), torch.arange(T, device="cuda")
    runs = ((lambda: Lora.apply(d["y"], d["x"], A, d["B"], plan, d["scales"]).square().sum(), A),
            (lambda: Heads.apply(d["y"][:, :64].unflatten(1, (1, 64)), d["y"][:, 64:].unflatten(1, (1, 64)), w, w, pos, freq)[0].pow(3).sum(), w))
    for run, leaf in runs:
        first, = torch.autograd.grad(run(), leaf)
        assert first.isfinite().all() and first.any()
        if once:  # the gradient comes, and torch refuses to go through it again
            again, = torch.autograd.grad(run(), leaf, create_graph=True)
            assert torch.equal(first, again)
            with pytest.raises(RuntimeError, match="once_differentiable"):
                again.sum().backward()
        else:
            with pytest.raises(RuntimeError, match="records no autograd graph, so there are no second"):
                torch.autograd.grad(run(), leaf, create_graph=True)
