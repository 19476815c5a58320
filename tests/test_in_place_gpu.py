"""What ``inplace=True`` and ``dx=`` of the adapter and head operators tell autograd, and what they refuse."""
import pytest
import torch

from test_adapters_gpu import make as make_adapters, on_gpu


def calls(pkg, layout):
    """(name, the call, the tensors it writes) on operands that `layout` brings into place."""
    T, n, r, K, N = 20, 2, 8, 64, 128
    d = on_gpu(make_adapters(T, n, r, K, N, "bf16", seed=1))
    plan = pkg.adapter_plan(d["ids"], n)
    y, dx = layout(d["y"]), layout(torch.zeros_like(d["x"]))
    q, k = layout(torch.randn(T, 2, 64, device="cuda")), layout(torch.randn(T, 1, 64, device="cuda"))
    pos, freq = torch.arange(T, device="cuda"), torch.rand(32, device="cuda")
    return [("lora_add", lambda: pkg.lora_add(y, d["x"], d["A"], d["B"], plan, inplace=True), (y,)),
            ("lora_add_backward", lambda: pkg.lora_add_backward(d["dy"], d["x"], d["A"], d["B"], plan, dx=dx), (dx,)),
            ("qk_norm_rope", lambda: pkg.qk_norm_rope(q, k, None, None, pos, freq, inplace=True), (q, k))]


def shifted(t):
    """One element off the alignment: the operators work on a copy."""
    return torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)


def sliced(t):
    return torch.zeros(*t.shape[:-1], 2 * t.size(-1), dtype=t.dtype, device="cuda")[..., :t.size(-1)].copy_(t)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [lambda t: t, shifted, sliced])
def test_saved_tensors_that_are_written_are_noticed(pkg, layout):
    for name, call, written in calls(pkg, layout):
        for t in written:
            leaf = torch.ones((), device="cuda", dtype=t.dtype, requires_grad=True)
            product = (leaf * t).sum()  # saves t
            before = t._version
            with torch.no_grad():
                call()
            assert t._version > before, name
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                product.backward()


@pytest.mark.gpu
def test_inference_tensors_are_written(pkg):
    with torch.inference_mode():
        listed = calls(pkg, lambda t: t.clone())
        plain = [[t.clone() for t in written] for _, _, written in listed]
        for _, call, _ in listed:
            call()
    again = [[t.clone() for t in written] for _, _, written in listed]
    for _, call, _ in listed:  # outside of the mode as well, as before
        call()
    for a, b, (name, _, written) in zip(plain, again, listed):
        assert all(t.is_inference() for t in written)
        assert all(not torch.equal(x, y) for x, y in zip(a, b)), name
