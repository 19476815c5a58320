"""Infinite and NaN operands of ``lora_add`` and ``lora_add_backward``: an output is infinite (with its sign),
NaN or finite exactly where the definition, evaluated in fp64, is; finite values are those of the call without the
infinities, bit by bit, wherever they do not depend on what was changed.
"""
import pytest
import torch

from test_adapters_gpu import make, on_gpu

INF, NAN = float("inf"), float("nan")
SIZES = [(80, 3, 16), (80, 3, 40), (1300, 3, 16), (1300, 3, 72), (9000, 5, 64)]
K, N = 72, 136
UNTOUCHED = {"x": "dx", "dy": "out", "A": "dA", "B": "dB"}  # what does not depend on an operand


def definition(c):
    """out, dx, dA, dB in fp64."""
    out, dx = c["y"].double(), torch.zeros(len(c["x"]), K, dtype=torch.float64)
    dA, dB = torch.zeros(c["A"].shape, dtype=torch.float64), torch.zeros(c["B"].shape, dtype=torch.float64)
    for a in range(len(c["A"])):
        t = c["ids"] == a
        x, g, A, B, s = (v.double() for v in (c["x"][t], c["dy"][t], c["A"][a], c["B"][a], c["scales"][a]))
        u, d = x @ A.T, s * (g @ B)
        out[t] += (s * u) @ B.T
        dx[t] = d @ A
        dA[a] = d.T @ x
        dB[a] = g.T @ (s * u)
    return out, dx, dA, dB


def kernels(pkg, c):
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], len(c["A"]))
    out = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, d["scales"])
    grads = pkg.lora_add_backward(d["dy"], d["x"], d["A"], d["B"], plan, d["scales"])
    return [t.cpu() for t in (out, *grads)]


def changed(c, operand):
    c = {k: v.clone() for k, v in c.items()}
    t = torch.nonzero(c["ids"] == 1).flatten()
    if operand == "B":
        c["B"][1, 3, 2], c["B"][1, 9, 0], c["B"][1, 9, 5], c["B"][1, 20, 7], c["B"][1, N - 1, 1] = INF, INF, -INF, NAN, -INF
    elif operand == "A":
        c["A"][1, 2, 3], c["A"][1, 5, K - 1], c["A"][0, 1, 9] = INF, -INF, NAN
    elif operand == "x":
        c["x"][t[0], 3], c["x"][t[5], 40], c["x"][t[9], K - 1] = INF, -INF, NAN
    elif operand == "dy":
        c["dy"][t[0], 3], c["dy"][t[5], 40], c["dy"][t[9], N - 1] = INF, -INF, NAN
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("operand", ["B", "A", "x", "dy"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,n,r", SIZES)
def test_infinities_are_the_definitions(pkg, T, n, r, dtype, operand):
    clean = make(T, n, r, K, N, dtype, "mixed", seed=T + r, grad_scale=0.5)
    clean["scales"] = clean["scales"].abs() + 0.25  # none is zero
    for name in ("x", "A", "B", "dy"):  # nor any operand: zero times infinity is NaN
        clean[name][clean[name] == 0] = 0.5
    c = changed(clean, operand)
    before, after = kernels(pkg, clean), kernels(pkg, c)
    for name, ref, got, want, plain in zip(("out", "dx", "dA", "dB"), before, after, definition(c), definition(clean)):
        assert torch.equal(got.isnan(), want.isnan()), name
        inf = want.isinf()
        assert torch.equal(got.isinf(), inf) and torch.equal(got[inf].double(), want[inf]), name
        same = want == plain
        assert torch.equal(got[same], ref[same]), name
        assert same.all() == (name == UNTOUCHED[operand]), name
