"""The operators around a shared projection, run together as a decoder layer uses them: randomized
Hadamard + FP8 quantize, FP8 product, low-rank adapters on slices of its output, norm and rotations of
the query and key heads.  Every stage is checked against the fp64 definition of what the stage before it
gave, with the tolerances of the single operators' tests."""
import pytest
import torch

from test_adapters_gpu import backward64 as lora_backward64, forward64 as lora64, within
from test_heads_gpu import U, backward64 as heads_backward64, forward64 as heads64, pair_matrices

pytestmark = pytest.mark.gpu

T, K, Hq, Hk, D, N_ADAPTERS, RANK = 300, 512, 4, 2, 64, 5, 16


def layer(seed=0):
    g = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g)
    bf = torch.bfloat16
    n = (Hq + 2 * Hk) * D
    pool = lambda width: (randn(N_ADAPTERS, RANK, K).mul(K ** -0.5).to(bf), randn(N_ADAPTERS, width, RANK).mul(0.1).to(bf))
    return dict(x=randn(T, K).to(bf), sign=(torch.randint(0, 2, (K,), generator=g) * 2 - 1).to(torch.int8),
                W=randn(n, K).mul(K ** -0.5).to(bf), ids=torch.randint(-1, N_ADAPTERS, (T,), generator=g),
                q=pool(Hq * D), v=pool(Hk * D), scales=torch.rand(N_ADAPTERS, generator=g) + 0.5,
                qw=(1 + 0.1 * randn(D)).to(bf), kw=(1 + 0.1 * randn(D)).to(bf),
                positions=torch.arange(T, dtype=torch.int32) * 37, inv_freq=10000.0 ** (-torch.arange(0, D, 2) / D))


def to_gpu(p):
    return {k: tuple(t.cuda() for t in v) if isinstance(v, tuple) else v.cuda() for k, v in p.items()}


def run(pkg, d, wq, ws):
    """A layer's projection for a batch: packed queries, keys and values, with the heads' rows in place."""
    plan = pkg.adapter_plan(d["ids"], N_ADAPTERS)
    q8, sx = pkg.rht_quant_fp8(d["x"], d["sign"])
    qkv = pkg.fp8_gemm_rowscale(q8, sx, wq, ws)
    product = qkv.clone()
    values = qkv[:, (Hq + Hk) * D:]
    pkg.lora_add(qkv[:, :Hq * D], d["x"], *d["q"], plan, d["scales"], inplace=True)
    pkg.lora_add(values, d["x"], *d["v"], plan, d["scales"], inplace=True)
    adapted = qkv.clone()
    q, k = qkv[:, :Hq * D].unflatten(1, (Hq, D)), qkv[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D))
    pkg.qk_norm_rope(q, k, d["qw"], d["kw"], d["positions"], d["inv_freq"], hadamard=True, inplace=True)
    return product, adapted, qkv


def test_layer_stage_by_stage(pkg):
    p = layer()
    d = to_gpu(p)
    wq, ws = pkg.rht_quant_fp8(d["W"], d["sign"])  # the weights are rotated the same way, once
    product, adapted, qkv = run(pkg, d, wq, ws)
    # the shared product: FP8 on both sides, so only loosely the unquantized one
    exact = p["x"].double() @ p["W"].double().T
    assert ((product.cpu().double() - exact).norm() / exact.norm()).item() < 0.06
    rows = {"q": slice(0, Hq * D), "v": slice((Hq + Hk) * D, None)}
    for name, cols in rows.items():
        case = dict(x=p["x"], A=p[name][0], B=p[name][1], scales=p["scales"], ids=p["ids"], y=product[:, cols].cpu())
        want, _, slack, _ = lora64(case, "bf16")
        within(adapted[:, cols], want, slack, name)
    keys = slice(Hq * D, (Hq + Hk) * D)
    assert torch.equal(adapted[:, keys], product[:, keys])
    rot = pair_matrices(p["positions"], p["inv_freq"], None, D, False)
    for cols, w, heads in ((rows["q"], "qw", Hq), (keys, "kw", Hk)):
        want = heads64(adapted[:, cols].cpu().unflatten(1, (heads, D)), p[w], rot, 1e-6, True)
        within(qkv[:, cols].unflatten(1, (heads, D)), want, 64 * U * want.norm(dim=-1, keepdim=True))
    assert torch.equal(qkv[:, rows["v"]], adapted[:, rows["v"]])


def test_layer_captured_and_replayed(pkg):
    cases = [layer(s) for s in (1, 2, 3)]
    d = to_gpu(cases[0])
    wq, ws = pkg.rht_quant_fp8(d["W"], d["sign"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(pkg, d, wq, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(pkg, d, wq, ws)
    for _ in range(2):
        for c in cases:
            for name in ("x", "ids", "positions", "scales"):
                d[name].copy_(c[name])
            graph.replay()
            eager = run(pkg, d, wq, ws)
            torch.cuda.synchronize()
            for a, b in zip(out, eager):
                assert torch.equal(a, b)


def test_gradients_through_the_layer(pkg):
    """A training step written as autograd functions around the operators and their backward passes."""

    class Lora(torch.autograd.Function):
        @staticmethod
        def forward(ctx, y, x, A, B, plan, scales):
            out, u = pkg.lora_add(y, x, A, B, plan, scales, return_shrunk=True)
            ctx.save_for_backward(x, A, B, u)
            ctx.plan, ctx.scales = plan, scales
            return out

        @staticmethod
        def backward(ctx, g):
            x, A, B, u = ctx.saved_tensors
            return (g, *pkg.lora_add_backward(g, x, A, B, ctx.plan, ctx.scales, shrunk=u), None, None)

    class Heads(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, qw, kw, positions, inv_freq):
            ctx.save_for_backward(q, k, qw, kw, positions, inv_freq)
            return pkg.qk_norm_rope(q, k, qw, kw, positions, inv_freq, hadamard=True)

        @staticmethod
        def backward(ctx, gq, gk):
            return (*pkg.qk_norm_rope_backward(gq, gk, *ctx.saved_tensors, hadamard=True), None, None)

    p = layer(7)
    d = to_gpu(p)
    plan = pkg.adapter_plan(d["ids"], N_ADAPTERS)
    gen = torch.Generator().manual_seed(8)
    y = torch.randn(T, (Hq + Hk) * D, generator=gen).to(torch.bfloat16)
    gq, gk = ((torch.randn(T, h, D, generator=gen) * 0.1).to(torch.bfloat16) for h in (Hq, Hk))
    A, B = (torch.cat([t, t.flip(-1)[:, :Hk * D] if i else t.new_empty(N_ADAPTERS, 0, K)], 1).cuda().requires_grad_()
            for i, t in enumerate(p["q"]))
    leaves = [y.cuda().requires_grad_(), d["x"].clone().requires_grad_(), A, B, d["qw"].clone().requires_grad_(),
              d["kw"].clone().requires_grad_()]
    out = Lora.apply(*leaves[:4], plan, d["scales"])
    heads = out.unflatten(1, (Hq + Hk, D))
    q, k = Heads.apply(heads[:, :Hq], heads[:, Hq:], *leaves[4:], d["positions"], d["inv_freq"])
    grads = torch.autograd.grad([q, k], leaves, [gq.cuda(), gk.cuda()])

    # the definition, stage by stage: the heads' gradients from the operator's own forward output
    rot = pair_matrices(p["positions"], p["inv_freq"], None, D, False)
    x64, dys = out.detach().cpu().unflatten(1, (Hq + Hk, D)), []
    for part, w, g, i in ((x64[:, :Hq], p["qw"], gq, 4), (x64[:, Hq:], p["kw"], gk, 5)):
        dx, dw, dx_mag, dw_mag = heads_backward64(part, w, g, rot, 1e-6, True)
        dys.append(dx)
        within(grads[i], dw, (96 + T * 3 + 20) * U * dw_mag, f"weight {i}")
    dy = grads[0].cpu()
    within(grads[0], torch.cat(dys, 1).flatten(1), torch.cat([96 * U * heads_backward64(part, w, g, rot, 1e-6, True)[2]
                                                              for part, w, g in ((x64[:, :Hq], p["qw"], gq), (x64[:, Hq:], p["kw"], gk))], 1)
           .expand(T, Hq + Hk, D).flatten(1), "dy")
    case = dict(x=p["x"], A=A.detach().cpu(), B=B.detach().cpu(), scales=p["scales"], ids=p["ids"], dy=dy)
    gx, dA, dB, gx_slack, dA_slack, dB_slack = lora_backward64(case, "bf16")
    within(grads[1], gx, gx_slack, "dx")
    within(grads[2], dA, dA_slack, "dA")
    within(grads[3], dB, dB_slack, "dB")
