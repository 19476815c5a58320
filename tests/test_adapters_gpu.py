"""GPU tests of ``adapter_plan``, ``lora_add`` and ``lora_add_backward`` against the definition in fp64.

Tolerances.  An output is rounded once: half a step of its type.  A matrix-core sum of n products is off
by at most (n / 8 + 64) u of the sum of their magnitudes, u = 2^-24 (at least eight products meet in one
step; 64 for the steps' own additions and the sums across wavefronts and parts).  The rank-space
vector between the products is two 16-bit pieces: 2^-16 of each value for bf16 (half a step of the half
step), 2^-22 for fp16, exact for fp32.  For the contraction over tokens the fp16 pieces share the scale of
a tile's largest value, which adds 2^-38 of that.
"""
import ctypes

import pytest
import torch

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PIECE = {"bf16": 2.0 ** -16, "fp16": 2.0 ** -22, "fp32": 0.0}


def within(got, want, slack, what=""):
    f = torch.finfo(got.dtype)
    tol = want.abs() * f.eps / 2 + f.tiny * f.eps / 2 + slack
    err = (got.cpu().double() - want).abs()
    assert got.shape == want.shape
    assert (err <= tol).all(), f"{what}: worst error {(err / tol.clamp_min(1e-300)).max().item()} of the bound"


def sums(n):
    return (n / 8 + 64) * U


def make(T, n, r, K, N, dtype, ids="mixed", seed=0, grad_scale=0.1):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    if ids == "mixed":
        i = torch.randint(-1, n, (T,), generator=g)
    elif ids == "runs":
        i = torch.sort(torch.randint(0, n, (T,), generator=g)).values
        i = (i * 7 + 3) % n
    elif ids == "none":
        i = torch.full((T,), -1)
    else:
        i = torch.full((T,), int(ids))
    randn = lambda *s: torch.randn(*s, generator=g)
    return dict(ids=i, x=randn(T, K).to(dt), A=(randn(n, r, K) * K ** -0.5).to(dt), B=(randn(n, N, r) * r ** -0.5).to(dt),
                scales=torch.rand(n, generator=g) * 2 - 0.5, y=randn(T, N).to(dt), dy=(randn(T, N) * grad_scale).to(dt))


def forward64(c, dtype, scales=True):
    """out and u with the magnitudes of their errors."""
    T, K = c["x"].shape
    n, N, r = c["B"].shape
    out, u = c["y"].double(), torch.zeros(T, r, dtype=torch.float64)
    out_slack, u_slack = out.abs() * U, torch.zeros(T, r, dtype=torch.float64)
    for a in range(n):
        t = c["ids"] == a
        if not t.any():
            continue
        x, A, B = c["x"][t].double(), c["A"][a].double(), c["B"][a].double()
        s = c["scales"][a].double() if scales else torch.tensor(1.0, dtype=torch.float64)
        u[t] = x @ A.T
        u_slack[t] = sums(K) * (x.abs() @ A.abs().T)
        out[t] += s * u[t] @ B.T
        out_slack[t] += s.abs() * (u_slack[t] + (PIECE[dtype] + sums(r)) * u[t].abs()) @ B.abs().T
    return out, u, out_slack, u_slack


def backward64(c, dtype, dx=None):
    T, K = c["x"].shape
    n, N, r = c["B"].shape
    gx = torch.zeros(T, K, dtype=torch.float64) if dx is None else dx.double()
    gx_slack = gx.abs() * U
    dA, dB = torch.zeros(n, r, K, dtype=torch.float64), torch.zeros(n, N, r, dtype=torch.float64)
    dA_slack, dB_slack = torch.zeros_like(dA), torch.zeros_like(dB)
    half = 2.0 ** -38 if dtype == "fp16" else 0.0
    for a in range(n):
        t = c["ids"] == a
        if not t.any():
            continue
        x, g, A, B, s = (v.double() for v in (c["x"][t], c["dy"][t], c["A"][a], c["B"][a], c["scales"][a]))
        u, u_slack = x @ A.T, sums(K) * (x.abs() @ A.abs().T)
        d, d_slack = s * g @ B, s.abs() * sums(N) * (g.abs() @ B.abs())
        gx[t] += d @ A
        gx_slack[t] += (d_slack + (PIECE[dtype] + sums(r)) * d.abs()) @ A.abs()
        own = PIECE[dtype] + sums(len(x))
        dA[a] = d.T @ x
        dA_slack[a] = (d_slack + own * d.abs() + half * d.abs().max()).T @ x.abs()
        dB[a] = s * g.T @ u
        dB_slack[a] = s.abs() * g.abs().T @ (u_slack + own * u.abs() + half * u.abs().max())
    return gx, dA, dB, gx_slack, dA_slack, dB_slack


def on_gpu(c):
    return {k: v.cuda() for k, v in c.items()}


# ---------------------------------------------------------------------------------------------
# the plan

@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("T,n", [(0, 3), (1, 1), (1, 1024), (63, 2), (64, 1), (65, 5), (1000, 64), (1024, 1024),
                                 (4096, 700), (4097, 3), (40000, 17), (40000, 900),
                                 (70000, 1), (300001, 40)])
def test_plan_groups_tokens_in_order(pkg, T, n, bits):
    g = torch.Generator().manual_seed(T + n)
    ids = torch.randint(-2, n + 2, (T,), generator=g, dtype=torch.int64)
    if T > 4:
        ids[1], ids[3] = 2 ** 31 - 1, -(2 ** 31)
        if bits == 64:
            ids[2] = 2 ** 32  # 0 in its low half: not adapter 0
    plan = pkg.adapter_plan(ids.cuda() if bits == 64 else ids.to(torch.int32).cuda(), n)
    key = torch.where((ids >= 0) & (ids < n), ids, n)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=n + 1)
    starts = torch.cumsum(counts, 0) - counts
    assert torch.equal(plan.order.cpu().long(), order) and torch.equal(plan.starts.cpu().long(), starts)
    # the tables of work: tiles of 64 and chunks of 128 to 512 tokens of one adapter
    groups = min(T, n + 1)
    size = 128 if T < 4096 else 256 if T < 8192 else 512  # of a chunk
    max_tiles, max_chunks = T // 64 + groups, T // size + groups
    buf = plan.buffer.cpu()
    n_tiles, n_chunks = buf[4 * max_tiles + 8 * max_chunks:][:2].tolist()
    tiles, chunks, slots, tile_of = [], [], 0, {}
    for a in range(n + 1):
        first, left = starts[a].item(), counts[a].item()
        tile_of[a] = len(tiles)
        tiles += [(a, first + i, min(64, left - i)) for i in range(0, left, 64)]
        if a == n:
            break
        many = left > size
        for i in range(0, left, size):
            chunks.append((a, first + i, min(size, left - i), slots if many else -1, tile_of[a] + i // 64))
            slots += many
    assert (n_tiles, n_chunks) == (len(tiles), len(chunks)) and n_tiles <= max_tiles and n_chunks <= max_chunks
    assert slots <= 2 * (T // size)
    assert buf[:4 * n_tiles].view(-1, 4)[:, :3].tolist() == [list(t) for t in tiles]
    assert buf[4 * max_tiles:][:8 * n_chunks].view(-1, 8)[:, :5].tolist() == [list(c) for c in chunks]


@pytest.mark.gpu
def test_plan_in_a_graph_follows_its_ids(pkg):
    T, n = 3000, 9
    ids = torch.zeros(T, dtype=torch.int32, device="cuda")
    pkg.adapter_plan(ids, n)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan = pkg.adapter_plan(ids, n)
    for seed in range(3):
        ids.copy_(torch.randint(-1, n, (T,), generator=torch.Generator().manual_seed(seed)))
        g.replay()
        eager = pkg.adapter_plan(ids, n)
        torch.cuda.synchronize()
        assert torch.equal(plan.order, eager.order) and torch.equal(plan.starts, eager.starts)


# ---------------------------------------------------------------------------------------------
# forward and backward

CASES = [
    # T, n, r, K, N, dtype, ids
    (1, 4, 16, 4096, 512, "bf16", "2"),
    (1, 1, 8, 8, 8, "fp32", "0"),
    (5, 3, 8, 24, 40, "bf16", "mixed"),
    (17, 3, 24, 200, 136, "fp16", "mixed"),
    (64, 50, 16, 1024, 1000, "bf16", "mixed"),
    (65, 1, 32, 512, 264, "fp32", "0"),
    (100, 3, 40, 1000, 520, "fp32", "runs"),
    (130, 2, 64, 264, 1544, "bf16", "runs"),
    (333, 5, 72, 328, 248, "fp16", "mixed"),
    (200, 3, 128, 520, 392, "bf16", "mixed"),
    (150, 2, 128, 136, 520, "fp32", "runs"),
    (1100, 2, 16, 520, 640, "bf16", "1"),
    (1601, 3, 24, 264, 136, "fp16", "runs"),
    (1300, 70, 8, 72, 264, "fp32", "mixed"),
    (40, 3, 16, 64, 64, "bf16", "none"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,r,K,N,dtype,ids", CASES)
def test_forward_against_the_definition(pkg, T, n, r, K, N, dtype, ids):
    c = make(T, n, r, K, N, dtype, ids, seed=T + r)
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], n)
    y0 = d["y"].clone()
    out, u = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, d["scales"], return_shrunk=True)
    want, want_u, slack, u_slack = forward64(c, dtype)
    within(out, want, slack, "out")
    within(u, want_u, u_slack, "u")
    assert torch.equal(d["y"], y0)
    none = c["ids"] < 0
    assert torch.equal(out.cpu()[none], c["y"][none]) and (u.cpu()[none] == 0).all()
    # in place, and without factors
    same = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, d["scales"], inplace=True)
    assert same is d["y"] and torch.equal(same, out)
    plain = pkg.lora_add(y0, d["x"], d["A"], d["B"], plan)
    want, _, slack, _ = forward64(c, dtype, scales=False)
    within(plain, want, slack, "no scales")


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,r,K,N,dtype,ids", CASES)
def test_backward_against_the_formulas(pkg, T, n, r, K, N, dtype, ids):
    c = make(T, n, r, K, N, dtype, ids, seed=T + r + 1)
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], n)
    _, u = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, d["scales"], return_shrunk=True)
    args = (d["dy"], d["x"], d["A"], d["B"], plan, d["scales"])
    got = pkg.lora_add_backward(*args, shrunk=u)
    gx, dA, dB, gx_slack, dA_slack, dB_slack = backward64(c, dtype)
    within(got[0], gx, gx_slack, "dx")
    within(got[1], dA, dA_slack, "dA")
    within(got[2], dB, dB_slack, "dB")
    used = torch.zeros(n, dtype=torch.bool)
    used[c["ids"][c["ids"] >= 0]] = True
    assert (got[1].cpu()[~used] == 0).all() and (got[2].cpu()[~used] == 0).all()
    assert (got[0].cpu()[c["ids"] < 0] == 0).all()
    # again, with u computed again: the same bits
    again = pkg.lora_add_backward(*args)
    for a, b in zip(got, again):
        assert torch.equal(a, b)
    # added to the projection's own gradient
    base = torch.randn(T, K, generator=torch.Generator().manual_seed(3)).to(DT[dtype])
    dx = base.cuda()
    res = pkg.lora_add_backward(*args, shrunk=u, dx=dx)
    assert res[0] is dx
    gx, _, _, gx_slack, _, _ = backward64(c, dtype, base)
    within(dx, gx, gx_slack, "dx added")
    assert torch.equal(dx.cpu()[c["ids"] < 0], base[c["ids"] < 0])


@pytest.mark.gpu
def test_backward_against_differences(pkg):
    """fp32: the map is linear in x and bilinear in A, B, so a central difference has rounding errors only:
    below 2e-4 of the largest gradient for a step of 2^-3."""
    c = make(9, 2, 8, 32, 24, "fp32", "mixed", seed=5, grad_scale=1.0)
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], 2)
    grads = dict(zip(("x", "A", "B"), pkg.lora_add_backward(d["dy"], d["x"], d["A"], d["B"], plan, d["scales"])))
    for name, grad in grads.items():
        for i in range(0, grad.numel(), 37):
            slope = 0.0
            for sign in (1.0, -1.0):
                v = d[name].clone().flatten()
                v[i] += sign * 0.125
                e = {**d, name: v.view(d[name].shape)}
                out = pkg.lora_add(e["y"], e["x"], e["A"], e["B"], plan, e["scales"])
                slope += sign * (out.double() * d["dy"].double()).sum().item()
            assert abs(slope / 0.25 - grad.flatten()[i].item()) <= 2e-4 * max(1.0, grad.abs().max().item()), (name, i)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-6, 3e4])
def test_fp16_ranges(pkg, scale):
    """Gradients near the smallest fp16 numbers, and a rank-space vector beyond the largest."""
    c = make(70, 2, 16, 256, 128, "fp16", "mixed", seed=6)
    if scale > 1:
        c["x"] = (c["x"].float().clamp(-2, 2) * scale).to(torch.float16)
        c["A"] = (c["A"].float() * 16).to(torch.float16)
        c["B"] = (c["B"].float() * 1e-5).to(torch.float16)  # subnormal fp16
        c["dy"] = (c["dy"].float() * 1e-3).to(torch.float16)
    else:
        c["dy"] = (c["dy"].float() * 1e-5).to(torch.float16)
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], 2)
    out, u = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, d["scales"], return_shrunk=True)
    want, want_u, slack, u_slack = forward64(c, "fp16")
    assert scale < 1 or want_u.abs().max() > 65504
    within(u, want_u, u_slack, "u")
    within(out, want, slack, "out")
    got = pkg.lora_add_backward(d["dy"], d["x"], d["A"], d["B"], plan, d["scales"], shrunk=u)
    gx, dA, dB, gx_slack, dA_slack, dB_slack = backward64(c, "fp16")
    within(got[0], gx, gx_slack, "dx")
    within(got[1], dA, dA_slack, "dA")
    within(got[2], dB, dB_slack, "dB")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_infinities_and_nan_stay_with_their_token_and_adapter(pkg, dtype):
    T, n, r, K, N = 80, 3, 8, 72, 40
    c = make(T, n, r, K, N, dtype, "mixed", seed=7)
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], n)
    ref = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan)
    gref = pkg.lora_add_backward(d["dy"], d["x"], d["A"], d["B"], plan)
    none = torch.nonzero(c["ids"] < 0).flatten()
    zero = torch.nonzero(c["ids"] == 0).flatten()
    x = d["x"].clone()
    x[none[0]] = float("nan")
    x[zero[1], 3] = float("inf")
    out = pkg.lora_add(d["y"], x, d["A"], d["B"], plan)
    keep = torch.ones(T, dtype=torch.bool)
    keep[zero[1]] = False
    assert torch.equal(out.cpu()[keep], ref.cpu()[keep])
    assert not torch.isfinite(out[zero[1]]).any()
    grads = pkg.lora_add_backward(d["dy"], x, d["A"], d["B"], plan)
    assert torch.equal(grads[0], gref[0])  # dx does not read x
    for i in (1, 2):
        assert torch.equal(grads[i][1:], gref[i][1:])
        assert torch.isfinite(gref[i]).all() and not torch.isfinite(grads[i][0]).all()
    # an adapter of NaN that no token uses, and NaN gradients of a token without an adapter
    A = torch.cat([d["A"], torch.full_like(d["A"][:1], float("nan"))])
    B = torch.cat([d["B"], torch.full_like(d["B"][:1], float("nan"))])
    dy = d["dy"].clone()
    dy[none[0]] = float("nan")
    wide = pkg.adapter_plan(d["ids"], n + 1)
    assert torch.equal(pkg.lora_add(d["y"], d["x"], A, B, wide), ref)
    grads = pkg.lora_add_backward(dy, d["x"], A, B, wide)
    assert torch.equal(grads[0], gref[0])
    for i in (1, 2):
        assert torch.equal(grads[i][:n], gref[i]) and (grads[i][n] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_operand_layouts(pkg, dtype):
    """Column slices, strides that are copied, transposed pools, int64 ids, empty batches."""
    T, n, r, K, N = 37, 3, 16, 64, 48
    c = make(T, n, r, K, N, dtype, "mixed", seed=9)
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], n)
    sc = d["scales"]
    ref, u = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, sc, return_shrunk=True)
    gref = pkg.lora_add_backward(d["dy"], d["x"], d["A"], d["B"], plan, sc, shrunk=u)
    dt = DT[dtype]

    def slices(t):
        wide = torch.zeros(T, t.size(1) + 32, dtype=dt, device="cuda")
        odd = torch.zeros(T, t.size(1) + 3, dtype=dt, device="cuda")
        gaps = torch.zeros(T, 2 * t.size(1), dtype=dt, device="cuda")
        turned = torch.zeros(t.size(1), T, dtype=dt, device="cuda").T
        return [w.copy_(t) for w in (wide[:, 16:-16], odd[:, 1:-2], gaps[:, ::2], turned)]

    for x, y, dy in zip(slices(d["x"]), slices(d["y"]), slices(d["dy"])):
        assert torch.equal(pkg.lora_add(y, x, d["A"], d["B"], plan, sc), ref)
        for a, b in zip(pkg.lora_add_backward(dy, x, d["A"], d["B"], plan, sc, shrunk=u), gref):
            assert torch.equal(a, b)
        base = y._base if y._base is not None else y
        outside = base.clone()
        assert pkg.lora_add(y, x, d["A"], d["B"], plan, sc, inplace=True) is y
        assert torch.equal(y, ref)
        y.copy_(d["y"])
        assert torch.equal(base, outside)  # nothing beside the slice was written
        dx = slices(torch.zeros_like(d["x"]))[0]
        whole = dx._base
        assert pkg.lora_add_backward(dy, x, d["A"], d["B"], plan, sc, shrunk=u, dx=dx)[0] is dx
        assert torch.equal(dx, gref[0]) and (whole[:, :16] == 0).all() and (whole[:, -16:] == 0).all()
    At = d["A"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(pkg.lora_add(d["y"], d["x"], At, d["B"], plan, sc), ref)
    one = d["x"][:1].expand(T, K)
    assert torch.equal(pkg.lora_add(d["y"], one, d["A"], d["B"], plan, sc), pkg.lora_add(d["y"], one.contiguous(), d["A"], d["B"], plan, sc))
    with pytest.raises(RuntimeError, match="share memory"):
        pkg.lora_add(d["y"][:1].expand(T, N), d["x"], d["A"], d["B"], plan, sc, inplace=True)
    with pytest.raises(RuntimeError, match="share memory"):
        pkg.lora_add_backward(d["dy"], d["x"], d["A"], d["B"], plan, sc, dx=one)
    empty = pkg.adapter_plan(d["ids"][:0], n)
    assert pkg.lora_add(d["y"][:0], d["x"][:0], d["A"], d["B"], empty, sc).shape == (0, N)
    grads = pkg.lora_add_backward(d["dy"][:0], d["x"][:0], d["A"], d["B"], empty, sc)
    assert grads[0].shape == (0, K) and (grads[1] == 0).all() and (grads[2] == 0).all()


@pytest.mark.gpu
def test_large_offsets(pkg):
    """Rows of x and y, and an adapter, that lie beyond 2^32 bytes of their base."""
    T, n, r, K, N = 70000, 2, 8, 32768, 32768
    x = torch.empty(T, K, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 1, 40000, 65536, 69999])
    ids = torch.full((T,), -1)
    ids[rows] = torch.tensor([0, 1, 1, 0, 1])
    g = torch.Generator().manual_seed(1)
    A = (torch.randn(n, r, K, generator=g) * K ** -0.5).to(torch.bfloat16)
    B = torch.randn(n, N, r, generator=g).to(torch.bfloat16)
    some = torch.randn(len(rows), K, generator=g).to(torch.bfloat16)
    x[rows.cuda()] = some.cuda()
    y = torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")
    plan = pkg.adapter_plan(ids.cuda(), n)
    pkg.lora_add(y, x, A.cuda(), B.cuda(), plan, inplace=True)
    c = dict(x=some, A=A, B=B, y=torch.zeros(len(rows), N, dtype=torch.bfloat16), ids=ids[rows])
    want, _, slack, _ = forward64(c, "bf16", scales=False)
    within(y[rows.cuda()], want, slack)
    y[rows.cuda()] = 0
    assert not y.any()


@pytest.mark.gpu
def test_streams_and_two_graphs(pkg):
    T, n, r, K, N = 600, 4, 16, 256, 512
    cases = [make(T, n, r, K, N, "bf16", "mixed", seed=s) for s in (31, 32, 33)]
    d = on_gpu(cases[0])

    def step():
        plan = pkg.adapter_plan(d["ids"], n)
        out, u = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, d["scales"], return_shrunk=True)
        return (out, u, *pkg.lora_add_backward(out, d["x"], d["A"], d["B"], plan, d["scales"], shrunk=u))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for turn in range(4):
        for c in cases:
            for k, v in c.items():
                d[k].copy_(v)
            graphs[turn % 2].replay()
            eager = step()
            torch.cuda.synchronize()
            for a, b in zip(outs[turn % 2], eager):
                assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------
# refusals, on the CPU

class _Plan:
    def __init__(self, tokens, n):
        self.buffer, self.tokens, self.n_adapters = torch.zeros(1, dtype=torch.int32), tokens, n


def _cpu(T=4, n=2, r=8, K=32, N=24, dtype=torch.bfloat16):
    return dict(y=torch.zeros(T, N, dtype=dtype), x=torch.zeros(T, K, dtype=dtype), A=torch.zeros(n, r, K, dtype=dtype),
                B=torch.zeros(n, N, r, dtype=dtype), plan=_Plan(T, n), scales=torch.ones(n))


@pytest.mark.parametrize("sizes,change,match", [
    ({}, dict(y=torch.zeros(4, 24, 1, dtype=torch.bfloat16)), "dimensions"),
    ({}, dict(x=torch.zeros(4, 32)), "share a dtype"),
    (dict(dtype=torch.float64), {}, "share a dtype"),
    ({}, dict(x=torch.zeros(5, 32, dtype=torch.bfloat16)), "shape mismatch"),
    ({}, dict(B=torch.zeros(2, 8, 24, dtype=torch.bfloat16)), "shape mismatch"),
    (dict(r=4), {}, "rank"),
    (dict(r=136), {}, "rank"),
    (dict(K=36), {}, "widths"),
    (dict(N=20), {}, "widths"),
    ({}, dict(plan=_Plan(5, 2)), "the plan is for"),
    ({}, dict(plan=_Plan(4, 3)), "the plan is for"),
    ({}, dict(scales=torch.ones(2, dtype=torch.bfloat16)), "scales"),
    ({}, dict(scales=torch.ones(3)), "scales"),
    ({}, {}, "GPU tensor"),
])
def test_refusals(pkg, sizes, change, match):
    args = {**_cpu(**sizes), **change}
    for f in (pkg.lora_add, pkg.lora_add_backward):
        with pytest.raises(RuntimeError, match=match):
            f(*args.values())


def test_plan_refusals(pkg):
    ids = torch.zeros(4, dtype=torch.int32)
    for bad, n, match in ((ids.float(), 2, "int32 or int64"), (ids.view(2, 2), 2, "int32 or int64"), (ids, 0, "n_adapters"),
                          (ids, 1025, "n_adapters"), (ids, 2, "GPU tensor")):
        with pytest.raises(RuntimeError, match=match):
            pkg.adapter_plan(bad, n)
    with pytest.raises(RuntimeError, match="at most"):
        pkg.adapter_plan(ids[:1].expand((1 << 24) + 1), 2)


def test_c_entry_refusals(pkg):
    import importlib
    lib = importlib.import_module(pkg.__name__ + "._lib").load()
    pack = importlib.import_module(pkg.__name__ + ".adapters")._LORA.pack
    DTYPE, SIZE, ALIGN, NULL, SHAPE, _, ALIAS = range(-1, -8, -1)
    p, q = 1 << 20, 1 << 21  # never followed: every call is refused or has nothing to do

    def sizes(T=4, xs=32, ys=24, os=32, n=2, r=8, K=32, N=24, dt=1):
        return pack(T, xs, ys, os, n, r, K, N, dt)

    def fwd(d, y=p, x=p, scales=None, plan=p, out=q, shrunk=None, ws=p):
        return lib.mi_lora_add(y, x, p, p, scales, plan, out, shrunk, ws, d, None)

    def bwd(d, y=p, x=p, scales=None, plan=p, out=q, shrunk=None, ws=p):
        return lib.mi_lora_add_backward(y, x, p, p, scales, plan, shrunk, None, out, p, p, ws, d, None)

    for f in (fwd, bwd):
        assert f(None) == NULL and f(sizes(dt=5)) == DTYPE
        assert f(sizes(r=4)) == SIZE and f(sizes(r=136)) == SIZE and f(sizes(r=12)) == SIZE
        for bad in (dict(T=(1 << 24) + 1), dict(n=0), dict(n=1025), dict(K=12), dict(K=0), dict(N=4), dict(N=(1 << 22) + 8)):
            assert f(sizes(**bad)) == SHAPE, bad
            assert lib.mi_lora_workspace(sizes(**bad), 0) == 0
        assert f(sizes(xs=33)) == ALIGN and f(sizes(ys=28)) == ALIGN and f(sizes(os=26)) == ALIGN
        assert f(sizes(xs=36, ys=28, os=36, dt=0), plan=None) == NULL
        for bad in ("y", "x", "plan", "out", "ws"):
            assert f(sizes(), **{bad: None}) == NULL, bad
            assert f(sizes(), **{bad: p + 8}) == ALIGN, bad
        assert f(sizes(), scales=p + 2) == ALIGN and f(sizes(), shrunk=p + 2) == ALIGN
    assert bwd(sizes(n=1024, r=128, K=1 << 18, xs=1 << 18, os=1 << 18)) == SHAPE  # 2^35 values of A
    assert fwd(sizes(os=16)) == SHAPE and bwd(sizes(os=24)) == SHAPE  # rows of the output would overlap
    assert fwd(sizes(T=0), y=None) == 0
    assert fwd(sizes(ys=24), y=p, out=p) == ALIAS
    assert lib.mi_lora_workspace(sizes(), 0) > 0 and lib.mi_lora_workspace(sizes(), 1) > lib.mi_lora_workspace(sizes(), 0)
    assert lib.mi_lora_workspace(None, 0) == 0
    out = (ctypes.c_uint64 * 3)()
    assert lib.mi_adapter_plan_layout(4, 2, None) == NULL and lib.mi_adapter_plan_layout(4, 0, out) == SHAPE
    assert lib.mi_adapter_plan_layout((1 << 24) + 1, 2, out) == SHAPE and lib.mi_adapter_plan_layout(100, 3, out) == 0
    assert out[1] + 100 == out[2] and out[2] + 4 <= out[0]
    assert lib.mi_adapter_plan(p, 16, 4, 2, p, None) == DTYPE and lib.mi_adapter_plan(p, 32, 4, 1025, p, None) == SHAPE
    assert lib.mi_adapter_plan(None, 32, 4, 2, p, None) == NULL and lib.mi_adapter_plan(p, 32, 4, 2, None, None) == NULL
    assert lib.mi_adapter_plan(p, 32, 4, 2, p + 4, None) == ALIGN and lib.mi_adapter_plan(p + 4, 64, 4, 2, p, None) == ALIGN


# ---------------------------------------------------------------------------------------------
# calls at the edge of what is allowed

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_input_gradient_written_over_the_input(pkg, dtype):
    """``dx`` may be ``x`` itself: dA is of the input as it was."""
    T, n, r, K, N = 300, 2, 16, 264, 136
    c = make(T, n, r, K, N, dtype, "mixed", seed=12)
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], n)
    args = (d["A"], d["B"], plan, d["scales"])
    want = pkg.lora_add_backward(d["dy"], d["x"], *args, dx=d["x"].clone())
    x = d["x"].clone()
    got = pkg.lora_add_backward(d["dy"], x, *args, dx=x)
    assert got[0] is x
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,r,K,N,dtype,ids", [(4200, 3, 16, 72, 8200, "bf16", "runs"), (4200, 3, 40, 72, 8200, "fp16", "mixed"),
                                                 (4200, 2, 8, 72, 4104, "fp32", "mixed")])
def test_backward_of_an_output_larger_than_the_caches_keep(pkg, T, n, r, K, N, dtype, ids):
    c = make(T, n, r, K, N, dtype, ids, seed=T + r)
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], n)
    got = pkg.lora_add_backward(d["dy"], d["x"], d["A"], d["B"], plan, d["scales"])
    gx, dA, dB, gx_slack, dA_slack, dB_slack = backward64(c, dtype)
    within(got[0], gx, gx_slack, "dx")
    within(got[1], dA, dA_slack, "dA")
    within(got[2], dB, dB_slack, "dB")
