"""GPU tests of ``qk_norm_rope`` and its backward pass against the definition in fp64.

Tolerances.  An output is rounded once to its type: at most half a step, ``finfo.eps / 2`` of the value
(bf16 2^-8, fp16 2^-11, fp32 2^-24; below the smallest normal number half the subnormal spacing).  What
comes before it is fp32, u = 2^-24: a sum of squares of D <= 512 values over 16 in a lane and 5 steps
across lanes (21 u, halved by the root), root, quotient and two products (5 u), sine and cosine (within
2^-22 of exact, 4 u, plus 2 u of the reduced angle), a rotation (3 u), and at most 9 butterfly stages
(9 u of the norm of the row): below 48 u of the row's norm, taken as 64 u.  Backwards the row passes the
same maps and two sums: 96 u of the sum of the terms' magnitudes.  A weight gradient adds one product
for every token and head on top: 96 u for each term and one u per addition in a row, of which a lane
makes at most tokens * ceil(heads / 2), and 20 of the trees.
"""
import itertools
import math

import pytest
import torch

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def hadamard64(n):
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.size(0) < n:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(n)


def pair_matrices(positions, inv_freq, sections, R, interleaved):
    """cos, sin [T, R/2] in fp64 and the pair members' indices."""
    pos = positions.double().reshape(-1, positions.shape[-1])
    owner = [a for a, c in enumerate(sections or (R // 2,)) for _ in range(c)]
    angle = pos[owner].T * inv_freq.double() if R else torch.zeros(positions.shape[-1], 0, dtype=torch.float64)
    i = torch.arange(R // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    return torch.cos(angle), torch.sin(angle), first, second


def forward64(x, w, rot, eps, hadamard):
    cos, sin, first, second = rot
    x = x.double()
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        n = n * w.double()
    out = n.clone()
    c, s = cos[:, None, :], sin[:, None, :]
    out[..., first] = n[..., first] * c - n[..., second] * s
    out[..., second] = n[..., second] * c + n[..., first] * s
    return out @ hadamard64(x.shape[-1]) if hadamard else out


def backward64(x, w, g, rot, eps, hadamard):
    """dx, dw and the magnitudes their rounding errors scale with."""
    cos, sin, first, second = rot
    x, g = x.double(), g.double()
    if hadamard:
        g = g @ hadamard64(x.shape[-1])
    b = g.clone()
    c, s = cos[:, None, :], sin[:, None, :]
    b[..., first] = g[..., first] * c + g[..., second] * s
    b[..., second] = g[..., second] * c - g[..., first] * s
    rho = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * rho
    wv = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    t = b * wv
    dx = rho * (t - n * (t * n).mean(-1, keepdim=True))
    row = t.norm(dim=-1, keepdim=True) + b.norm(dim=-1, keepdim=True) * wv.abs().max()
    dx_mag = rho * (row + n.abs() * row * n.norm(dim=-1, keepdim=True) / x.shape[-1])
    dw = (b * n).sum((0, 1))
    dw_mag = (b.norm(dim=-1, keepdim=True) * n.abs()).sum((0, 1))
    return dx, dw, dx_mag, dw_mag


def within(got, want, slack):
    """|got - want| <= half a step of got's type + slack, element by element."""
    f = torch.finfo(got.dtype)
    tol = want.abs() * f.eps / 2 + f.tiny * f.eps / 2 + slack
    err = (got.cpu().double() - want).abs()
    assert got.shape == want.shape
    worst = (err / tol.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert (err <= tol).all(), f"worst error {worst} of the bound"


def make(T, Hq, Hk, D, R, dtype, axes=1, seed=0, pos64=False, freq64=False, far=4096):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    qkv = (torch.randn(T, (Hq + 2 * Hk) * D, generator=g) * 1.5).to(dt)
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dt) for _ in range(2)]
    pos = torch.randint(-3, far, (T,) if axes == 1 else (axes, T), generator=g, dtype=torch.int64)
    freq = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))
    sections = None
    if axes > 1:
        cut = [R // 2 * a // (axes + 1) for a in range(1, axes)]
        sections = tuple(b - a for a, b in zip([0, *cut], [*cut, R // 2]))
    return qkv, w, pos if pos64 else pos.to(torch.int32), freq if freq64 else freq.float(), sections


def split(qkv, Hq, Hk, D):
    return (qkv[:, :Hq * D].unflatten(1, (Hq, D)), qkv[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D)))


CASES = [
    # T, Hq, Hk, D, R, dtype, axes, interleaved, hadamard
    (1, 32, 8, 128, 128, "bf16", 1, False, True),
    (1, 1, 1, 64, 64, "fp32", 1, False, False),
    (3, 5, 3, 64, 64, "bf16", 1, True, True),
    (7, 20, 4, 80, 80, "fp16", 3, False, False),
    (5, 3, 1, 96, 48, "bf16", 2, False, False),
    (9, 4, 2, 128, 64, "fp16", 1, False, True),
    (9, 4, 2, 128, 64, "fp32", 1, True, True),
    (6, 9, 2, 256, 64, "fp32", 4, False, True),
    (4, 3, 2, 512, 512, "bf16", 1, False, True),
    (4, 3, 2, 512, 128, "fp16", 1, False, True),
    (4, 3, 2, 512, 496, "fp32", 1, False, False),
    (5, 2, 1, 16, 16, "bf16", 1, False, True),
    (5, 17, 33, 32, 16, "fp32", 1, False, True),
    (5, 2, 1, 32, 0, "fp16", 1, False, True),
    (33, 7, 1, 112, 112, "bf16", 1, True, False),
    (1023, 2, 1, 64, 64, "bf16", 1, False, True),
    (1024, 2, 1, 64, 32, "fp16", 3, False, True),
    (1027, 9, 2, 128, 128, "fp32", 1, False, False),
    (8200, 3, 1, 48, 32, "bf16", 1, False, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,Hq,Hk,D,R,dtype,axes,interleaved,hadamard", CASES)
def test_forward_against_the_definition(pkg, T, Hq, Hk, D, R, dtype, axes, interleaved, hadamard):
    qkv, w, pos, freq, sections = make(T, Hq, Hk, D, R, dtype, axes, seed=T + D, pos64=T % 2 == 0, freq64=T % 3 == 0)
    q, k = split(qkv, Hq, Hk, D)
    dev = qkv.cuda()
    qd, kd = split(dev, Hq, Hk, D)
    before = dev.clone()
    out = pkg.qk_norm_rope(qd, kd, w[0].cuda(), w[1].cuda(), pos.cuda(), freq.cuda(), eps=1e-5, sections=sections,
                           interleaved=interleaved, hadamard=hadamard)
    rot = pair_matrices(pos, freq, sections, R, interleaved)
    for o, x, ww in zip(out, (q, k), w):
        want = forward64(x, ww, rot, 1e-5, hadamard)
        assert o.dtype == x.dtype and o.is_contiguous()
        within(o, want, 64 * U * want.norm(dim=-1, keepdim=True))
    assert torch.equal(dev, before)
    # in place: the same values, and the value heads behind them stay as they were
    res = pkg.qk_norm_rope(qd, kd, w[0].cuda(), w[1].cuda(), pos.cuda(), freq.cuda(), eps=1e-5, sections=sections,
                           interleaved=interleaved, hadamard=hadamard, inplace=True)
    assert res[0] is qd and res[1] is kd
    assert torch.equal(qd, out[0]) and torch.equal(kd, out[1])
    assert torch.equal(dev[:, (Hq + Hk) * D:], before[:, (Hq + Hk) * D:])


@pytest.mark.gpu
@pytest.mark.parametrize("T,Hq,Hk,D,R,dtype,axes,interleaved,hadamard", CASES)
def test_backward_against_the_formula(pkg, T, Hq, Hk, D, R, dtype, axes, interleaved, hadamard):
    qkv, w, pos, freq, sections = make(T, Hq, Hk, D, R, dtype, axes, seed=T + D + 1)
    q, k = split(qkv, Hq, Hk, D)
    gen = torch.Generator().manual_seed(5)
    grads = [(torch.randn(x.shape, generator=gen) * 0.1).to(x.dtype) for x in (q, k)]
    qd, kd = split(qkv.cuda(), Hq, Hk, D)
    args = (grads[0].cuda(), grads[1].cuda(), qd, kd, w[0].cuda(), w[1].cuda(), pos.cuda(), freq.cuda())
    opts = dict(eps=1e-5, sections=sections, interleaved=interleaved, hadamard=hadamard)
    got = pkg.qk_norm_rope_backward(*args, **opts)
    again = pkg.qk_norm_rope_backward(*args, **opts)
    rot = pair_matrices(pos, freq, sections, R, interleaved)
    for i, (x, ww, g, H) in enumerate(zip((q, k), w, grads, (Hq, Hk))):
        dx, dw, dx_mag, dw_mag = backward64(x, ww, g, rot, 1e-5, hadamard)
        within(got[i], dx, 96 * U * dx_mag)
        within(got[2 + i], dw, (96 + T * ((H + 1) // 2) + 20) * U * dw_mag)
        assert torch.equal(got[i], again[i]) and torch.equal(got[2 + i], again[2 + i])


@pytest.mark.gpu
def test_backward_against_differences(pkg):
    """Central differences of the kernel's own forward in fp32: step h, error h^2 * third derivative
    plus rounding / h; both are below 2e-3 of the largest gradient at these sizes."""
    T, Hq, Hk, D, R = 2, 1, 1, 32, 16
    qkv, w, pos, freq, _ = make(T, Hq, Hk, D, R, "fp32", seed=3)
    qd, kd = split(qkv.cuda(), Hq, Hk, D)
    w = [t.cuda() for t in w]
    gen = torch.Generator().manual_seed(4)
    gq, gk = (torch.randn(T, 1, D, generator=gen).cuda() for _ in range(2))

    def loss(q, wq):
        out = pkg.qk_norm_rope(q, kd, wq, w[1], pos.cuda(), freq.cuda(), hadamard=True)
        return (out[0].double() * gq.double()).sum().item()

    dq, _, dwq, _ = pkg.qk_norm_rope_backward(gq, gk, qd, kd, w[0], w[1], pos.cuda(), freq.cuda(), hadamard=True)
    h = 2.0 ** -8
    for target, grad in ((qd.contiguous(), dq), (w[0], dwq)):
        flat = target.flatten()
        for i in range(0, flat.numel(), 7):
            step = torch.zeros_like(flat)
            step[i] = h
            up, down = (flat + step).view(target.shape), (flat - step).view(target.shape)
            if target.dim() == 3:
                slope = (loss(up, w[0]) - loss(down, w[0])) / (2 * h)
            else:
                slope = (loss(qd, up) - loss(qd, down)) / (2 * h)
            assert abs(slope - grad.flatten()[i].item()) <= 2e-3 * max(1.0, grad.abs().max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("freq64", [False, True])
def test_far_positions(pkg, freq64):
    pos = torch.tensor([2 ** 31 - 1, 2 ** 24 + 1, 1_000_003, -(2 ** 31), 131071], dtype=torch.int64)
    T, D = len(pos), 64
    qkv, w, _, freq, _ = make(T, 2, 1, D, D, "fp32", freq64=freq64, seed=8)
    q, k = split(qkv, 2, 1, D)
    qd, kd = split(qkv.cuda(), 2, 1, D)
    out = pkg.qk_norm_rope(qd, kd, None, None, pos.cuda(), freq.cuda())
    # a product of 2^31 radians is rounded to 2^-22 in fp64 here and in the definition alike
    slack = 64 * U + (2 * pos.abs().double() * 2.0 ** -52)[:, None, None]
    want = forward64(q, None, pair_matrices(pos, freq, None, D, False), 1e-6, False)
    within(out[0], want, slack * want.norm(dim=-1, keepdim=True))


@pytest.mark.gpu
def test_zero_rows_infinities_and_nan_stay_in_their_head(pkg):
    T, Hq, Hk, D, R = 6, 3, 2, 64, 32
    qkv, w, pos, freq, _ = make(T, Hq, Hk, D, R, "bf16", seed=9)
    clean = split(qkv.cuda(), Hq, Hk, D)
    args = (w[0].cuda(), w[1].cuda(), pos.cuda(), freq.cuda())
    ref = pkg.qk_norm_rope(*clean, *args)
    bad = qkv.clone()
    bq, bk = split(bad, Hq, Hk, D)
    bq[1, 0] = 0.0
    bq[2, 1, 40] = float("nan")
    bk[3, 1, 5] = float("inf")
    out = pkg.qk_norm_rope(*split(bad.cuda(), Hq, Hk, D), *args)
    assert (out[0][1, 0] == 0).all()
    assert out[0][2, 1].isnan().all()  # the mean is NaN
    assert out[1][3, 1, 5].isnan()     # inf * 0
    others = (out[1][3, 1].isnan() | (out[1][3, 1] == 0)).cpu()
    partner = torch.zeros(D, dtype=torch.bool)
    partner[[5, 5 + R // 2]] = True
    assert others.all() and (out[1][3, 1].isnan().cpu() == partner).all()
    keep_q = torch.ones(T, Hq, dtype=torch.bool)
    keep_q[1, 0] = keep_q[2, 1] = False
    keep_k = torch.ones(T, Hk, dtype=torch.bool)
    keep_k[3, 1] = False
    assert torch.equal(out[0].cpu()[keep_q], ref[0].cpu()[keep_q])
    assert torch.equal(out[1].cpu()[keep_k], ref[1].cpu()[keep_k])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_operand_layouts(pkg, dtype):
    """Views, strides the kernels do not take (copied), empty batches and head counts, fp32 weights."""
    T, Hq, Hk, D = 5, 4, 2, 32
    qkv, w, pos, freq, _ = make(T, Hq, Hk, D, D, dtype, seed=12)
    dev = qkv.cuda()
    q, k = (t.contiguous() for t in split(dev, Hq, Hk, D))
    wq, wk, pos, freq = w[0].cuda(), w[1].cuda(), pos.cuda(), freq.cuda()
    ref = pkg.qk_norm_rope(q, k, wq, wk, pos, freq)
    # one element off the alignment, heads before tokens, and a strided last axis
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    gaps = torch.zeros(T, Hq, 2 * D, dtype=q.dtype, device="cuda")[..., ::2].copy_(q)
    for other in (odd, turned, gaps):
        assert torch.equal(pkg.qk_norm_rope(other, k, wq, wk, pos, freq)[0], ref[0])
        res = pkg.qk_norm_rope(other, k.clone(), wq, wk, pos, freq, inplace=True)
        assert res[0] is other and torch.equal(other, ref[0]) and torch.equal(res[1], ref[1])
    one = q[:1].expand(T, Hq, D)
    same = pkg.qk_norm_rope(one, k, wq, wk, pos, freq)[0]
    assert torch.equal(same, pkg.qk_norm_rope(one.contiguous(), k, wq, wk, pos, freq)[0])
    with pytest.raises(RuntimeError, match="share memory"):
        pkg.qk_norm_rope(one, k, wq, wk, pos, freq, inplace=True)
    # positions and weights that are views, fp32 weights beside 16-bit heads
    wide = torch.stack([pos, pos], 1)[:, 0]
    assert torch.equal(pkg.qk_norm_rope(q, k, wq.float(), wk.float(), wide, freq)[0], ref[0])
    # empty: no tokens, no key heads
    none = pkg.qk_norm_rope(q[:0], k[:0], wq, wk, pos[:0], freq)
    assert none[0].shape == (0, Hq, D) and none[1].shape == (0, Hk, D)
    grads = pkg.qk_norm_rope_backward(q[:0], k[:0], q[:0], k[:0], wq, wk, pos[:0], freq)
    assert (grads[2] == 0).all() and (grads[3] == 0).all() and grads[2].dtype == wq.dtype
    only_q = pkg.qk_norm_rope(q, k[:, :0], wq, None, pos, freq)
    assert torch.equal(only_q[0], ref[0]) and only_q[1].shape == (T, 0, D)
    full = pkg.qk_norm_rope_backward(q, k, q, k, wq, wk, pos, freq)
    part = pkg.qk_norm_rope_backward(q, k, q, k, wq, None, pos, freq)
    assert torch.equal(full[0], part[0]) and torch.equal(full[2], part[2]) and part[3] is None
    alone = pkg.qk_norm_rope_backward(q, k[:, :0], q, k[:, :0], wq, wk, pos, freq)
    assert torch.equal(full[0], alone[0]) and torch.equal(full[2], alone[2]) and (alone[3] == 0).all()


@pytest.mark.gpu
def test_one_token_of_very_many_heads(pkg):
    """A token's heads shared by as many workgroups as the pass has at most."""
    T, Hq, Hk, D = 1, 40000, 3, 16
    qkv, w, pos, freq, _ = make(T, Hq, Hk, D, D, "bf16", seed=15)
    q, k = split(qkv, Hq, Hk, D)
    qd, kd = split(qkv.cuda(), Hq, Hk, D)
    args = (w[0].cuda(), w[1].cuda(), pos.cuda(), freq.cuda())
    rot = pair_matrices(pos, freq, None, D, False)
    out = pkg.qk_norm_rope(qd, kd, *args)
    want = forward64(q, w[0], rot, 1e-6, False)
    within(out[0], want, 64 * U * want.norm(dim=-1, keepdim=True))
    g = (torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(1)) * 0.1).to(torch.bfloat16)
    got = pkg.qk_norm_rope_backward(g.cuda(), torch.zeros_like(kd), qd, kd, *args)
    dx, dw, dx_mag, dw_mag = backward64(q, w[0], g, rot, 1e-6, False)
    within(got[0], dx, 96 * U * dx_mag)
    within(got[2], dw, (96 + Hq // 2 + 20) * U * dw_mag)
    assert (got[3] == 0).all()


@pytest.mark.gpu
def test_rows_behind_a_view_are_left_alone(pkg):
    """In place on the first tokens of a larger buffer: what lies behind and between stays."""
    T, Hq, Hk, D = 6, 2, 1, 64
    qkv, w, pos, freq, _ = make(T + 3, Hq, Hk, D, D, "bf16", seed=13)
    dev = qkv.cuda()
    before = dev.clone()
    q, k = split(dev[:T], Hq, Hk, D)
    pkg.qk_norm_rope(q, k, w[0].cuda(), w[1].cuda(), pos[:T].cuda(), freq.cuda(), inplace=True)
    assert torch.equal(dev[T:], before[T:]) and torch.equal(dev[:, (Hq + Hk) * D:], before[:, (Hq + Hk) * D:])
    assert not torch.equal(dev[:T, :D], before[:T, :D])


@pytest.mark.gpu
def test_hadamard_option_is_the_packages_transform(pkg):
    """The fused rotation against the stand-alone transform of the un-rotated fp32 output; scores of
    queries with keys do not change (both are orthogonal up to fp32 rounding)."""
    T, Hq, Hk, D = 12, 4, 4, 128
    qkv, w, pos, freq, _ = make(T, Hq, Hk, D, D, "fp32", seed=14)
    q, k = split(qkv.cuda(), Hq, Hk, D)
    args = (w[0].cuda(), w[1].cuda(), pos.cuda(), freq.cuda())
    plain = pkg.qk_norm_rope(q, k, *args)
    turned = pkg.qk_norm_rope(q, k, *args, hadamard=True)
    for a, b in zip(plain, turned):
        ht = pkg.hadamard_transform(a)
        # 7 stages each side, u of the row's norm per stage
        assert ((ht - b).abs() <= 32 * U * a.norm(dim=-1, keepdim=True)).all()
    s0 = (plain[0].double()[:, None] * plain[1].double()[None]).sum(-1)
    s1 = (turned[0].double()[:, None] * turned[1].double()[None]).sum(-1)
    bound = plain[0].double().norm(dim=-1)[:, None] * plain[1].double().norm(dim=-1)[None]
    assert ((s0 - s1).abs() <= 128 * U * bound).all()


@pytest.mark.gpu
def test_streams_and_graph_replays(pkg):
    T, Hq, Hk, D = 300, 4, 2, 128
    sets = [make(T, Hq, Hk, D, D, "bf16", seed=s) for s in (20, 21, 22)]
    w, freq = [t.cuda() for t in sets[0][1]], sets[0][3].cuda()
    buf, pos = sets[0][0].cuda(), sets[0][2].cuda()
    q, k = split(buf, Hq, Hk, D)

    def both():
        out = pkg.qk_norm_rope(q, k, *w, pos, freq, hadamard=True)
        return (*out, *pkg.qk_norm_rope_backward(*out, q, k, *w, pos, freq, hadamard=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both())
        graphs.append(g)
    for turn in range(3):
        for s in sets:
            buf.copy_(s[0])
            pos.copy_(s[2])
            graphs[turn % 2].replay()
            eager = both()
            torch.cuda.synchronize()
            for a, b in zip(outs[turn % 2], eager):
                assert torch.equal(a, b)


def _cpu_args(dtype=torch.bfloat16, T=4, Hq=2, Hk=1, D=64, R=64):
    return dict(q=torch.zeros(T, Hq, D, dtype=dtype), k=torch.zeros(T, Hk, D, dtype=dtype),
                q_weight=torch.ones(D, dtype=dtype), k_weight=torch.ones(D, dtype=dtype),
                positions=torch.zeros(T, dtype=torch.int32), inv_freq=torch.ones(R // 2))


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(4, 128, dtype=torch.bfloat16)), "must be"),
    (dict(q=torch.zeros(4, 2, 64, dtype=torch.float64)), "share a dtype"),
    (dict(k=torch.zeros(4, 1, 64)), "share a dtype"),
    (dict(k=torch.zeros(5, 1, 64, dtype=torch.bfloat16)), "shape mismatch"),
    (dict(q=torch.zeros(4, 2, 72, dtype=torch.bfloat16), k=torch.zeros(4, 1, 72, dtype=torch.bfloat16)), "multiple of 16"),
    (dict(q=torch.zeros(4, 2, 528, dtype=torch.bfloat16), k=torch.zeros(4, 1, 528, dtype=torch.bfloat16)), "multiple of 16"),
    (dict(inv_freq=torch.ones(12)), "multiple of 8"),
    (dict(inv_freq=torch.ones(40)), "at most"),
    (dict(inv_freq=torch.ones(32, dtype=torch.bfloat16)), "fp32 or fp64"),
    (dict(positions=torch.zeros(4)), "int32 or int64"),
    (dict(positions=torch.zeros(5, dtype=torch.int32)), "positions must be"),
    (dict(positions=torch.zeros(5, 4, dtype=torch.int32)), "up to four axes"),
    (dict(positions=torch.zeros(2, 4, dtype=torch.int32)), "need sections"),
    (dict(sections=(16, 16)), "sections"),
    (dict(sections=(40, -8), positions=torch.zeros(2, 4, dtype=torch.int32)), "negative"),
    (dict(sections=(16, 8), positions=torch.zeros(2, 4, dtype=torch.int32)), "share of"),
    (dict(q_weight=torch.ones(32, dtype=torch.bfloat16)), "64 entries"),
    (dict(q_weight=torch.ones(64, dtype=torch.float16)), "heads' dtype or fp32"),
    (dict(q_weight=torch.ones(64)), "share a dtype"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(), "GPU tensor"),
])
def test_refusals(pkg, change, match):
    args = {**_cpu_args(), **change}
    opts = {n: args.pop(n) for n in ("sections", "eps") if n in args}
    with pytest.raises(RuntimeError, match=match):
        pkg.qk_norm_rope(*args.values(), **opts)
    with pytest.raises(RuntimeError, match=match):
        pkg.qk_norm_rope_backward(args["q"], args["k"], *args.values(), **opts)


def test_hadamard_refuses_other_head_sizes(pkg):
    args = _cpu_args(D=48, R=48)
    with pytest.raises(RuntimeError, match="power-of-two"):
        pkg.qk_norm_rope(*args.values(), hadamard=True)


def test_c_entry_refusals(pkg):
    import importlib
    lib = importlib.import_module(pkg.__name__ + "._lib").load()
    heads = importlib.import_module(pkg.__name__ + ".heads")
    DTYPE, SIZE, ALIGN, NULL, SHAPE = range(-1, -6, -1)
    p = 1 << 20  # an address that is never followed: every call is refused, or has nothing to do

    def desc(T=4, ts=(128, 64, 128, 64, 128, 64), hs=(64,) * 6, Hq=2, Hk=1, D=64, R=64, axes=1, ends=(32, 0, 0, 0),
             dt=1, wdt=1, pb=32, fb=32, flags=0, eps=1e-6):
        return heads._HEADS.pack(T, *ts, *hs, Hq, Hk, D, R, axes, *ends, dt, wdt, pb, fb, flags, eps)

    def call(d, q=p, w=p, pos=p, out=p):
        return lib.mi_qk_norm_rope(q, p, w, p, pos, p, out, p, d, None)

    def back(d, q=p, ws=p, pos=p):
        return lib.mi_qk_norm_rope_backward(q, p, p, p, p, p, pos, p, p, p, p, p, ws, d, None)

    for f in (call, back):
        assert f(None) == NULL
        assert f(desc(dt=7)) == DTYPE and f(desc(wdt=2)) == DTYPE
        assert f(desc(pb=16)) == DTYPE and f(desc(fb=16)) == DTYPE
        assert f(desc(D=72)) == SIZE and f(desc(D=8)) == SIZE and f(desc(D=528)) == SIZE
        assert f(desc(R=24, ends=(12, 0, 0, 0))) == SIZE and f(desc(R=80, ends=(40, 0, 0, 0))) == SIZE
        assert f(desc(D=48, R=48, ends=(24, 0, 0, 0), flags=2)) == SIZE
        assert f(desc(flags=4)) == SHAPE
        assert f(desc(axes=0)) == SHAPE and f(desc(axes=5)) == SHAPE
        assert f(desc(ends=(31, 0, 0, 0))) == SHAPE and f(desc(axes=2, ends=(32, 16, 0, 0))) == SHAPE
        assert f(desc(eps=-1.0)) == SHAPE and f(desc(eps=float("nan"))) == SHAPE
        assert f(desc(Hq=65537)) == SHAPE and f(desc(T=1 << 40)) == SHAPE
        assert f(desc(), q=None) == NULL and f(desc(), pos=None) == NULL
        assert f(desc(), q=p + 2) == ALIGN and f(desc(), pos=p + 2) == ALIGN and f(desc(pb=64), pos=p + 4) == ALIGN
        assert f(desc(ts=(128, 64, 48, 64, 48, 64))) == SHAPE and f(desc(hs=(64, 64, 0, 64, 0, 64))) == SHAPE  # outputs overlap
        assert f(desc(ts=(129, 64, 128, 64, 128, 64))) == ALIGN and f(desc(hs=(64, 65, 64, 64, 64, 64))) == ALIGN
    assert call(desc(), w=p + 2) == ALIGN and back(desc(), ws=None) == NULL and back(desc(), ws=p + 4) == ALIGN
    assert call(desc(T=0), q=None) == 0 and call(desc(Hq=0, Hk=0), q=None) == 0
    assert lib.mi_qk_norm_rope_workspace(0, 64) == 0
    sizes = [lib.mi_qk_norm_rope_workspace(t, 64) for t in (1, 1023, 1024, 4096, 1 << 39)]
    assert all(0 < s <= 1024 * 64 * 4 for s in sizes)


def test_differentiable_inputs_are_refused_under_grad_mode(pkg):
    args = _cpu_args()
    args["q"] = args["q"].float().requires_grad_()
    for n in ("k", "q_weight", "k_weight"):
        args[n] = args[n].float()
    # the device is checked first; the rule itself needs no device
    import importlib
    ops = importlib.import_module(pkg.__name__ + ".ops")
    with pytest.raises(RuntimeError, match="no autograd graph"):
        ops._no_graph("qk_norm_rope", args["q"], None)
    with torch.no_grad():
        ops._no_graph("qk_norm_rope", args["q"], None)


def test_lane_layout_covers_every_value_once():
    """The lane and unit arithmetic of the kernels, restated: for every head size, rotary width and pair
    order each eight-value unit has one owner, pairs share a lane, and mirrors of Gray-coded lanes
    differ in one bit of the unit index."""
    for D, R, neighbours in itertools.product(range(16, 513, 16), range(0, 513, 16), (False, True)):
        if R > D:
            continue
        rl, owners = R // 16, {}
        for lane in range(D // 16):
            halves = lane < rl and not neighbours
            owners[lane] = (lane, lane + rl) if halves else (2 * lane, 2 * lane + 1)
        assert sorted(u for pair in owners.values() for u in pair) == list(range(D // 8))
        for f in range(R // 2):
            a, b = (2 * f, 2 * f + 1) if neighbours else (f, f + R // 2)
            lane = next(l for l, units in owners.items() if a // 8 in units)
            assert b // 8 in owners[lane] and lane == f // 8
    for lane in range(32):
        for bit in range(5):
            other = lane ^ ((2 << bit) - 1)
            assert (lane ^ lane >> 1) ^ (other ^ other >> 1) == 1 << bit


@pytest.mark.gpu
def test_in_place_on_one_memory_is_refused(pkg):
    q = torch.randn(4, 2, 64, device="cuda")
    pos, freq = torch.arange(4, device="cuda"), torch.rand(32, device="cuda")
    with pytest.raises(RuntimeError, match="share memory"):
        pkg.qk_norm_rope(q, q, None, None, pos, freq, inplace=True)
    same = pkg.qk_norm_rope(q, q, None, None, pos, freq)
    assert torch.equal(same[0], same[1])
