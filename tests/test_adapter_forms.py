"""Every form that ``lora_add`` and ``lora_add_backward`` take, by batch size, rank and type, against the definition in
fp64: workgroups of 16 tokens, of 64 that add up the parts of P themselves, and of 64 that read vectors made
once, each with padded ranks of 16, 32, 64 and 128.  That the cases reach them all is counted on the CPU, from the cut
that the library's own workspace sizes confirm.

Tolerances are those of the smaller cases' tests, with rank-space vectors that are whole in bf16 (as in fp32).
"""
import itertools

import pytest
import torch

from test_adapter_workspace_cpu import Cut, padded
from test_adapters_gpu import DT, backward64, forward64, make, on_gpu, within

CODE = {"fp32": 0, "bf16": 1, "fp16": 2}
EXACT_AS = {"fp32": "fp32", "bf16": "fp32", "fp16": "fp16"}


def cases():
    """(T, n, r, K, N, dtype, ids): for each type and rank one of each form, none a multiple of a tile or block."""
    for dtype in CODE:
        block = 64 if dtype == "fp32" else 128
        for r in (8, 16, 24, 40, 64, 72, 128):
            yield 333, 3, r, 9 * block + 24, 9 * block + 8, dtype, "mixed"        # 16 tokens a workgroup
            yield 1300, 3, r, 3 * block + 40, 5 * block + 24, dtype, "mixed"      # own sums
            if r == 128:  # few tokens of many adapters: too much to add up again in every workgroup
                yield 70, 60, r, 19 * block + 8, 60 * block + 8, dtype, "mixed"
            yield 4390, 7, r, 19 * block + 8, 17 * block + 40, dtype, "runs" if r == 40 else "mixed"  # vectors made once


def form(T, n, r, K, N, dtype):
    c = Cut(T, n, r, K, N, CODE[dtype])
    return "few" if c.few else "own" if c.own else "vectors"


def test_cases_reach_every_form():
    reached = {(dtype, padded(r), form(T, n, r, K, N, dtype)) for T, n, r, K, N, dtype, _ in cases()}
    assert reached == set(itertools.product(CODE, (16, 32, 64, 128), ("few", "own", "vectors")))
    for T, n, r, K, N, dtype, _ in cases():
        c = Cut(T, n, r, K, N, CODE[dtype])
        if form(T, n, r, K, N, dtype) != "own":
            assert c.splits > 1 and c.parts > 1
    # on both sides of the borders between the last two
    assert [form(70, 60, r, 19 * 128 + 8, 60 * 128 + 8, "bf16") for r in (64, 72)] == ["own", "vectors"]
    near = [form(4390, 7, 8, 19 * 128 + 8, N, "bf16") for N in range(128, 4096, 128)]
    assert near[0] == "own" and near[-1] == "vectors" and near == sorted(near)


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,r,K,N,dtype,ids", cases())
def test_forward_of_every_form(pkg, T, n, r, K, N, dtype, ids):
    c = make(T, n, r, K, N, dtype, ids, seed=T + r)
    if ids == "runs":
        c["ids"][T // 3:T // 2] = -1
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], n)
    out, u = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, d["scales"], return_shrunk=True)
    want, want_u, slack, u_slack = forward64(c, EXACT_AS[dtype])
    within(u, want_u, u_slack, "u")
    within(out, want, slack, "out")
    none = c["ids"] < 0
    assert none.any() and torch.equal(out.cpu()[none], c["y"][none]) and (u.cpu()[none] == 0).all()
    assert torch.equal(pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, d["scales"]), out)
    plain = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan)
    want, _, slack, _ = forward64(c, EXACT_AS[dtype], scales=False)
    within(plain, want, slack, "no scales")
    same = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, d["scales"], inplace=True)
    assert same is d["y"] and torch.equal(same, out)


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,r,K,N,dtype,ids", cases())
def test_backward_of_every_form(pkg, T, n, r, K, N, dtype, ids):
    c = make(T, n, r, K, N, dtype, ids, seed=T + r + 1)
    if ids == "runs":
        c["ids"][T // 3:T // 2] = -1
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], n)
    _, u = pkg.lora_add(d["y"], d["x"], d["A"], d["B"], plan, d["scales"], return_shrunk=True)
    args = (d["dy"], d["x"], d["A"], d["B"], plan, d["scales"])
    got = pkg.lora_add_backward(*args, shrunk=u)
    gx, dA, dB, gx_slack, dA_slack, dB_slack = backward64(c, EXACT_AS[dtype])
    within(got[0], gx, gx_slack, "dx")
    within(got[1], dA, dA_slack, "dA")
    within(got[2], dB, dB_slack, "dB")
    assert (got[0].cpu()[c["ids"] < 0] == 0).all()
    for _ in range(2):  # u computed again; the same bits every time
        for a, b in zip(got, pkg.lora_add_backward(*args)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("n,chunk", [(20, 128), (18, 256)])
def test_backward_with_a_token_beyond_a_chunk_each(pkg, n, chunk):
    """As many partial rows as a batch can have: every adapter has one chunk and a token."""
    r, K, N, T = 16, 136, 520, n * (chunk + 1)
    c = make(T, n, r, K, N, "bf16", seed=n)
    c["ids"] = torch.arange(T) % n
    d = on_gpu(c)
    plan = pkg.adapter_plan(d["ids"], n)
    got = pkg.lora_add_backward(d["dy"], d["x"], d["A"], d["B"], plan, d["scales"])
    gx, dA, dB, gx_slack, dA_slack, dB_slack = backward64(c, "fp32")
    within(got[0], gx, gx_slack, "dx")
    within(got[1], dA, dA_slack, "dA")
    within(got[2], dB, dB_slack, "dB")


@pytest.mark.gpu
def test_adapters_beyond_four_gigabytes(pkg):
    """The first, the last and a middle one of 1024 adapters of rank 128, 4.3 GB each of A and of B."""
    T, n, r, K, N = 40, 1024, 128, 16416, 16416
    assert n * r * K * 2 > 2 ** 32
    used = [0, 511, n - 1]
    c = make(T, len(used), r, K, N, "bf16", "mixed", seed=3)
    A, B = torch.zeros(n, r, K, dtype=DT["bf16"], device="cuda"), torch.zeros(n, N, r, dtype=DT["bf16"], device="cuda")
    for i, a in enumerate(used):
        A[a], B[a] = c["A"][i].cuda(), c["B"][i].cuda()
    scales = torch.ones(n, device="cuda")
    scales[used] = c["scales"].cuda()
    ids = torch.tensor([-1, *used])[c["ids"] + 1]
    plan = pkg.adapter_plan(ids.cuda(), n)
    out, u = pkg.lora_add(c["y"].cuda(), c["x"].cuda(), A, B, plan, scales, return_shrunk=True)
    want, want_u, slack, u_slack = forward64(c, "fp32")
    within(u, want_u, u_slack, "u")
    within(out, want, slack, "out")
    dx, dA, dB = pkg.lora_add_backward(c["dy"].cuda(), c["x"].cuda(), A, B, plan, scales, shrunk=u)
    del A, B
    gx, want_A, want_B, gx_slack, A_slack, B_slack = backward64(c, "fp32")
    within(dx, gx, gx_slack, "dx")
    within(dA[used], want_A, A_slack, "dA")
    within(dB[used], want_B, B_slack, "dB")
    dA[used], dB[used] = 0, 0
    assert not dA.any() and not dB.any()


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,bits", [(5000, 9, 32), (40000, 900, 64)])
def test_plan_of_a_long_batch_in_a_graph(pkg, T, n, bits):
    """Two launches, captured: every replay follows its ids."""
    dtype = torch.int32 if bits == 32 else torch.int64
    ids = torch.zeros(T, dtype=dtype, device="cuda")
    pkg.adapter_plan(ids, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = pkg.adapter_plan(ids, n)
    for seed in range(4):
        new = torch.randint(-1, n, (T,), generator=torch.Generator().manual_seed(seed))
        if seed == 2:
            new = torch.sort(new).values
        ids.copy_(new)
        graph.replay()
        eager = pkg.adapter_plan(ids, n)
        torch.cuda.synchronize()
        key = torch.where(new >= 0, new, n)
        assert torch.equal(plan.order.cpu().long(), torch.argsort(key, stable=True))
        assert torch.equal(plan.order, eager.order) and torch.equal(plan.starts, eager.starts)
