"""Cases of the low-rank adapter and head-rotation operators, with their plain forms.

Five operators that stand around a shared (rotated, FP8) projection:

* ``plan``      tokens of a batch grouped by adapter           ``adapter_plan``
* ``lora``      the adapters' update added to a projection     ``lora_add``
* ``lora_grad`` its gradients                                  ``lora_add_backward``
* ``heads``     norm, position rotation and Hadamard rotation of query and key heads
                                                               ``qk_norm_rope``
* ``heads_grad`` its gradients                                 ``qk_norm_rope_backward``

``run`` computes a case in elementary torch operations in fp32 (``own`` false) or through the
package's kernels (``own`` true); ``exact`` computes it in fp64 from the definition.
"""
import importlib
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = "cuda"


def _package():
    return importlib.import_module("6s894_project_2025_amd")


# ---------------------------------------------------------------------------------------------
# cases

def listed():
    return [
        # one serving step of a large batch: a token per request, adapters in no order
        {"name": "plan_decode_256", "op": "plan", "T": 256, "n": 64, "batch": "tokens"},
        # a training or prompt batch: long runs of one adapter
        {"name": "plan_prompts_32768", "op": "plan", "T": 32768, "n": 32, "batch": "requests"},

        # latency of a single request's single token beside a 4096 x 4096 projection
        {"name": "lora_one_token", "op": "lora", "T": 1, "n": 4, "r": 16, "K": 4096, "N": 4096,
         "dtype": "bf16", "batch": "tokens"},
        # a serving step: 64 requests, most with an adapter of their own, the 4096 -> 14336 layer
        {"name": "lora_decode_64", "op": "lora", "T": 64, "n": 48, "r": 16, "K": 4096, "N": 14336,
         "dtype": "bf16", "batch": "tokens"},
        # 8192 prompt tokens of several requests, rank 64, the 4096 -> 14336 layer
        {"name": "lora_prompts_8192", "op": "lora", "T": 8192, "n": 8, "r": 64, "K": 4096, "N": 14336,
         "dtype": "bf16", "batch": "requests"},

        # a small ragged fine-tuning batch with sizes that fill no tile, fp16
        {"name": "lora_grad_ragged_1003", "op": "lora_grad", "T": 1003, "n": 5, "r": 24, "K": 1000,
         "N": 1544, "dtype": "fp16", "batch": "requests"},
        # fine-tuning step of four adapters at once, 8192 tokens, the 4096 -> 14336 layer
        {"name": "lora_grad_8192", "op": "lora_grad", "T": 8192, "n": 4, "r": 16, "K": 4096, "N": 14336,
         "dtype": "bf16", "batch": "requests"},

        # latency of a single token: 32 query and 8 key heads of 128, far into a long context
        {"name": "heads_one_token", "op": "heads", "T": 1, "Hq": 32, "Hk": 8, "D": 128, "R": 128,
         "dtype": "bf16", "axes": 1, "pairs": "halves", "hadamard": True, "batch": "tokens"},
        # image and video tokens with three position axes, heads of 80, an odd count
        {"name": "heads_three_axes_1347", "op": "heads", "T": 1347, "Hq": 20, "Hk": 4, "D": 80, "R": 80,
         "dtype": "fp16", "axes": 3, "pairs": "halves", "hadamard": False, "batch": "requests"},
        # 8192 prompt tokens; the heads leave rotated by the Hadamard matrix, ready to be quantized
        {"name": "heads_prompts_8192", "op": "heads", "T": 8192, "Hq": 32, "Hk": 8, "D": 128, "R": 128,
         "dtype": "bf16", "axes": 1, "pairs": "halves", "hadamard": True, "batch": "requests"},

        # small fp32 training batch, neighbouring pairs, a partial rotation of large heads
        {"name": "heads_grad_333", "op": "heads_grad", "T": 333, "Hq": 8, "Hk": 2, "D": 256, "R": 64,
         "dtype": "fp32", "axes": 1, "pairs": "neighbours", "hadamard": False, "batch": "requests"},
        # training on 8192 tokens
        {"name": "heads_grad_8192", "op": "heads_grad", "T": 8192, "Hq": 32, "Hk": 8, "D": 128, "R": 128,
         "dtype": "bf16", "axes": 1, "pairs": "halves", "hadamard": True, "batch": "requests"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "lora", "lora", "lora_grad", "heads", "heads", "heads_grad"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    batch = rng.choice(["tokens", "requests"])
    if op == "plan":
        T = _log_int(rng, 64, 32768)
        return {"op": op, "T": T, "n": _log_int(rng, 2, 256), "batch": batch if T > 4000 else "tokens"}
    if op in ("lora", "lora_grad"):
        T = _log_int(rng, 1 if op == "lora" else 64, 8192)
        if dtype == "fp32":
            T = min(T, 2048)
        return {"op": op, "T": T, "n": _log_int(rng, 1, 64 if op == "lora" else 16),
                "r": 8 * rng.randint(1, 8), "K": 8 * _log_int(rng, 16, 512),
                "N": 8 * _log_int(rng, 16, 1792), "dtype": dtype, "batch": batch}
    D = rng.choice([64, 80, 96, 128, 128, 256])
    Hk = rng.randint(1, 8)
    Hq = Hk * rng.choice([1, 2, 4, 8])
    T = _log_int(rng, 1 if op == "heads" else 64, 8192)
    T = max(1, min(T, 8192 * 40 * 128 // ((Hq + Hk) * D * (2 if dtype == "fp32" else 1))))
    R = rng.choice([D, D, D, D // 2 if D % 32 == 0 else D])
    return {"op": op, "T": T, "Hq": Hq, "Hk": Hk, "D": D, "R": R, "dtype": dtype,
            "axes": rng.choice([1, 1, 2, 3]), "pairs": rng.choice(["halves", "halves", "neighbours"]),
            "hadamard": D & (D - 1) == 0 and rng.random() < 0.5, "batch": batch}


def work(case):
    e = 4 if case.get("dtype") == "fp32" else 2
    T = case["T"]
    if case["op"] == "plan":
        return {"bytes": 4 * (2 * T + case["n"] + 1), "flops": T}
    if case["op"] in ("lora", "lora_grad"):
        r, K, N = case["r"], case["K"], case["N"]
        used = min(case["n"], T)
        adapters = used * r * (K + N) * e
        if case["op"] == "lora":
            return {"bytes": T * (K + 2 * N) * e + adapters + 4 * T, "flops": 2 * T * r * (K + N)}
        gradients = case["n"] * r * (K + N) * e
        return {"bytes": T * (2 * K + N) * e + 4 * T * r + adapters + gradients + 4 * T,
                "flops": 4 * T * r * (K + N)}
    H, D = case["Hq"] + case["Hk"], case["D"]
    passes = 2 if case["op"] == "heads" else 3
    per_value = (6 + (int(math.log2(D)) if case["hadamard"] else 0)) * (passes - 1)
    return {"bytes": passes * T * H * D * e + 4 * T * case["axes"], "flops": per_value * T * H * D}


# ---------------------------------------------------------------------------------------------
# inputs

def _generators(seed):
    return (torch.Generator().manual_seed(seed), torch.Generator(device=_DEV).manual_seed(seed + 1))


def _request_lengths(T, g):
    """Ragged request lengths that add up to T: as many as a batch of this size would hold."""
    count = max(1, min(T, 1 + T // 700))
    w = torch.rand(count, generator=g) + 0.05
    cuts = (torch.cumsum(w, 0) / w.sum() * T).round().to(torch.int64)
    cuts[-1] = T
    return torch.diff(cuts, prepend=torch.zeros(1, dtype=torch.int64))


def _adapter_ids(case, g):
    """An adapter for each token; about one token or request in sixteen has none (-1)."""
    T, n = case["T"], case["n"]
    if case["batch"] == "tokens":
        ids = torch.randint(0, n, (T,), generator=g)
        if T > 1:
            ids[torch.rand(T, generator=g) < 1 / 16] = -1
        return ids.to(torch.int32)
    lengths = _request_lengths(T, g)
    of = torch.randint(0, n, (len(lengths),), generator=g)
    of[torch.rand(len(lengths), generator=g) < 1 / 16] = -1
    of[0] = 0
    return torch.repeat_interleave(of, lengths).to(torch.int32)


def _randn(shape, scale, dtype, g):
    return (torch.randn(shape, generator=g, device=_DEV) * scale).to(dtype)


def _lora_inputs(case, seed):
    host, dev = _generators(seed)
    T, n, r, K, N = (case[k] for k in ("T", "n", "r", "K", "N"))
    dt = _DTYPES[case["dtype"]]
    ids = _adapter_ids(case, host)
    # activations with a few outlier channels, as a projection's input has them
    x = torch.randn((T, K), generator=dev, device=_DEV)
    x[:, torch.randperm(K, generator=host)[:max(1, K // 100)].to(_DEV)] *= 8.0
    s = {"ids": ids.to(_DEV), "x": x.to(dt),
         "A": _randn((n, r, K), K ** -0.5, dt, dev), "B": _randn((n, N, r), 0.02, dt, dev),
         "scales": (torch.rand(n, generator=dev, device=_DEV) + 0.5) * 2.0,
         # the tokens of each adapter: what a program that has no plan operator keeps
         "groups": [(a, torch.nonzero(ids == a).flatten().to(_DEV)) for a in range(n) if (ids == a).any()]}
    if case["op"] == "lora":
        s["y"] = _randn((T, N), 1.0, dt, dev)
    else:
        s["dy"] = _randn((T, N), 0.01, dt, dev)
        u = torch.zeros((T, r), device=_DEV)
        for a, t in s["groups"]:
            u[t] = s["x"][t].float() @ s["A"][a].float().T
        s["shrunk"] = u  # what the forward pass left
    return s


def _sections(case):
    """Frequencies per position axis: a quarter for time, the rest shared by height and width."""
    f, axes = case["R"] // 2, case["axes"]
    if axes == 1:
        return (f,)
    first = f // 4 if axes == 3 else f // 2
    rest = f - first
    return (first, rest) if axes == 2 else (first, rest // 2, rest - rest // 2)


def _positions(case, g):
    T, axes = case["T"], case["axes"]
    if case["batch"] == "tokens":  # a token each, anywhere in a context of up to 131072
        base = torch.randint(0, 131072, (T,), generator=g)
    else:
        base = torch.cat([torch.arange(int(l)) for l in _request_lengths(T, g)])
    if axes == 1:
        return base.to(torch.int32)
    width = 28  # frames of 28 x 28 patches
    t, h, w = base // (width * width), base // width % width, base % width
    return torch.stack([t, h, w] if axes == 3 else [h, w]).to(torch.int32)


def _hadamard_matrix(n):
    i = torch.arange(n)
    bits = i[:, None] & i[None, :]
    sign = torch.zeros_like(bits)
    while bool(bits.any()):
        sign ^= bits & 1
        bits = bits >> 1
    return (1 - 2 * sign).to(torch.float64) / math.sqrt(n)


def _heads_inputs(case, seed):
    host, dev = _generators(seed)
    T, Hq, Hk, D, R = (case[k] for k in ("T", "Hq", "Hk", "D", "R"))
    dt = _DTYPES[case["dtype"]]
    # queries, keys and values leave the projection in one row per token
    qkv = _randn((T, (Hq + 2 * Hk) * D), 1.5, dt, dev)
    s = {"q": qkv[:, :Hq * D].unflatten(1, (Hq, D)),
         "k": qkv[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D)),
         "qw": (1.0 + _randn((D,), 0.1, torch.float32, dev)).to(dt),
         "kw": (1.0 + _randn((D,), 0.1, torch.float32, dev)).to(dt),
         "positions": _positions(case, host).to(_DEV),
         "inv_freq": (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).float().to(_DEV),
         "sections": _sections(case)}
    if case["hadamard"]:
        s["H"] = _hadamard_matrix(D).float().to(_DEV)
    if case["op"] == "heads_grad":
        s["dq"] = _randn((T, Hq, D), 0.01, dt, dev)
        s["dk"] = _randn((T, Hk, D), 0.01, dt, dev)
    return s


def prepare(case, seed):
    if case["op"] == "plan":
        state = {"ids": _adapter_ids(case, _generators(seed)[0]).to(_DEV)}
    elif case["op"] in ("lora", "lora_grad"):
        state = _lora_inputs(case, seed)
        if own:  # once a batch: every projection of every layer uses it
            state["plan"] = _package().adapter_plan(state["ids"], case["n"])
    else:
        state = _heads_inputs(case, seed)
    state["case"] = case
    return state


# ---------------------------------------------------------------------------------------------
# plain forms, fp32

_EPS = 1e-6


def _plain_plan(s):
    n = s["case"]["n"]
    ids = s["ids"].long()
    key = torch.where((ids >= 0) & (ids < n), ids, n)
    ordered, order = torch.sort(key, stable=True)
    starts = torch.searchsorted(ordered, torch.arange(n + 1, device=_DEV))
    return order.to(torch.int32), starts.to(torch.int32)


def _plain_lora(s):
    x, y, A, B = s["x"], s["y"], s["A"], s["B"]
    out = y.clone()
    for a, t in s["groups"]:
        u = x[t].float() @ A[a].float().T
        out[t] = (y[t].float() + (u * s["scales"][a]) @ B[a].float().T).to(y.dtype)
    return out


def _plain_lora_grad(s):
    x, dy, A, B, u = s["x"], s["dy"], s["A"], s["B"], s["shrunk"]
    dx, dA, dB = torch.zeros_like(x), torch.zeros_like(A), torch.zeros_like(B)
    for a, t in s["groups"]:
        xa, ga = x[t].float(), dy[t].float() * s["scales"][a]
        du = ga @ B[a].float()
        dx[t] = (du @ A[a].float()).to(x.dtype)
        dA[a] = (du.T @ xa).to(A.dtype)
        dB[a] = (ga.T @ u[t]).to(B.dtype)
    return dx, dA, dB


def _plain_angles(s):
    """cos and sin of every token's angles, [T, 1, R/2]; the angles in fp64."""
    c, pos, freq = s["case"], s["positions"].double(), s["inv_freq"].double()
    if c["axes"] > 1:
        axis = torch.repeat_interleave(torch.arange(c["axes"], device=_DEV),
                                       torch.tensor(s["sections"], device=_DEV), output_size=c["R"] // 2)
        pos = pos[axis].T
    else:
        pos = pos[:, None]
    angle = (pos * freq)[:, None, :]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _plain_rotate(v, cos, sin, c):
    R = c["R"]
    if c["pairs"] == "halves":
        a, b = v[..., :R // 2], v[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = v[..., 0:R:2], v[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, v[..., R:]], dim=-1)


def _plain_heads(s):
    c = s["case"]
    cos, sin = _plain_angles(s)
    out = []
    for v, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        f = v.float()
        f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + _EPS) * w.float()
        f = _plain_rotate(f, cos, sin, c)
        if c["hadamard"]:
            f = f @ s["H"]
        out.append(f.to(v.dtype))
    return tuple(out)


def _plain_heads_grad(s):
    c = s["case"]
    cos, sin = _plain_angles(s)
    grads, weight_grads = [], []
    for v, w, d in ((s["q"], s["qw"], s["dq"]), (s["k"], s["kw"], s["dk"])):
        f, g = v.float(), d.float()
        if c["hadamard"]:
            g = g @ s["H"]  # symmetric
        g = _plain_rotate(g, cos, -sin, c)
        inv = torch.rsqrt((f * f).mean(-1, keepdim=True) + _EPS)
        normed, gw = f * inv, g * w.float()
        grads.append((inv * (gw - normed * (gw * normed).mean(-1, keepdim=True))).to(v.dtype))
        weight_grads.append((g * normed).sum((0, 1)).to(w.dtype))
    return (*grads, *weight_grads)


_PLAIN = {"plan": _plain_plan, "lora": _plain_lora, "lora_grad": _plain_lora_grad,
          "heads": _plain_heads, "heads_grad": _plain_heads_grad}


def _kernels(s):
    hada, c = _package(), s["case"]
    if c["op"] == "plan":
        plan = hada.adapter_plan(s["ids"], c["n"])
        return plan.order, plan.starts
    if c["op"] == "lora":
        return hada.lora_add(s["y"], s["x"], s["A"], s["B"], s["plan"], s["scales"])
    if c["op"] == "lora_grad":
        return hada.lora_add_backward(s["dy"], s["x"], s["A"], s["B"], s["plan"], s["scales"],
                                      shrunk=s["shrunk"])
    options = dict(eps=_EPS, sections=s["sections"], interleaved=c["pairs"] == "neighbours",
                   hadamard=c["hadamard"])
    if c["op"] == "heads":
        return hada.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["positions"], s["inv_freq"], **options)
    return hada.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["qw"], s["kw"], s["positions"],
                                      s["inv_freq"], **options)


def run(state):
    return _kernels(state) if own else _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------
# the definition in fp64

def _exact_plan(case, seed):
    ids = _adapter_ids(case, _generators(seed)[0]).tolist()
    n = case["n"]
    lists = [[] for _ in range(n + 1)]
    for t, a in enumerate(ids):
        lists[a if 0 <= a < n else n].append(t)
    starts, order = [], []
    for members in lists:
        starts.append(len(order))
        order += members
    return (torch.tensor(order, dtype=torch.int32, device=_DEV),
            torch.tensor(starts, dtype=torch.int32, device=_DEV))


def _exact_lora(case, seed):
    s = _lora_inputs(case, seed)
    ids = s["ids"].long()
    out = s["y"].double()
    for a in torch.unique(ids[ids >= 0]).tolist():
        rows = (ids == a)
        W = s["B"][a].double() @ s["A"][a].double() * s["scales"][a].double()
        out[rows] += s["x"][rows].double() @ W.T
    return out


def _exact_lora_grad(case, seed):
    s = _lora_inputs(case, seed)
    ids = s["ids"].long()
    dx = torch.zeros(s["x"].shape, dtype=torch.float64, device=_DEV)
    dA = torch.zeros(s["A"].shape, dtype=torch.float64, device=_DEV)
    dB = torch.zeros(s["B"].shape, dtype=torch.float64, device=_DEV)
    for a in torch.unique(ids[ids >= 0]).tolist():
        rows = (ids == a)
        x, g = s["x"][rows].double(), s["dy"][rows].double()
        A, B, c = s["A"][a].double(), s["B"][a].double(), s["scales"][a].double()
        dW = g.T @ x  # gradient of the adapter's whole matrix c * B @ A
        dA[a], dB[a] = c * (B.T @ dW), c * (dW @ A.T)
        dx[rows] = c * (g @ B) @ A
    return dx, dA, dB


def _exact_rotated(v, w, s, case, H):
    """The definition on complex numbers: pair i of a head turns by position * frequency."""
    R, dev = case["R"], v.device
    normed = v / torch.sqrt(v.square().mean(-1, keepdim=True) + _EPS) * w
    pos = s["positions"].double().reshape(case["axes"], -1)
    owner = [a for a, count in enumerate(s["sections"]) for _ in range(count)]
    angle = pos[torch.tensor(owner, device=dev)].T * s["inv_freq"].double()
    first = (torch.arange(R // 2, device=dev) if case["pairs"] == "halves"
             else 2 * torch.arange(R // 2, device=dev))
    second = first + (R // 2 if case["pairs"] == "halves" else 1)
    z = torch.complex(normed[..., first], normed[..., second])
    z = z * torch.polar(torch.ones_like(angle), angle)[:, None, :]
    out = normed.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out @ H if H is not None else out


def _exact_heads(case, seed):
    s = _heads_inputs(case, seed)
    H = _hadamard_matrix(case["D"]).to(_DEV) if case["hadamard"] else None
    return tuple(_exact_rotated(s[v].double(), s[w].double(), s, case, H) for v, w in (("q", "qw"), ("k", "kw")))


def _exact_heads_grad(case, seed):
    s = _heads_inputs(case, seed)
    H = _hadamard_matrix(case["D"]).to(_DEV) if case["hadamard"] else None
    grads, weight_grads = [], []
    for v, w, d in (("q", "qw", "dq"), ("k", "kw", "dk")):
        leaf = s[v].double().requires_grad_()
        weight = s[w].double().requires_grad_()
        out = _exact_rotated(leaf, weight, s, case, H)
        gv, gw = torch.autograd.grad(out, (leaf, weight), s[d].double())
        grads.append(gv)
        weight_grads.append(gw)
    return (*grads, *weight_grads)


_EXACT = {"plan": _exact_plan, "lora": _exact_lora, "lora_grad": _exact_lora_grad,
          "heads": _exact_heads, "heads_grad": _exact_heads_grad}


def exact(case, seed):
    return _EXACT[case["op"]](case, seed)
