"""Which tensors may be written in place: the package's test for shared memory against all pairs of elements."""
import importlib
import random

import pytest
import torch


@pytest.fixture(scope="module")
def apart(pkg):
    return importlib.import_module(pkg.__name__ + ".ops")._apart


def places(t):
    at = [t.data_ptr()]
    for stride, n in zip(t.stride(), t.shape):
        at = [a + i * stride * t.element_size() for a in at for i in range(n)]
    return at


def by_pairs(*tensors):
    size = tensors[0].element_size()
    at = sorted(a for t in tensors for a in places(t))
    return all(b - a >= size for a, b in zip(at, at[1:]))


def view(rng, base, dims):
    """Any view of at most a few dozen elements that lies in `base`."""
    while True:
        shape = [rng.choice([0, 1, 1, 2, 3, 4]) if rng.random() < 0.9 else 5 for _ in range(dims)]
        strides = [rng.choice([0, 1, 1, 2, 3, 4, 6, 8, 12, 16]) for _ in range(dims)]
        offset = rng.choice([0, 1, 2, 3, 4, 8, 12, 40])
        if offset + sum(s * max(0, n - 1) for n, s in zip(shape, strides)) < base.numel():
            return base.as_strided(shape, strides, offset)


@pytest.mark.parametrize("dims", [2, 3])
def test_against_all_pairs(apart, dims):
    rng = random.Random(dims)
    base, answers = torch.zeros(100), set()
    for _ in range(4000):
        t, other = view(rng, base, dims), view(rng, base, dims)
        assert apart(t) == by_pairs(t), (t.shape, t.stride())
        want = by_pairs(t, other)
        assert apart(t, other) == want, (t.shape, t.stride(), t.storage_offset(), other.shape, other.stride(), other.storage_offset())
        answers.add(want)
    assert answers == {True, False}


def test_layouts_of_use(apart):
    T, Hq, Hk, D = 7, 4, 2, 8
    qkv = torch.zeros(T, (Hq + 2 * Hk) * D)
    q, k = qkv[:, :Hq * D].unflatten(1, (Hq, D)), qkv[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D))
    assert apart(q, k) and apart(k, q)
    assert not apart(q, qkv[:, (Hq - 1) * D:(Hq + 1) * D].unflatten(1, (2, D)))  # the last query head once more
    assert not apart(q, qkv[:, D // 2:D // 2 + D].unflatten(1, (1, D)))
    assert not apart(q[1:], q[:-1]) and apart(q[3:], q[:3])
    turned = torch.zeros(Hq + Hk, T, D).transpose(0, 1)
    assert apart(turned[:, :Hq], turned[:, Hq:]) and not apart(turned[:, :Hq], turned[:, Hq - 1:])
    pairs = torch.zeros(T, Hq, 2, D)  # a key head beside each query head
    assert apart(pairs[:, :, 0], pairs[:, :, 1]) and not apart(pairs[:, :, 0], pairs[:, 1:, 0])
    fine = torch.zeros(T, Hq, D, 2)
    assert apart(fine[..., 0], fine[..., 1]) and not apart(fine[..., 0], fine[..., 0])
    rows = torch.zeros(40)
    assert apart(rows.as_strided((4, 8), (8, 1))) and not apart(rows.as_strided((4, 8), (7, 1)))
    assert not apart(rows[:8].expand(4, 8)) and apart(rows[:8].expand(1, 8))


@pytest.mark.gpu
def test_operators_refuse_shared_memory_in_place(pkg):
    T, D, n, r, K, N = 8, 64, 2, 8, 64, 128
    pos, freq = torch.arange(T, device="cuda"), torch.rand(D // 2, device="cuda")
    buf = torch.randn(T + 1, 4 * D, device="cuda").bfloat16()
    q = buf[:T, :2 * D].unflatten(1, (2, D))
    for k in (buf[:T, D:2 * D], buf[:T, D + 8:2 * D + 8], buf[1:, :D], buf.flatten()[:T * D].view(T, D)):
        with pytest.raises(RuntimeError, match="share memory"):
            pkg.qk_norm_rope(q, k[:, None], None, None, pos, freq, inplace=True)
        pkg.qk_norm_rope(q, k[:, None], None, None, pos, freq)
    sliding = buf.as_strided((T, 2, D), (D, D, 1))
    with pytest.raises(RuntimeError, match="share memory"):
        pkg.qk_norm_rope(sliding, buf[:T, 3 * D:].unflatten(1, (1, D)), None, None, pos, freq, inplace=True)
    bf = lambda *s: torch.randn(*s, device="cuda").bfloat16()
    plan = pkg.adapter_plan(torch.zeros(T, dtype=torch.int32, device="cuda"), n)
    x, A, B = bf(T, K), bf(n, r, K), bf(n, N, r)
    for row in (lambda width: width - 1, lambda width: 8, lambda width: 1, lambda width: 0):
        y, dx = buf.as_strided((T, N), (row(N), 1)), buf.as_strided((T, K), (row(K), 1))
        with pytest.raises(RuntimeError, match="share memory"):
            pkg.lora_add(y, x, A, B, plan, inplace=True)
        with pytest.raises(RuntimeError, match="share memory"):
            pkg.lora_add_backward(bf(T, N), x, A, B, plan, dx=dx)
        pkg.lora_add(y, x, A, B, plan)


def test_layouts_of_use_are_told_from_their_strides(pkg, monkeypatch):
    """The comparison of all rows takes 40 ms for 8192 tokens of 64 heads: no usual layout comes to it."""
    ops = importlib.import_module(pkg.__name__ + ".ops")
    monkeypatch.setattr(ops, "_apart_one_by_one", lambda *tensors: pytest.fail("compared one by one"))
    T, H, D = 8192, 32, 128
    packed = torch.empty(T, (H + 16) * D, device="meta")
    per_head = torch.empty(T, H, 3, D, device="meta")
    per_group = torch.empty(T, 8, 6, D, device="meta")
    heads_first = torch.empty(H + 16, T, D, device="meta")
    pairs = torch.empty(T, H, D, 2, device="meta")
    for q, k in ((packed[:, :H * D].unflatten(1, (H, D)), packed[:, H * D:(H + 8) * D].unflatten(1, (8, D))),
                 (packed[:, 16 * D:].unflatten(1, (H, D)), packed[:, :8 * D].unflatten(1, (8, D))),
                 (per_head[:, :, 0], per_head[:, :, 1]), (per_head[:, :, 2], per_head[:, :, 0]),
                 (per_group[:, :, 3], per_group[:, :, 4]),
                 (heads_first[:H].transpose(0, 1), heads_first[H:H + 8].transpose(0, 1)),
                 (pairs[..., 0], pairs[..., 1]), (packed[:1, :H * D].unflatten(1, (H, D)), packed[1:2, :D].unflatten(1, (1, D)))):
        assert at_addresses(ops._apart, q, k)
        assert ops._apart(q) and ops._apart(k)


def at_addresses(f, *tensors):
    """A call on tensors without memory, which have offsets but no addresses."""
    class At:
        def __init__(self, t):
            self.t, self.shape = t, t.shape

        def data_ptr(self):
            return (1 << 20) + self.t.storage_offset() * self.t.element_size()

        def __getattr__(self, name):
            return getattr(self.t, name)

    return f(*(At(t) for t in tensors))
