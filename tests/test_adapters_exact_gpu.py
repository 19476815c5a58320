"""``lora_add`` and ``lora_add_backward`` on numbers whose sums are exact in fp32, so that an output is the
exact result, rounded once.

The rank-space vectors (u forward, d backward) come out as ``256 a + b + c / 256`` with integers
``|a|, |b|, |c| <= 100``: multiples of 2^-8 below 2^15, 23 significand bits.  Two of them that differ in their last
digit alone meet with opposite signs, and what is left, ``(c - c') / 256``, has 8 bits: any output type holds it.
Every product is one of such a number (or of its 16-bit pieces) with a power of two, and every partial sum is a
multiple of 2^-8 below 2^16, which fp32 holds.  So there is no rounding at all, and the tolerance is zero;
a rank-space vector kept to 17 bits would be off by up to 25700 * 2^-18, 25 times the smallest difference.
"""
import pytest
import torch

from test_adapters_gpu import DT

DIGITS = (256.0, 1.0, 1.0 / 256)

# tokens, adapters, rank, dtype: the 16-token workgroups, sums of P by the expansion, vectors made once
SIZES = [(40, 2, 16, "bf16"), (40, 2, 64, "bf16"), (40, 2, 128, "fp16"), (40, 3, 24, "fp32"), (1300, 3, 16, "bf16"),
         (1300, 3, 16, "fp16"), (1300, 3, 40, "bf16"), (1300, 2, 128, "bf16"), (1300, 3, 64, "fp16"), (1300, 3, 72, "fp32"),
         (9000, 5, 64, "bf16"), (9000, 5, 32, "fp16"), (9000, 5, 16, "bf16"), (9000, 5, 64, "fp32")]


def digits(shape, width, g):
    """Rows of ``width`` whose first four values are digits."""
    out = torch.zeros(*shape, width, dtype=torch.float64)
    out[..., :4] = torch.randint(-100, 101, (*shape, 4), generator=g).double()
    return out


def reader(n, r, width):
    """[n, r, width]: rank 2i reads digits 0, 1, 2 of a row and rank 2i + 1 digits 0, 1, 3."""
    out = torch.zeros(n, r, width, dtype=torch.float64)
    out[..., 0], out[..., 1] = DIGITS[:2]
    out[:, 0::2, 2] = out[:, 1::2, 3] = DIGITS[2]
    return out


def differences(n, width, r, g):
    """[n, width, r]: each row takes one pair of ranks with opposite signs."""
    out = torch.zeros(n, width, r, dtype=torch.float64)
    pair = torch.randint(0, r // 2, (n, width, 1), generator=g)
    sign = torch.randint(0, 2, (n, width, 1), generator=g).double() * 2 - 1
    return out.scatter(2, 2 * pair, sign).scatter(2, 2 * pair + 1, -sign)


def partners(ids, digit_rows, width, g):
    """Rows whose first two digits are alike within an adapter, and [tokens, width] with one pair of an adapter's
    tokens, of opposite signs, in each column."""
    other = torch.zeros(len(ids), width, dtype=torch.float64)
    members = [torch.nonzero(ids == a).flatten() for a in range(int(ids.max()) + 1)]
    for m in members:
        digit_rows[m, :2] = digit_rows[m[0], :2]
    for col in range(width):
        for m in members:
            p = m[torch.randperm(len(m), generator=g)[:2]]
            other[p[0], col], other[p[1], col] = 1.0, -1.0
    return digit_rows, other


def setting(T, n, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(-1, n, (T,), generator=g)
    ids[:2 * n] = torch.arange(n).repeat(2)  # two tokens of each at least
    scales = 2.0 ** torch.randint(-1, 2, (n,), generator=g)
    return g, ids, scales, lambda t: t.to(DT[dtype]).cuda()


def check(got, want):
    rounded = want.to(got.dtype)
    assert torch.equal(rounded.double(), want)  # the exact result needs no rounding
    wrong = (got.cpu() != rounded).sum().item()
    assert wrong == 0, f"{wrong} of {got.numel()} wrong, worst {(got.cpu().double() - want).abs().max().item()}"


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,r,dtype", SIZES)
def test_output_is_the_rounded_exact_sum(pkg, T, n, r, dtype):
    g, ids, scales, to = setting(T, n, dtype, T + r)
    K, N = 72, 136
    x, A, B = digits((T,), K, g), reader(n, r, K), differences(n, N, r, g)
    plan = pkg.adapter_plan(ids.cuda(), n)
    y = torch.zeros(T, N, dtype=torch.float64)
    out, u = pkg.lora_add(to(y), to(x), to(A), to(B), plan, scales.cuda(), return_shrunk=True)
    on = (ids >= 0).double()[:, None]
    u64 = on * (x @ A[0].T)  # every adapter reads the same digits
    check(u, u64)
    want = y
    for a in range(n):
        t = ids == a
        want[t] = scales[a].double() * u64[t] @ B[a].T
    check(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,r,dtype", SIZES)
def test_input_gradient_is_the_rounded_exact_sum(pkg, T, n, r, dtype):
    g, ids, scales, to = setting(T, n, dtype, T + r + 1)
    K, N = 136, 72
    dy, B, A = digits((T,), N, g), reader(n, r, N).transpose(1, 2), differences(n, K, r, g).transpose(1, 2)
    plan = pkg.adapter_plan(ids.cuda(), n)
    dx, _, _ = pkg.lora_add_backward(to(dy), to(torch.zeros(T, K)), to(A), to(B), plan, scales.cuda())
    want = torch.zeros(T, K, dtype=torch.float64)
    for a in range(n):
        t = ids == a
        want[t] = scales[a].double() * (dy[t] @ B[a]) @ A[a]
    check(dx, want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,r,dtype", SIZES)
def test_weight_gradients_are_the_rounded_exact_sums(pkg, T, n, r, dtype):
    g, ids, scales, to = setting(T, n, dtype, T + r + 2)
    K, N = 136, 72
    plan = pkg.adapter_plan(ids.cuda(), n)
    # dA: d from the digits, x the pairs
    dy, x = partners(ids, digits((T,), N, g), K, g)
    B = reader(n, r, N).transpose(1, 2)
    _, dA, _ = pkg.lora_add_backward(to(dy), to(x), to(torch.zeros(n, r, K)), to(B), plan, scales.cuda())
    want = torch.stack([scales[a].double() * (dy[ids == a] @ B[a]).T @ x[ids == a] for a in range(n)])
    check(dA, want)
    # dB: u from the digits, dy the pairs
    x, dy = partners(ids, digits((T,), K, g), N, g)
    A = reader(n, r, K)
    _, _, dB = pkg.lora_add_backward(to(dy), to(x), to(A), to(torch.zeros(n, N, r)), plan, scales.cuda())
    want = torch.stack([scales[a].double() * dy[ids == a].T @ (x[ids == a] @ A[a].T) for a in range(n)])
    check(dB, want)
