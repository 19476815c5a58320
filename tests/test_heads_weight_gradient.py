"""Weight gradients of ``qk_norm_rope_backward``, whose sums go over every token and head, with a tolerance that a
missing wavefront or a missing row of partial sums does not fit into.

A term ``g_i n_i`` (n the normed head, g the gradient in front of the norm's weight) is off by 96 u of the row's norm
(u = 2^-24; the rotations and the two sums behind it).  The additions: a lane adds one term for each of its items, then
come at most 6 steps across lane groups, 2 across wavefronts, 2 rows of partial sums and 8 steps of a tree
over 256 threads, each off by u of the sum of the terms' magnitudes.  How many items a wavefront has is counted here
as the launch cuts the work.
"""
import pytest
import torch

from test_heads_gpu import U, backward64, hadamard64, make, pair_matrices, split

# T, Hq, Hk, D, R, dtype, interleaved, hadamard: many units a wavefront, many passes a unit, few heads, a long batch
CASES = [
    (8200, 3, 1, 48, 32, "bf16", False, False),
    (1027, 9, 2, 128, 128, "fp32", False, True),
    (3001, 32, 8, 128, 128, "bf16", False, True),
    (5003, 1, 1, 64, 64, "fp16", True, False),
    (2049, 20, 4, 80, 80, "fp16", False, False),
    (1500, 5, 3, 512, 128, "bf16", False, False),
    (1, 40000, 3, 16, 16, "bf16", False, False),
    (3, 9000, 1, 32, 16, "fp32", False, True),
]
MOST = 512


def items(T, H, others, D):
    """Items of a wavefront at most, and workgroups, of the side with H heads beside `others`."""
    lg = next(i for i in range(6) if 16 << i >= D)
    groups = 64 >> lg
    passes, rest = -(-H // groups), -(-others // groups)
    waves = 4 * (1 + T * passes * (MOST - 2) // (T * (passes + rest)))
    parts = 0
    while 2 << parts <= passes and T << parts < waves:
        parts += 1
    units = T << parts
    each = -(-units // waves)
    return each * -(-passes // (1 << parts)), -(-(-(-units // each)) // 4)


def reference(T, Hq, Hk, D, R, dtype, interleaved, hadamard):
    qkv, w, pos, freq, _ = make(T, Hq, Hk, D, R, dtype, seed=T + D)
    gen = torch.Generator().manual_seed(6)
    heads = split(qkv, Hq, Hk, D)
    grads = [(torch.randn(x.shape, generator=gen) * 0.1).to(x.dtype) for x in heads]
    w = [t.float() for t in w]  # fp32 weights: their gradients come out in fp32
    rot = pair_matrices(pos, freq, None, R, interleaved)
    return qkv, heads, grads, w, pos, freq, rot


def terms(x, w, g, rot, hadamard):
    """g_i n_i of every token and head."""
    cos, sin, first, second = rot
    x, g = x.double(), g.double()
    if hadamard:
        g = g @ hadamard64(x.shape[-1])
    b = g.clone()
    c, s = cos[:, None, :], sin[:, None, :]
    b[..., first] = g[..., first] * c + g[..., second] * s
    b[..., second] = g[..., second] * c - g[..., first] * s
    return b * x * (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt()


def tolerance(each, dw, dw_mag, count):
    return dw.abs() * U + 96 * U * dw_mag + (count + 18) * U * each.abs().sum((0, 1))


@pytest.mark.parametrize("T,Hq,Hk,D,R,dtype,interleaved,hadamard", CASES)
def test_a_missing_part_does_not_fit_the_tolerance(T, Hq, Hk, D, R, dtype, interleaved, hadamard):
    _, heads, grads, w, _, _, rot = reference(T, Hq, Hk, D, R, dtype, interleaved, hadamard)
    for x, ww, g, H, others in zip(heads, w, grads, (Hq, Hk), (Hk, Hq)):
        _, dw, _, dw_mag = backward64(x, ww, g, rot, 1e-5, hadamard)
        each = terms(x, ww, g, rot, hadamard)
        assert torch.allclose(each.sum((0, 1)), dw, rtol=1e-9, atol=1e-12)
        count, blocks = items(T, H, others, D)
        assert blocks <= MOST
        tol = tolerance(each, dw, dw_mag, count)
        assert tol.square().mean().sqrt() <= 0.02 * dw.square().mean().sqrt()
        # a wavefront's worth of heads: any 64 / 2^lg of them
        flat = each.flatten(0, 1)
        lost = flat[:max(1, len(flat) // (4 * blocks))].sum(0)
        assert (lost.abs() > tol).any() and (dw.abs() > tol).float().mean() > 0.9


@pytest.mark.gpu
@pytest.mark.parametrize("T,Hq,Hk,D,R,dtype,interleaved,hadamard", CASES)
def test_weight_gradients(pkg, T, Hq, Hk, D, R, dtype, interleaved, hadamard):
    qkv, heads, grads, w, pos, freq, rot = reference(T, Hq, Hk, D, R, dtype, interleaved, hadamard)
    q, k = split(qkv.cuda(), Hq, Hk, D)
    args = (grads[0].cuda(), grads[1].cuda(), q, k, w[0].cuda(), w[1].cuda(), pos.cuda(), freq.cuda())
    opts = dict(eps=1e-5, interleaved=interleaved, hadamard=hadamard)
    got = pkg.qk_norm_rope_backward(*args, **opts)
    again = pkg.qk_norm_rope_backward(*args, **opts)
    for i, (x, ww, g, H, others) in enumerate(zip(heads, w, grads, (Hq, Hk), (Hk, Hq))):
        _, dw, _, dw_mag = backward64(x, ww, g, rot, 1e-5, hadamard)
        tol = tolerance(terms(x, ww, g, rot, hadamard), dw, dw_mag, items(T, H, others, D)[0])
        err = (got[2 + i].cpu().double() - dw).abs()
        assert (err <= tol).all(), f"worst error {(err / tol).max().item()} of the bound"
        assert torch.equal(got[2 + i], again[2 + i])
