"""Workspaces of ``lora_add`` and ``lora_add_backward``: what they hold, counted here, against the library's size; and
that the rows of partial weight gradients are as many as a batch can need, and no more than that."""
import importlib
import random

import pytest

ELEMENT = {0: 4, 1: 2, 2: 2}  # fp32, bf16, fp16
VEC = {0: 4, 1: 8, 2: 8}      # values of 16 bytes


def chunk_of(T):
    return 128 if T < 4096 else 256 if T < 8192 else 512


def slots_of(T, n):
    return T // chunk_of(T) + min(n, T // chunk_of(T))


def tiles_of(T, n):
    return T // 64 + min(T, n + 1)


def padded(r):
    return next(p for p in (16, 32, 64, 128) if r <= p)


def cut(tiles, blocks, least, most):
    parts = min(max(8, most // tiles) if tiles else 8, max(1, blocks // least))
    return parts // 8 * 8 if parts > 8 else parts


class Cut:
    """How a batch's forward pass is cut: the 16-token form, parts of the contraction and of the expansion, and
    whether the expansion adds up the parts of P itself."""

    def __init__(self, T, n, r, K, N, dtype):
        block = 16 * VEC[dtype]
        self.tiles = tiles_of(T, n)
        self.few = self.tiles <= 16
        self.splits = cut(self.tiles, -(-K // block), 4 if self.few else 2, 1024)
        self.parts = cut(self.tiles, -(-N // block), 4 if self.few else 2, 1024 if self.few else 8192)
        self.sums = self.splits * padded(r) * 4
        self.own = self.few or (self.sums * self.parts * T <= 16 << 20 and self.sums * self.parts * self.tiles * 64 <= 192 << 20)


def whole(*sizes):
    return sum(-(-s // 256) * 256 for s in sizes)


def pieces(r, dtype):
    return padded(r) * 64 * (6 if dtype == 1 else 4)


def vectors(r, dtype):
    return 8192 if dtype == 1 and padded(r) == 16 else pieces(r, dtype)


def forward_bytes(T, n, r, K, N, dtype):
    c = Cut(T, n, r, K, N, dtype)
    return whole(c.sums * T, *([] if c.own else [c.tiles * vectors(r, dtype), c.tiles * 256]))


def backward_bytes(T, n, r, K, N, dtype):
    tiles = tiles_of(T, n)
    sums = max(-(-N // (64 * VEC[dtype])) * padded(r) * 4, Cut(T, n, r, K, N, dtype).sums)
    return whole(sums * T, n * r * K * ELEMENT[dtype], tiles * vectors(r, dtype), tiles * 256,
                 *2 * [tiles * pieces(r, dtype), tiles * 4], slots_of(T, n) * r * (K + N) * 4)


@pytest.fixture(scope="module")
def size(pkg):
    lib = importlib.import_module(pkg.__name__ + "._lib").load()
    pack = importlib.import_module(pkg.__name__ + ".adapters")._LORA.pack
    return lambda T, n, r, K, N, dtype, backward: lib.mi_lora_workspace(pack(T, K, N, N, n, r, K, N, dtype), backward)


def test_sizes_are_what_is_held(size):
    rng = random.Random(1)
    for _ in range(2000):
        case = (int(2 ** rng.uniform(0, 20)), rng.randint(1, 1024) if rng.random() < 0.5 else rng.randint(1, 8), 8 * rng.randint(1, 16),
                8 * rng.randint(1, 2000), 8 * rng.randint(1, 2000), rng.randint(0, 2))
        assert size(*case, 0) == forward_bytes(*case), case
        assert size(*case, 1) == backward_bytes(*case), case


def test_rows_of_partial_gradients_suffice_and_are_reached():
    """Slots are ceil(c / chunk) for each adapter with c > chunk tokens."""
    rng = random.Random(2)

    def used(counts, chunk):
        return sum(-(-c // chunk) for c in counts if c > chunk)

    for T, n in [(1, 1), (128, 2), (129, 1), (200, 3), (4095, 40), (4096, 3), (8191, 9), (8192, 16), (65536, 4), (100000, 300)]:
        chunk = chunk_of(T)
        most = 0
        for _ in range(300):
            cuts = sorted(rng.randint(0, T) for _ in range(n - 1))
            most = max(most, used([b - a for a, b in zip([0, *cuts], [*cuts, T])], chunk))
        # the worst: adapters of one chunk and a token, the rest to one of them
        many = min(n, T // (chunk + 1))
        if many:
            counts = [chunk + 1] * many
            counts[0] += T - sum(counts)
            most = max(most, used(counts, chunk))
        assert most <= slots_of(T, n), (T, n, most)
        assert T <= chunk or slots_of(T, n) <= most + 2, (T, n, most)


def test_backward_workspace_of_a_long_batch(size):
    """65536 tokens, 4096 -> 14336, rank 64, eight adapters: 136 rows of 4.5 MiB, not 256 of them."""
    rows, row = 65536 // 512 + 8, 64 * (4096 + 14336) * 4
    assert size(65536, 8, 64, 4096, 14336, 1, 1) < rows * row + (1 << 29) + (1 << 27)
