"""The quotients by reciprocals with which kernels find a workgroup's crew, and a row's token and head."""

import random


def test_crews():
    # crews * units <= 512 where there are several crews; a unit of one is taken apart.
    for units in range(2, 257):
        reciprocal = -(-2 ** 32 // units)
        assert reciprocal < 2 ** 32
        for x in range(512 // units * units):
            assert x * reciprocal >> 32 == x // units


def test_rows():
    rng = random.Random(1)
    top = 2 ** 31
    for d in [*range(1, 300), *(rng.randrange(1, 2 ** 30) for _ in range(300)), 2 ** 29 + 1, 2 ** 30 - 1, 2 ** 30]:
        shift = (d - 1).bit_length()
        m = -(-2 ** (31 + shift) // d) if shift else 0
        assert m < 2 ** 32
        last = (top - 1) // d * d
        for n in [0, 1, d - 1, d, d + 1, last, max(last - 1, 0), top - 1, *(rng.randrange(top) for _ in range(20))]:
            assert (n if shift == 0 else (n * m >> 32) >> (shift - 1)) == n // d
