"""The quotient by a reciprocal with which attention over scaled caches finds a workgroup's crew."""


def test_quotients_by_reciprocals_are_exact():
    # crews * units <= 512 where there are several crews; a unit of one is taken apart.
    for units in range(2, 257):
        reciprocal = -(-2 ** 32 // units)
        assert reciprocal < 2 ** 32
        for x in range(512 // units * units):
            assert x * reciprocal >> 32 == x // units
