"""The Python layer works out most workspaces of the int8 layers itself: they are those of the C size calls."""
import random

import pytest

from cuop_b200 import _native as N
from cuop_b200 import int8 as I
from test_weight_operators_cpu import A


@pytest.mark.parametrize("gated", [False, True])
def test_scratch_is_what_the_size_call_says(gated):
    size = N.lib().cuopx_int8_gated_linear_workspace_size if gated else N.lib().cuopx_int8_linear_workspace_size
    rng = random.Random(1)
    sizes = [0, 1, 2, 3, 8, 15, 16, 17, 31, 64, 65, 100, 128, 129, 500, 512, 1000, 1024, 4095, 4096, 8191, 8192, 8193, 20000]
    edges = [(1, n, k) for n in (1, 8192, 9000, 20000) for k in (8192, 8193)] + [(8, 1024, 1024), (8, 1024, 1025), (16, 512, 512),
                                                                                (17, 481, 481), (16, 513, 512), (2, 4096, 4097)]
    for case in range(6000):
        m, n, k = edges[case] if case < len(edges) else (rng.choice(sizes) for _ in range(3))
        ldx, ldw = (k + rng.choice((0, 1, 8, 16, -k % 16)) for _ in range(2))
        given = rng.random() < 0.4
        head = (rng.choice((N.F16, N.BF16)), 0, m, n, k, A + 2 * rng.choice((0, 0, 0, 4, 8)), ldx, 6 * A if given else 0,
                2 * A + rng.choice((0, 0, 0, 1, 8, 16)), ldw, 3 * A, 0, 0, 0, 4 * A, n)
        assert I._scratch(size, head) == size(I._INT8.pack(*head, 0, 0)), head
