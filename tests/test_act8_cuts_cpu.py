"""How calls on 8-bit activations are cut, by the rules of ek_internal.h compiled for the host: against times measured on
MI355X, and that every cut's items cover the rows and fit their lists."""
import pytest

import act8_rules

pytestmark = pytest.mark.skipif(not act8_rules.available(), reason="no g++ or no HIP headers")


# hidden, inter, rows of the calls, us streamed in items of up to 64 rows, us with tiles for the calls of more than 16 rows
MEASURED = [
    (7168, 2048, [20], 50, 75), (7168, 2048, [40], 48, 82), (7168, 2048, [200], 67, 135), (7168, 2048, [500], 102, 152),
    (7168, 2048, [20] * 4, 80, 99), (7168, 2048, [100] * 4, 168, 146), (7168, 2048, [200] * 4, 251, 215), (7168, 2048, [40] * 16, 318, 198),
    (7168, 2048, [1] * 4 + [40] * 4, 143, 146), (7168, 2048, [1] * 4 + [100] * 4, 199, 183), (7168, 2048, [1] * 4 + [40] * 16, 346, 234),
    (7168, 2048, [1] * 16 + [20], 182, 197), (7168, 2048, [1] * 16 + [40], 189, 209), (7168, 2048, [1] * 16 + [100], 216, 245),
    (7168, 2048, [1] * 16 + [200], 267, 310), (7168, 2048, [1] * 16 + [100] * 4, 285, 253), (7168, 2048, [1] * 16 + [40] * 16, 429, 307),
    (7168, 2048, [8] * 40 + [20], 357, 372), (7168, 2048, [8] * 40 + [200], 446, 486), (7168, 2048, [8] * 40 + [100] * 4, 465, 430),
    (7168, 2048, [8] * 40 + [40] * 16, 606, 486),
    (2048, 768, [40], 35, 45), (2048, 768, [200], 35, 73), (2048, 768, [100] * 4, 61, 78), (2048, 768, [1] * 4 + [500], 99, 139),
    (2048, 768, [1] * 16 + [200] * 4, 95, 128), (2048, 768, [8] * 40 + [200], 108, 148), (2048, 768, [8] * 40 + [40] * 16, 130, 135)]


def test_batches_of_calls_take_the_faster_cut():
    got = act8_rules.ask([f"b {h} {i} {len(r)} " + " ".join(map(str, r)) for h, i, r, _, _ in MEASURED])
    for (h, i, r, streamed, tiles), (pick,) in zip(MEASURED, got):
        assert (streamed if pick else tiles) <= 1.05 * min(streamed, tiles), (h, i, r)


def test_a_batch_without_long_calls_has_no_tiles():
    assert act8_rules.ask(["b 7168 2048 0", "b 7168 2048 3 1 16 0", "b 2048 768 1 16"]) == [[0], [0], [0]]


def test_items_cover_their_segment():
    sizes = list(range(1, 1100)) + [4096, 4097, 65535, 131071]
    for n, out in zip(sizes, act8_rules.ask([f"i {n}" for n in sizes])):
        at = 0
        for first, rows in zip(out[::2], out[1::2]):
            assert first == at and 1 <= rows <= 256 and (first + rows == n or rows % 32 == 0), (n, out)
            at += rows
        assert at == n and len(out) // 2 == (n + 255) // 256


def test_lists_hold_every_cut():
    """The worst routings for each class: as many segments of the class's shortest length as there are experts or pairs for."""
    calls = [(P, E, h, i) for P in (1, 15, 16, 17, 64, 200, 1024, 1025, 5000, 65536) for E in (1, 3, 16, 40, 128, 256) for h, i in ((256, 192), (7168, 2048))]
    for (P, E, h, i), (k, stream, tile) in zip(calls, act8_rules.ask([f"c {P} {E} {h} {i}" for P, E, h, i in calls])):
        if k == 3:
            worst_stream, worst_tile = P // 64 + min(P, E), 0
        else:
            least = 1 if k == 2 else 17
            segments = min(E, P // least)
            worst_tile = segments + max(0, P - segments * least) // 256
            worst_stream = 0 if k == 2 else min(P, E)
        assert stream >= worst_stream and tile >= worst_tile, (P, E, k)
