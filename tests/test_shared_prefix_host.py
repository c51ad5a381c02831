"""The layout of shared prefixes, checked without a GPU."""
import random

import pytest
import torch

from rvllm_b200.errors import KernelError
from rvllm_b200.kernels import SharedPrefixes


def unpack(s):
    """The array as the kernels read it (csrc/shared_prefix.cuh)."""
    v, B = s.device_ints.tolist(), s.num_seqs
    tiles, items = s.capacity
    at = (4 + 3 * B + 2 * tiles + 3) // 4 * 4
    ranges = [v[at + 8 * i:at + 8 * i + 8] for i in range(items)]
    rows = {r[5]: r[2:5] for r in ranges[:v[0]]}
    return dict(items_used=v[0], tiles_used=v[1], own_start=v[4:4 + B], place=v[4 + B:4 + 2 * B], members=v[4 + 2 * B:4 + 3 * B],
                parts=[v[4 + 3 * B + 2 * i:4 + 3 * B + 2 * i + 2] for i in range(tiles)], tiles=rows, items=ranges, size=len(v))


@pytest.mark.parametrize("seed", range(12))
def test_every_row_and_key_once(seed):
    rng = random.Random(seed)
    nkv = rng.choice((1, 2, 4, 8))
    nh = nkv * rng.choice((1, 2, 4, 7, 32, 128))
    B = rng.randint(1, 300)
    free = list(range(B))
    rng.shuffle(free)
    groups = []
    while free and rng.random() < 0.8:
        n = rng.randint(1, min(len(free), 200))
        groups.append(([free.pop() for _ in range(n)], rng.choice((0, 1, 63, 64, 65, rng.randint(1, 40000)))))
    s = SharedPrefixes(groups, B, nh, nkv, "cpu")
    u = unpack(s)
    assert u["size"] == SharedPrefixes.ints(B, s.capacity)
    per = nh // nkv
    of = {m: (g, t) for g, (ms, t) in enumerate(groups) for m in ms if len(ms) > 1 and t > 0}
    rows = set()
    for b in range(B):
        if b not in of:
            assert u["own_start"][b] == 0 and u["place"][b] == -1
            continue
        tile, row = divmod(u["place"][b], 128)
        seq, first, count = u["tiles"][tile]
        assert of[b][1] == u["own_start"][b] and seq in groups[of[b][0]][0]
        assert row % per == 0 and row + per <= 128 and u["members"][first + row // per] == b and row // per < count
        rows.add((tile, row))
    assert len(rows) == len(of)
    for t in range(u["tiles_used"]):
        first, n = u["parts"][t]
        at = 0
        for lo, hi, seq, _, _, tile, _, _ in u["items"][first:first + n]:
            assert tile == t and lo == at and lo % 64 == 0 and lo < hi
            at = hi
        assert at == u["own_start"][u["tiles"][t][0]]
    assert u["items_used"] == sum(n for _, n in u["parts"][:u["tiles_used"]])


def test_ranges_fill_the_places_once():
    s = SharedPrefixes([(list(range(64)), 4096)], 64, 32, 8, "cpu")
    assert s.num_tiles == 2 and 0.6 * 148 < s.num_items * 8 <= 148
    s = SharedPrefixes([(list(range(4)), 32768)], 4, 32, 8, "cpu")
    assert 0.9 * 296 < s.num_items * 8 <= 296


def test_a_capacity_fixes_the_size():
    sizes = {SharedPrefixes(g, 8, 16, 4, "cpu", capacity=(3, 90)).device_ints.numel() for g in ([], [([0, 1], 50)], [([0, 1], 50), ([5, 3, 2], 700)])}
    assert len(sizes) == 1
    with pytest.raises(KernelError):
        SharedPrefixes([([0, 1], 5), ([2, 3], 5)], 8, 16, 4, "cpu", capacity=(1, 90))
    with pytest.raises(KernelError):
        SharedPrefixes([([0, 1], 5000)], 8, 16, 4, "cpu", capacity=(1, 2))


@pytest.mark.parametrize("groups", [[([0, 0], 5)], [([0, 1], 5), ([1, 2], 5)], [([0, 9], 5)], [([-1, 0], 5)], [([0, 1], -1)], [([0, 1], 2 ** 31)]])
def test_refused_groups(groups):
    with pytest.raises(KernelError):
        SharedPrefixes(groups, 4, 8, 2, "cpu")


def test_refused_heads():
    for heads in ((8, 3), (0, 1), (8, 0)):
        with pytest.raises(KernelError):
            SharedPrefixes([], 4, *heads, "cpu")
    with pytest.raises(KernelError):
        SharedPrefixes([([0, 1], 5)], 4, 256, 1, "cpu")
