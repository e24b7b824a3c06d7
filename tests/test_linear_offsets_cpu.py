"""Offsets of packed sequences that are out of order or out of range, walked as the kernels of linear attention's prompts walk them (items, places of
segments): nothing outside the tokens and the workspace is reached (no GPU needed)."""
import random

import pytest

CHUNK = 64


def walk(cu, total, seg_chunks, per, items):
    """(first token, tokens, place, place of the state before it or None, segments) of every item, as LinWalker::locate finds them."""
    def offset(i):
        return min(max(cu[i], 0), total)
    slots = []
    for s in range(len(cu) - 1):
        b = offset(s)
        n = max(offset(s + 1), b) - b
        segments = max(1, -(-(-(-n // CHUNK)) // seg_chunks))
        slots += [(b, n, i, segments) for i in range(segments)]
    for it in range(items):
        if it // per >= len(slots):
            continue
        b, n, segment, segments = slots[it // per]
        if segments > 1:
            b, n = b + segment * seg_chunks * CHUNK, min(n - segment * seg_chunks * CHUNK, seg_chunks * CHUNK)
        before = None
        if segment > 0:
            before = it - per
        elif segments > 1 and it // per + segments <= items // per:
            before = it + (segments - 1) * per
        yield b, n, it, before, segments


def joined(cu, total, seg_chunks, per, items, chain):
    """(places that the joining launch reads and writes, place of the initial state or None) of a chain, as gdn_linear_combine_kernel has it."""
    seq, rest = divmod(chain, per)
    first = 0
    for s in range(seq + 1):
        b = min(max(cu[s], 0), total)
        segments = max(1, -(-(-(-(min(max(cu[s + 1], b), total) - b) // CHUNK)) // seg_chunks))
        first += segments if s < seq else 0
    n = min(segments - 1, items // per - first)
    return [(first + i) * per + rest for i in range(max(n, 0))], (first + n) * per + rest if n > 0 and first + segments <= items // per else None


def check(cu, total, seg_chunks, per):
    seqs = len(cu) - 1
    items = (seqs + total // (CHUNK * seg_chunks)) * per
    for b, n, place, before, segments in walk(cu, total, seg_chunks, per, items):
        assert 0 <= b and 0 <= n and b + n <= total, (b, n)
        assert before is None or 0 <= before < items
        assert segments == 1 or n > 0
    for chain in range(seqs * per):
        places, initial = joined(cu, total, seg_chunks, per, items, chain)
        assert all(0 <= p < items for p in places) and (initial is None or 0 <= initial < items)


@pytest.mark.parametrize("cu,total", [([0, 64, 64, 130], 150), ([0, 90, 40, 1 << 30], 150), ([-5, -1, 2000, 149], 150), ([0, 6000, 0, 6000, 0, 6000], 6000),
                                      ([6000, 0, 6000], 6000), ([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], 6000), ([5999, 5999, 6001], 6000)], ids=str)
@pytest.mark.parametrize("seg_chunks,per", [(1, 1), (4, 2), (9, 6)])
def test_given(cu, total, seg_chunks, per):
    check(cu, total, seg_chunks, per)


def test_drawn():
    rng = random.Random(0)
    for _ in range(300):
        total = rng.randint(1, 5000)
        check([rng.randint(-100, total + 200) for _ in range(rng.randint(2, 40))], total, rng.randint(1, 12), rng.randint(1, 8))
