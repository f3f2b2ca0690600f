"""The paged attention's schedule in plain Python (csrc/paged_attention.hip: cut_of, the workgroups' parts, the
joins' part numbers): every chunk of every item is taken once, every partial sum has a slot of its own, and each
join finds the parts of its item."""

import random

import pytest

CHUNK = 128


def cut_of(chunks, items, parts):
    if 2 * items <= parts:
        per = max(-(-chunks // (parts - items)), 1)
        return per, per
    return max(-(-chunks // parts), 1), 1


def rounded(n, unit):
    return -(-n // unit) * unit


def run(seqs, n_kv, rows_of_tile, parts):
    """seqs: (rows, keys) of each sequence; the parts of each item as (workgroup, first chunk, end, slot)."""
    shape = [(-(-rows // rows_of_tile), max(-(-keys // CHUNK), 1)) for rows, keys in seqs]
    per, unit = cut_of(sum(t * n_kv * c for t, c in shape), sum(t * n_kv for t, _ in shape), parts)
    first, total = [], 0
    for t, c in shape:
        first.append(total)
        total += t * n_kv * rounded(c, unit)
    taken, slots = {}, set()
    for w in range(parts):
        c, end, b = min(w * per, total), min(w * per + per, total), None
        for i, (t, k) in enumerate(shape):
            if first[i] <= c < first[i] + t * n_kv * rounded(k, unit):
                b = i
        seq0 = None if b is None else first[b]
        while c < end and b < len(seqs):
            t, k = shape[b]
            span = rounded(k, unit)
            if c >= seq0 + span * t * n_kv:
                seq0, b = seq0 + span * t * n_kv, b + 1
                continue
            item = (c - seq0) // span
            item0 = seq0 + item * span
            j0, j1 = c - item0, min(k, end - item0)
            assert 0 <= j0 < j1 <= k
            slot = None
            if not (j0 == 0 and j1 == k):
                slot = 2 * w + (1 if j0 == 0 else 0)
                assert slot not in slots and slot < 2 * parts
                slots.add(slot)
            taken.setdefault((b, item), []).append((w, j0, j1, slot))
            c = item0 + span
    return shape, first, total, per, unit, taken


@pytest.mark.parametrize("seed", range(60))
def test_every_chunk_once_and_joins_find_their_parts(seed):
    rng = random.Random(seed)
    n = rng.choice([1, 2, 7, 40, 100])
    seqs = [(rng.choice([0, 1, 6, 30, 70]), rng.choice([0, 1, 127, 128, 129, 5000, rng.randrange(9000)]))
            for _ in range(n)]
    n_kv, tile, most = rng.choice([1, 2, 8]), rng.choice([16, 32, 64]), rng.choice([1, 3, 64, 256, 512])
    # the host's bound of the list, by which it sets the number of parts
    items = (sum(r for r, _ in seqs) // tile + n) * n_kv
    parts = max(min(items * max(-(-max(k for _, k in seqs) // CHUNK), 1) + items, most), 1)
    shape, first, total, per, unit, taken = run(seqs, n_kv, tile, parts)
    for b, (tiles, chunks) in enumerate(shape):
        for item in range(tiles * n_kv):
            got = taken[b, item]
            assert [j for _, j0, j1, _ in got for j in range(j0, j1)] == list(range(chunks))
            c0 = first[b] + item * rounded(chunks, unit)
            w0, w1 = c0 // per, (c0 + chunks - 1) // per
            assert w1 < parts and [w for w, _, _, _ in got] == list(range(w0, w1 + 1))
            if w0 != w1:
                assert [s for _, _, _, s in got] == [2 * w0 + 1] + [2 * w for w in range(w0 + 1, w1 + 1)]
            # the join by workgroups: the one whose part the item begins in finds it at its part's end
            end = w0 * per + per
            if w0 != w1:
                assert end < total
                at = max(i for i in range(len(seqs)) if first[i] <= end - 1)
                assert at == b and (end - 1 - first[b]) // rounded(chunks, unit) == item


def test_items_cut_for_themselves_fit_the_parts():
    for items in range(1, 60):
        for parts in range(2 * items, 2 * items + 90, 7):
            for chunks in (items, items + 1, 10 * items + 3, 997 * items):
                per, unit = cut_of(chunks, items, parts)
                assert unit == per and chunks // per + items <= parts


def test_parts_are_dealt_to_xcds_in_runs():
    """The order of the parts where sequences have several row tiles: each taken once, and the workgroups of an XCD
    (every eighth) take neighbouring ones."""
    for used in list(range(1, 70)) + [255, 256, 509, 512]:
        part = [(w & 7) * (used >> 3) + min(w & 7, used & 7) + (w >> 3) for w in range(used)]
        assert sorted(part) == list(range(used))
        for x in range(8):
            mine = part[x::8]
            assert mine == list(range(mine[0], mine[0] + len(mine))) if mine else True
