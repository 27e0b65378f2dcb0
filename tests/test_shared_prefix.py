"""The plan of the attention whose requests share prefixes, on the CPU: every key that a row sees is
in exactly one of the row's ranges, ranges have places of their own, and the places are the ones that
the merge looks at.  And what the launcher refuses."""

import numpy as np
import pytest
import torch

from distengine_b200.kernels.shared_prefix import SharedPrefixAttention, Tile, plan_shared

TILES = {
    "one": (Tile("rows", 8, 32, 592),) * 2,
    "two": (Tile("wide", 128, 128, 148), Tile("narrow", 16, 64, 592)),
    "few": (Tile("wide", 32, 64, 3), Tile("narrow", 8, 1, 5)),
    "places": (Tile("wide", 128, 128, 148, 2), Tile("narrow", 16, 64, 592)),
}
STEPS = {
    # tokens a request, requests a group, prefix a group, keys of its own before this step's tokens
    "beams": ([1] * 4, [4], [512], [20, 0, 3, 64]),
    "alone": ([1, 1, 1], [1, 1, 1], [700, 0, 33], [0, 5, 1]),
    "mixed": ([1, 1, 3, 1, 7, 2, 1], [3, 1, 2, 1], [1003, 50, 64, 0], [5, 0, 9, 100, 0, 300, 1]),
    "none": ([0, 1, 0, 0, 2], [2, 1, 2], [77, 40, 100], [0, 4, 0, 0, 8]),
    "many": ([1] * 130, [130], [4097], list(range(130))),
    "long": ([1] * 3, [3], [200_003], [0, 70_000, 5]),
    "nothing": ([], [], [], []),
}


def _seen(plan, tiles, group, kv_heads, qlen, sizes, prefix, own):
    """row of a token and query head -> how often each of its keys is in one of its ranges."""
    first = np.cumsum([0] + sizes[:-1])
    group_of = np.repeat(np.arange(len(sizes)), sizes)
    pos0 = [prefix[group_of[s]] + own[s] for s in range(len(qlen))]
    tok0 = np.cumsum([0] + qlen)[:-1]
    used = np.zeros(plan.partial_rows, dtype=int)
    by_row = {}
    rows_of = {t.name: t for t in tiles}
    for name, items in plan.items.items():
        t = rows_of[name]
        for it in items.tolist():
            at, n, row0, seq, begin, end, split, base = it
            assert 0 < n <= t.rows and 0 <= base and base + t.rows * t.places <= plan.partial_rows
            assert plan.shapes[name] == (t.rows, t.unit)
            used[base: base + t.rows * t.places] += 1
            if end < 0:                               # as range_of in the kernels' header
                assert at == tok0[seq]
                stop = max(begin, pos0[seq] + (row0 + n - 1) // group + 1)
                splits, part = split >> 16, split & 0xffff
                each = -(-(-(-(stop - begin) // splits)) // t.unit) * t.unit
                lo = min(stop, begin + part * each)
                hi = min(stop, lo + each)
            else:
                assert seq == first[group_of[seq]] and at == tok0[seq]
                lo, hi = begin, end
                assert begin < end and begin % t.unit == 0 and split == t.places - 1
            for r in range(n):
                token = at + (row0 + r) // group
                limit = hi
                if end < 0:
                    limit = min(hi, pos0[seq] + (row0 + r) // group + 1)
                by_row.setdefault((token, (row0 + r) % group), []).append(
                    (lo, max(lo, limit), base + r))
                if end >= 0 and split:                # the place of the range's other half
                    by_row[token, (row0 + r) % group].append((lo, lo, base + t.rows + r))
    assert (used == 1).all()
    return by_row, pos0, tok0


@pytest.mark.parametrize("tiles", sorted(TILES))
@pytest.mark.parametrize("step", sorted(STEPS))
@pytest.mark.parametrize("group,kv_heads", [(1, 1), (8, 4), (5, 3)])
@pytest.mark.parametrize("tail", [0, 100])
def test_every_key_once(tiles, step, group, kv_heads, tail):
    qlen, sizes, prefix, own = STEPS[step]
    wide, narrow = TILES[tiles]
    plan = plan_shared(qlen, sizes, prefix, group, kv_heads, lambda rows, keys: wide,
                       lambda rows, keys: narrow, tail)
    assert plan.tokens == sum(qlen) and plan.token_seq.tolist() == sum(
        ([s] * n for s, n in enumerate(qlen)), [])
    by_row, pos0, tok0 = _seen(plan, {wide, narrow}, group, kv_heads, qlen, sizes, prefix, own)
    assert len(by_row) == sum(qlen) * group
    for (token, head), ranges in by_row.items():
        s = int(plan.token_seq[token])
        at = 0
        for lo, hi, _ in sorted(ranges):
            if lo < hi:
                assert lo == at, (token, head)
                at = hi
        assert at == pos0[s] + token - tok0[s] + 1
        # the merge's places, as in shared_merge_kernel
        mine = plan.seqs[s].tolist()
        places = []
        for start, base, chunks, rows in ((mine[1], *mine[2:5]), (mine[0], *mine[5:8])):
            for c in range(chunks):
                r = (token - start) * group + head
                places.append(base + (r // rows * chunks + c) * rows + r % rows)
        assert sorted(places) == sorted(p for _, _, p in ranges)


def test_the_shared_prefix_is_read_once():
    """The keys that the items of a group's prefix name are the prefix, once a tile of rows."""
    wide, narrow = TILES["two"]
    plan = plan_shared([1] * 16, [16], [5000], 8, 8, lambda rows, keys: wide,
                       lambda rows, keys: narrow, 32)
    shared = plan.items["wide"]
    assert int((shared[:, 5] - shared[:, 4]).sum()) == 5000      # 128 rows: one tile
    assert (plan.items["narrow"][:, 4] == 5000).all()


def test_refused_plans():
    tile = TILES["one"][0]
    make = lambda *a, **k: plan_shared(*a, 4, 2, lambda r, k: tile, lambda r, k: tile, **k)
    for args in (([1, 1], [1], [5]), ([1, 1], [2, 0], [5, 5]), ([1, -1], [2], [5]),
                 ([1, 1], [2], [5, 6]), ([1, 1], [2], [-5]), ([1, 1], [3, -1], [5, 5])):
        with pytest.raises(ValueError, match="shared prefix"):
            make(*args)
    with pytest.raises(ValueError, match="shared prefix"):
        make([1, 1], [2], [5], tail=-1)
    with pytest.raises(ValueError, match="shared prefix"):
        make([1, 1], [2], [1 << 31])
    with pytest.raises(ValueError, match="shared prefix"):
        make([1 << 27], [1], [0])


def test_refused_layers():
    for args in ((torch.float16, 4, 2, 64, 0.1), (torch.bfloat16, 4, 3, 64, 0.1),
                 (torch.bfloat16, 4, 2, 63, 0.1), (torch.bfloat16, 4, 2, 258, 0.1),
                 (torch.bfloat16, 4, 2, 64, 0.0), (torch.bfloat16, 4, 2, 64, -1.0),
                 (torch.bfloat16, 4, 0, 64, 0.1), (torch.bfloat16, 0, 2, 64, 0.1),
                 (torch.bfloat16, 4, 2, 64, float("nan"))):
        with pytest.raises((ValueError, TypeError)):
            SharedPrefixAttention(*args)


def _call(**changed):
    heads, kv_heads, d = 4, 2, 16
    layer = SharedPrefixAttention(torch.float32, heads, kv_heads, d, 0.25, "cpu")
    tile = TILES["one"][0]
    plan = plan_shared([1, 1], [2], [16], heads // kv_heads, kv_heads, lambda r, k: tile,
                       lambda r, k: tile).to("cpu")
    args = dict(q=torch.zeros(2, heads * d), out=torch.zeros(2, heads * d),
                k_pages=torch.zeros(4, kv_heads, 16, d), v_pages=torch.zeros(4, kv_heads, 16, d),
                block_table=torch.zeros(2, 2, dtype=torch.int32),
                seq_slot=torch.zeros(2, dtype=torch.int32),
                seq_pos0=torch.full((2,), 16, dtype=torch.int32), plan=plan)
    args.update(changed)
    layer.run(**args)


@pytest.mark.parametrize("name,value", [
    ("q", torch.zeros(2, 64, dtype=torch.bfloat16)), ("q", torch.zeros(3, 64)),
    ("q", torch.zeros(2, 63)), ("q", torch.zeros(64, 2).t()), ("q", torch.zeros(1, 64).expand(2, 64)),
    ("out", torch.zeros(2, 65)), ("out", torch.zeros(1, 64)), ("out", torch.zeros(1, 64).expand(2, 64)),
    ("k_pages", torch.zeros(4, 2, 16, 17)), ("k_pages", torch.zeros(5, 2, 16, 16)),
    ("v_pages", torch.zeros(4, 16, 2, 16).transpose(1, 2)),
    ("k_pages", torch.zeros(4, 2, 16, 16, dtype=torch.bfloat16)),
    ("block_table", torch.zeros(2, 2)), ("block_table", torch.zeros(2, dtype=torch.int32)),
    ("seq_slot", torch.zeros(3, dtype=torch.int32)), ("seq_pos0", torch.zeros(2)),
])
def test_refused_calls(name, value):
    with pytest.raises(ValueError, match="shared prefix"):
        _call(**{name: value})


def test_a_call_off_the_current_device_is_refused():
    with pytest.raises(ValueError, match="current CUDA device"):
        _call()
    plan = plan_shared([1, 1], [2], [16], 2, 2, lambda r, k: TILES["one"][0],
                       lambda r, k: TILES["one"][0])
    with pytest.raises(ValueError, match="not on the device"):
        _call(plan=plan)


@pytest.mark.parametrize("group,kv_heads", [(4, 2), (2, 4), (1, 2), (4, 1)])
def test_a_plan_for_other_heads_is_refused(group, kv_heads):
    """Its rows would lie outside q."""
    from distengine_b200.kernels.shared_prefix import SharedPlan
    tile = TILES["one"][0]
    plan = plan_shared([1, 1], [2], [16], group, kv_heads, lambda r, k: tile, lambda r, k: tile)
    with pytest.raises(ValueError, match="shared prefix: the plan"):
        _call(plan=plan.to("cpu"))
    with pytest.raises(ValueError, match="shared prefix: the plan"):
        _call(plan=SharedPlan(plan.items, plan.shapes, plan.seqs, plan.token_seq, plan.partial_rows,
                              plan.most_parts, plan.tokens).to("cpu"))


def test_a_plan_keeps_its_heads():
    tile = TILES["places"][0]
    plan = plan_shared([1, 1], [2], [16], 5, 3, lambda r, k: tile, lambda r, k: tile).to("cpu")
    assert (plan.group, plan.kv_heads, plan.turns) == (5, 3, True)


@pytest.mark.parametrize("scale", [1e-46, 1e-40, 1e39, 1e300])
def test_scales_that_are_no_float32_numbers_are_refused(scale):
    """The kernels take it as one: 0 or an infinity would make every result NaN.  A launcher that may share
    does not then."""
    from distengine_b200.kernels.attention import AttentionLauncher
    with pytest.raises(ValueError, match="shared prefix: the scale"):
        SharedPrefixAttention(torch.float32, 4, 2, 64, scale)
    assert AttentionLauncher(torch.float32, 4, 2, 64, scale, None, share=True).shared is None
    SharedPrefixAttention(torch.float32, 4, 2, 64, 1e-30)
