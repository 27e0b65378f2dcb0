"""Selection of the next beams and reordering of their rows, against the definitions in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, NAN = float("inf"), float("nan")


def _select(logits, scores, take, scratch=None):
    from distengine_b200.kernels import ops
    groups = scores.shape[0]
    best = torch.full((groups, take), 5.0, device=DEV)
    beam, token = (torch.full((groups, take), 77, dtype=torch.int32, device=DEV) for _ in range(2))
    ops.beam_select(logits, scores, best, beam, token, scratch)
    torch.cuda.synchronize()
    return best.cpu(), beam.cpu(), token.cpu()


def _want(logits, scores, take):
    """Candidates ordered by total (64 bits), then beam, then logit, then token.  The sums of
    exponentials are correctly rounded (``fsum``): rows of the same logits in another order tie."""
    groups, beams = scores.shape
    vocabulary = logits.shape[1]
    x = logits.double().cpu()
    x = x - x.amax(1, keepdim=True)
    sums = torch.tensor([math.fsum(row) for row in x.exp().tolist()], dtype=torch.float64)
    total = scores.double().cpu().view(-1, 1) + (x - sums.log()[:, None])
    total = torch.where(total.isnan(), -INF, total).view(groups, -1)
    best = torch.full((groups, take), -INF, dtype=torch.float64)
    beam, token = (torch.full((groups, take), -1, dtype=torch.int32) for _ in range(2))
    for g in range(groups):
        order = total[g].sort(descending=True, stable=True).indices[:take]
        order = order[total[g][order] > -INF]
        best[g, : len(order)] = total[g][order]
        beam[g, : len(order)] = (order // vocabulary).int()
        token[g, : len(order)] = (order % vocabulary).int()
    return best, beam, token


def _check(logits, scores, take, **how):
    best, beam, token = _select(logits.to(DEV), scores.to(DEV), take, **how)
    want, want_beam, want_token = _want(logits, scores, take)
    assert torch.equal(beam, want_beam) and torch.equal(token, want_token)
    there = want > -INF
    assert torch.equal(best > -INF, there)
    # one rounding to float32 of a total in 64 bits; the sum of exponentials is off by up to 2e-6 of
    # itself (csrc/beam.cu), which is as much off the total
    off = (best.double() - want).abs()[there]
    assert bool((off <= 2.0 ** -24 * want.abs()[there] + 2e-6).all()), off.max().item()


def _inputs(groups, beams, vocabulary, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(groups * beams, vocabulary, generator=g) * std
    return logits, -10.0 + torch.randn(groups, beams, generator=g)


@pytest.mark.parametrize("groups,beams,vocabulary,take", [
    (1, 1, 1, 1), (1, 1, 1, 4), (2, 3, 2, 6), (1, 4, 7, 64), (3, 2, 31, 5), (1, 4, 32000, 8),
    (5, 5, 50021, 10), (64, 8, 1003, 16), (2, 32, 4097, 64), (1, 32, 128256, 64), (7, 1, 33000, 2),
    (1, 2, 151_936, 3), (300, 2, 517, 4), (1, 1, 300_007, 64)])
def test_sizes(groups, beams, vocabulary, take):
    _check(*_inputs(groups, beams, vocabulary, vocabulary), take)


@pytest.mark.parametrize("std", [0.01, 1.0, 30.0, 1e4])
def test_distributions(std):
    """Nearly even rows, where scores decide, and rows in which one token has all."""
    _check(*_inputs(6, 4, 32001, int(std), std), 8)
    logits, scores = _inputs(6, 4, 32001, 5, std)
    _check(logits, scores * 50, 8)


def test_strides():
    logits, scores = _inputs(3, 4, 1001, 1)
    for pad in (1, 3, 4, 24):
        wide = torch.full((12, 1001 + pad), 1e9, device=DEV)
        wide[:, :1001] = logits
        best, beam, token = _select(wide[:, :1001], scores.to(DEV), 8)
        _, want_beam, want_token = _want(logits, scores, 8)
        assert torch.equal(beam, want_beam) and torch.equal(token, want_token)
    whole = torch.full((12 * 1001 + 3,), 1e9, device=DEV)       # rows off any 16-byte boundary
    whole[3:] = logits.flatten()
    _, beam, token = _select(whole[3:].view(12, 1001), scores.to(DEV), 8)
    assert torch.equal(beam, want_beam) and torch.equal(token, want_token)


@pytest.mark.parametrize("vocabulary", [9, 1000, 32000, 128256])
@pytest.mark.parametrize("take", [1, 8, 64])
def test_equal_logits(vocabulary, take):
    """Ties: lower beam, then lower token, whether all are equal or the last place is."""
    scores = torch.tensor([[-1.0, -1.0, -1.0], [-2.0, -1.0, -1.0]])
    _check(torch.zeros(6, vocabulary), scores, take)
    _check(torch.full((6, vocabulary), -7.5), scores, take)
    logits = torch.zeros(6, vocabulary)
    logits[:, -3:] = 1.0
    logits[:, 4] = 2.0
    _check(logits, scores, take)
    signed = torch.zeros(6, vocabulary)
    signed[:, ::2] = -0.0
    _check(signed, scores, take)
    few = torch.randint(-2, 3, (6, vocabulary), generator=torch.Generator().manual_seed(take)).float()
    _check(few, scores, take)


def test_sorted_rows():
    """Rows that rise or fall: the best tokens are in one place."""
    for vocabulary in (40, 32000, 128256):
        up = torch.linspace(-5, 5, vocabulary).repeat(4, 1)
        down = up.flip(1)
        scores = torch.tensor([[-1.0, -1.25, -1.5, -0.5]])
        for x in (up, down, torch.cat((up[:2], down[:2]))):
            _check(x, scores, 64)


@pytest.mark.parametrize("vocabulary", [50, 32000])
def test_masks(vocabulary):
    """Masked tokens, rows with no token left, beams that are dead, groups with nothing."""
    logits, scores = _inputs(5, 4, vocabulary, 3)
    drop = torch.rand(logits.shape, generator=torch.Generator().manual_seed(4))
    logits[drop < 0.9] = -INF
    logits[3] = -INF
    logits[4:8] = -INF
    logits[5, 17] = 1.0
    logits[8:12] = -INF
    scores[3, 1:] = -INF
    scores[4] = -INF
    _check(logits, scores, 8)
    _check(logits, scores, 64)
    _check(torch.full((4, vocabulary), torch.finfo(torch.float32).min),
           torch.tensor([[0.0, -1.0], [-INF, 0.0]]), 4)


def test_values_that_are_not_finite():
    """A row with NaN or plus infinity has no candidates; the other rows keep theirs."""
    logits, scores = _inputs(4, 3, 5000, 6)
    logits[0, 4000], logits[4, 0], logits[5, 10] = NAN, INF, NAN
    logits[7] = NAN
    logits[9, 1:9] = torch.tensor([INF, NAN, -INF, INF, 3.0, INF, NAN, INF])
    scores[2, 0] = NAN
    _check(logits, scores, 6)


@pytest.mark.parametrize("gap", [0.0, 1e-9, 3e-8, 1e-7, 1e-6])
@pytest.mark.parametrize("vocabulary", [300, 32000])
def test_nearly_equal_totals(gap, vocabulary):
    """Candidates of different beams whose totals are closer than float32 can tell apart."""
    g = torch.Generator().manual_seed(vocabulary)
    for trial in range(6):
        logits = torch.randn(8, vocabulary, generator=g) * 2
        scores = torch.zeros(2, 4)
        # scores that bring the rows' best totals together, as near as float32 scores can
        top = torch.log_softmax(logits.double(), 1).amax(1).view(2, 4)
        scores = (-3.0 - top + gap * torch.arange(4)).float()
        _check(logits, scores, 8)
        # the same row twice, then once with its tokens turned round: the sums differ by order only
        logits[1], logits[2] = logits[0], logits[0].flip(0)
        _check(logits, torch.full((2, 4), -1.0), 8)


@pytest.mark.parametrize("vocabulary", [517, 32001, 50021, 128257])
@pytest.mark.parametrize("take", [1, 2, 5])
def test_the_last_place_among_equal_totals(vocabulary, take):
    """Two beams with one row, in which more tokens are equal than are taken: the lower beam has every place,
    also where the other one's sum comes out larger and its tokens would fill the list."""
    g = torch.Generator().manual_seed(vocabulary + take)
    for _ in range(3):
        row = torch.randn(6, vocabulary, generator=g) * 2
        for r in row:
            r[torch.randperm(vocabulary, generator=g)[: take + 2]] = float(r.max()) + 1.0
        _check(row.repeat_interleave(2, 0), torch.full((6, 2), -1.0), take)


@pytest.mark.parametrize("take", [1, 2, 3, 9])
def test_the_last_place_among_many_beams(take):
    """Eight beams whose best totals are nearly equal: whoever has the last place is compared with all."""
    g = torch.Generator().manual_seed(take)
    for vocabulary in (300, 32001):
        logits = torch.randn(96, vocabulary, generator=g) * 2
        top = torch.log_softmax(logits.double(), 1).amax(1).view(12, 8)
        _check(logits, (-3.0 - top).float(), take)


@pytest.mark.parametrize("vocabulary", [5000, 128256, 1 << 20, 1 << 24])
@pytest.mark.parametrize("part", [0.5, 0.99, 1.01, 1.5])
def test_nearly_equal_totals_of_peaked_rows(vocabulary, part):
    """A token that has nearly all and, behind it, very many that have next to nothing: together they are what
    decides.  One beam's total is ``part`` of their weight above, less that weight; the other's is 0."""
    bits = vocabulary.bit_length()
    for least in (bits - 64.0, bits - 63.1, -46.1):              # logarithms to base 2 of one token's weight
        logits = torch.full((2, vocabulary), -200.0)
        logits[0] = least * math.log(2.0)
        logits[:, vocabulary // 3] = 0.0
        weight = math.log1p((vocabulary - 1) * math.exp(float(logits[0, 0])))
        scores = torch.tensor([[part * weight, 0.0]], dtype=torch.float32)
        assert weight < 1e-4 and abs(float(scores[0, 0]) / weight - part) < 1e-6
        _, beam, token = _select(logits.to(DEV), scores.to(DEV), 1)
        assert token.tolist() == [[vocabulary // 3]]
        assert beam.tolist() == [[0 if part > 1.0 else 1]], (least, weight)


def test_streams_and_graphs():
    """Two captured selections replayed side by side."""
    from distengine_b200.kernels import ops
    jobs = []
    for seed in range(2):
        logits, scores = (t.to(DEV) for t in _inputs(3, 4, 9001, seed))
        out = (torch.zeros(3, 8, device=DEV), torch.zeros(3, 8, dtype=torch.int32, device=DEV),
               torch.zeros(3, 8, dtype=torch.int32, device=DEV))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ops.beam_select(logits, scores, *out)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.beam_select(logits, scores, *out)
        jobs.append((stream, graph, logits, scores, out))
    for _ in range(20):
        for stream, graph, *_ in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, logits, scores, out in jobs:
        _, beam, token = _want(logits, scores, 8)
        assert torch.equal(out[1].cpu(), beam) and torch.equal(out[2].cpu(), token)


def test_scratch_of_the_caller():
    from distengine_b200.kernels import ops
    logits, scores = _inputs(3, 4, 9001, 2)
    size = ops.beam_scratch(3, 4, 9001, 8)
    scratch = torch.full((size + 64,), 255, dtype=torch.uint8, device=DEV)
    for _ in range(2):                              # whatever it holds before
        _check(logits, scores, 8, scratch=scratch[:size])
        assert bool((scratch[size:] == 255).all())
    with pytest.raises(ValueError, match="scratch"):
        _select(logits.to(DEV), scores.to(DEV), 8, scratch[: size - 1])


def test_refusals_of_the_selection():
    f = lambda *shape: torch.zeros(*shape, device=DEV)
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)
    from distengine_b200.kernels import ops
    good = dict(logits=f(6, 50), scores=f(2, 3), best=f(2, 4), beam=i(2, 4), token=i(2, 4))
    ops.beam_select(**good)
    for name, value in (("logits", f(5, 50)), ("logits", f(6, 50).double()), ("logits", f(50, 6).t()),
                        ("logits", f(1, 50).expand(6, 50)), ("logits", f(6, 0)), ("scores", f(3, 2).t()),
                        ("scores", f(6)), ("best", f(2, 65)), ("best", f(2, 0)), ("beam", f(2, 4)),
                        ("token", i(2, 5)), ("token", i(4, 2).t()), ("best", f(2, 8)[:, ::2]),
                        ("scores", f(2, 3).cpu()), ("logits", f(6, 50).cpu())):
        with pytest.raises(ValueError):
            ops.beam_select(**{**good, name: value})
    with pytest.raises(ValueError):
        ops.beam_select(f(33, 5), f(1, 33), f(1, 4), i(1, 4), i(1, 4))
    ops.beam_select(f(0, 5), f(0, 3), f(0, 4), i(0, 4), i(0, 4))          # no groups: nothing to do


# ------------------------------------------------------------------------------- reordering
def _moved(rows, slots, parent):
    want = rows.clone()
    for g in range(slots.shape[0]):
        for b in range(slots.shape[1]):
            if slots[g, b] >= 0 and parent[g, b] >= 0:
                want[:, slots[g, b]] = rows[:, slots[g, parent[g, b]]]
    return want


def _reorder(rows, slots, parent):
    from distengine_b200.kernels import ops
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.beam_reorder(rows, slots.to(DEV), parent.to(DEV), status)
    torch.cuda.synchronize()
    return int(status.item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8, torch.float64])
@pytest.mark.parametrize("shape", [(1, 9, 1), (3, 40, 7), (2, 70, 16, 5), (4, 33, 2048), (1, 40, 100_003)])
@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 4), (2, 4), (4, 8), (1, 9), (1, 32), (8, 3)])
def test_rows_change_places(dtype, shape, groups, beams):
    if groups * beams > shape[1]:
        return
    g = torch.Generator().manual_seed(beams)
    rows = torch.randint(0, 250, shape, generator=g).to(dtype)
    slots = torch.randperm(shape[1], generator=g)[: groups * beams].view(groups, beams).int()
    for parent in (torch.randint(0, beams, (groups, beams), generator=g).int(),
                   torch.arange(beams).flip(0).repeat(groups, 1).int(),
                   torch.arange(beams).roll(1).repeat(groups, 1).int(),
                   torch.zeros(groups, beams, dtype=torch.int32),
                   torch.arange(beams).repeat(groups, 1).int()):
        device = rows.to(DEV)
        assert _reorder(device, slots, parent) == 0
        assert torch.equal(device.cpu(), _moved(rows, slots, parent))


def test_rows_off_alignment():
    whole = torch.arange(2 * 10 * 33 + 1, dtype=torch.int32, device=DEV)
    rows = whole[1:].view(2, 10, 33)
    before = rows.cpu().clone()
    slots, parent = torch.tensor([[7, 2, 5]], dtype=torch.int32), torch.tensor([[1, 2, 0]], dtype=torch.int32)
    assert _reorder(rows, slots, parent) == 0
    assert torch.equal(rows.cpu(), _moved(before, slots, parent)) and int(whole[0]) == 0


def test_beams_that_stay():
    """-1: a beam without a row, or without a parent."""
    rows = torch.randn(2, 12, 100)
    slots = torch.tensor([[3, -1, 5, 7], [-1, -1, 0, 1]], dtype=torch.int32)
    parent = torch.tensor([[2, 0, -1, 0], [0, 1, 3, 2]], dtype=torch.int32)
    device = rows.to(DEV)
    assert _reorder(device, slots, parent) == 0
    assert torch.equal(device.cpu(), _moved(rows, slots, parent))


def test_what_cannot_be_moved_stays():
    rows = torch.randn(2, 12, 100)
    for slots, parent, moved in (
            ([[3, 12, 5]], [[1, 0, 0]], {5: 3}),               # a slot behind the pool; beam 0's source
            ([[3, -2, 5]], [[2, 0, 1]], {3: 5}),
            ([[3, 4, 5]], [[3, 0, 1]], {4: 3, 5: 4}),          # no such parent
            ([[3, -1, 5]], [[1, 0, 0]], {5: 3}),               # the parent has no row
            ([[3, 4, 3]], [[1, 0, 1]], {}),                    # a row named twice
            ([[3, 4], [4, 6], [7, 8]], [[1, 0]] * 3, {7: 8, 8: 7})):
        device = rows.to(DEV)
        status = _reorder(device, torch.tensor(slots, dtype=torch.int32),
                          torch.tensor(parent, dtype=torch.int32))
        want = rows.clone()
        for to, source in moved.items():
            want[:, to] = rows[:, source]
        assert status == 5 and torch.equal(device.cpu(), want), (slots, parent)


def test_a_parent_below_minus_one_is_no_parent():
    rows = torch.randn(2, 12, 100)
    device = rows.to(DEV)
    assert _reorder(device, torch.tensor([[3, 4, 5]], dtype=torch.int32),
                    torch.tensor([[-2, 0, -1]], dtype=torch.int32)) == 5
    want = rows.clone()
    want[:, 4] = rows[:, 3]
    assert torch.equal(device.cpu(), want)


def test_refusals_of_the_reordering():
    from distengine_b200.kernels import ops
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)
    rows = torch.zeros(2, 8, 16, device=DEV)
    for args in ((rows.transpose(0, 1), i(1, 2), i(1, 2)), (rows[0, 0], i(1, 2), i(1, 2)),
                 (rows, i(1, 2), i(1, 3)), (rows, i(1, 33), i(1, 33)), (rows, i(2), i(2)),
                 (rows, i(1, 2).long(), i(1, 2)), (rows, i(1, 2).cpu(), i(1, 2)),
                 (rows.cpu(), i(1, 2), i(1, 2)), (rows, i(2, 1).t(), i(1, 4)[:, ::2])):
        with pytest.raises(ValueError):
            ops.beam_reorder(*args)
    with pytest.raises(ValueError, match="status"):
        ops.beam_reorder(rows, i(1, 2), i(1, 2), torch.zeros(1, device=DEV))
    ops.beam_reorder(rows, i(0, 2), i(0, 2))
    ops.beam_reorder(rows[:0], i(1, 2), i(1, 2))


def test_large_rows_and_graphs():
    """Offsets beyond 32 bits, and a captured call whose parents change between replays."""
    from distengine_b200.kernels import ops
    rows = torch.zeros(5, 9, 30_000_000, dtype=torch.int32, device=DEV)
    rows += torch.arange(45, dtype=torch.int32, device=DEV).view(5, 9, 1)
    slots = torch.tensor([[8, 0, 4]], dtype=torch.int32, device=DEV)
    parent = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV)
    ops.beam_reorder(rows, slots, parent)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.beam_reorder(rows, slots, parent)
    names = list(range(9))
    for p in ([1, 2, 0], [0, 0, 1], [2, 2, 2]):
        parent.copy_(torch.tensor([p], dtype=torch.int32))
        graph.replay()
        taken = [names[[8, 0, 4][x]] for x in p]
        names[8], names[0], names[4] = taken
        for at in (0, 12_345_678, 29_999_999):
            assert rows[:, :, at].cpu().tolist() == [[9 * l + n for n in names] for l in range(5)]


def test_the_status_of_calls_without_a_word():
    """It is kept until it is read, also where the device's first such call was a captured one."""
    from distengine_b200.kernels import ops
    ops.take_status()
    words, kept = ops._status_words, dict(ops._status_words)
    rows = torch.randn(2, 12, 100, device=DEV)
    slots = torch.tensor([[3, 12, 5]], dtype=torch.int32, device=DEV)
    parent = torch.tensor([[1, 0, 0]], dtype=torch.int32, device=DEV)
    stays = torch.arange(3, dtype=torch.int32, device=DEV)[None]
    try:
        words.clear()
        assert ops.take_status() == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.beam_reorder(rows, slots, stays)
        graph.replay()
        assert ops.take_status() == 0
        ops.beam_reorder(rows, slots, parent)
        graph.replay()
        assert ops.take_status(DEV) == 5 and ops.take_status("cuda") == 0
        with torch.cuda.graph(graph := torch.cuda.CUDAGraph()):
            ops.beam_reorder(rows, slots, parent)
        assert ops.take_status() == 0
        graph.replay()
        assert ops.take_status(torch.device(DEV)) == 5 and ops.take_status(0) == 0
    finally:
        words.clear()
        words.update(kept)
    with pytest.raises(ValueError, match="status"):
        ops.take_status("cpu")
