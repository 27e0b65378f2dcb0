"""The host's half of beam search, on the CPU: requests that share pages, contents that change hands, the
choice of beams and hypotheses, and the whole search over a toy model against one that keeps every
sequence by itself."""

import math

import numpy as np
import pytest
import torch

from distengine_b200.cache import CacheManager, OutOfPages, OutOfSlots, PagePool
from distengine_b200.engine import beam as beam_module
from distengine_b200.engine.beam import BeamSearch, Hypothesis, _Search, choose, is_done
from distengine_b200.parts.base import PagedKVSpec, StateSpec


def _cache(pages=40, slots=8, page=4, specs=None):
    specs = specs or [PagedKVSpec(2, 4), PagedKVSpec(2, 4, window=6), StateSpec((3,)),
                      (PagedKVSpec(1, 8, values_in_keys=True), StateSpec((2, 2)))]
    return CacheManager(specs, [None] * len(specs), page, pages, slots, 64, torch.float32, "cpu",
                        poison_freed_pages=True)


def _write(cache, name, new_len, stamp):
    """Feed a request up to new_len: every position holds the stamp and the position."""
    old = cache.length(name)
    cache.reserve([(name, new_len)])
    slot = cache.slot(name)
    for group in cache.paged:
        for pos in range(old, new_len):
            page = group.tables[name][pos // cache.page_size]
            group.k[:, page, :, pos % cache.page_size] = 1000 * stamp + pos
            group.v[:, page, :, pos % cache.page_size] = 1000 * stamp + pos
    for sgroup in cache.states:
        sgroup.state[:, slot] = 1000 * stamp + new_len
    cache.commit(name, new_len)


def _content(cache, name):
    """What a request holds: the readable positions of each paged group, and its states."""
    out, n = [], cache.length(name)
    for group in cache.paged:
        first = 0 if group.spec.window is None else max(0, n - group.spec.window + 1)
        out.append([float(group.k[0, group.tables[name][p // cache.page_size], 0, p % cache.page_size, 0])
                    for p in range(first, n)])
    return out + [sgroup.state[:, cache.slot(name)].flatten().tolist() for sgroup in cache.states]


def test_a_shared_page_is_free_when_all_gave_it_back():
    pool = PagePool(3)
    a, b = pool.take(2)
    pool.share([a])
    assert pool.holders(a) == 2 and pool.num_shared == 1
    assert pool.give([a, b]) == [b] and pool.num_free == 2 and pool.num_shared == 0
    assert pool.give([a]) == [a] and pool.num_free == 3
    for call in (pool.give, pool.share):
        with pytest.raises(KeyError):
            call([a])


@pytest.mark.parametrize("length", [1, 3, 4, 5, 8, 17])
def test_a_copy_holds_the_same_and_goes_its_own_way(length):
    cache = _cache()
    cache.admit("a")
    _write(cache, "a", length, 1)
    before, free = _content(cache, "a"), cache.num_free_pages()
    cache.fork("a", ["b", "c"])
    cache.check_invariants()
    assert cache.num_free_pages() == free - (2 if length % 4 else 0)
    assert _content(cache, "b") == before == _content(cache, "c") == _content(cache, "a")
    for stamp, name in enumerate("abc", 2):
        _write(cache, name, length + 9, stamp)
    assert _content(cache, "a") != _content(cache, "b") != _content(cache, "c")
    for name in "abc":
        assert _content(cache, name)[0][:length] == before[0]
    cache.check_invariants()
    for name in "bac":
        cache.release(name)
        cache.check_invariants()
    assert cache.num_free_pages() == 40


def test_forks_that_are_refused_change_nothing():
    cache = _cache(pages=5, slots=4)
    cache.admit("a")
    _write(cache, "a", 9, 1)
    for copies, error in ((["b", "c", "d", "e"], OutOfSlots), (["b", "c", "d"], OutOfPages),
                          (["b", "b"], ValueError), (["a"], ValueError), ([""], ValueError)):
        with pytest.raises(error):
            cache.fork("a", copies)
        cache.check_invariants()
        assert sorted(cache.live) == ["a"]
    with pytest.raises(KeyError):
        cache.fork("x", ["b"])
    cache.reserve([("a", 10)])
    cache.commit("a", 10, tentative=True)
    with pytest.raises(ValueError, match="tentative"):
        cache.fork("a", ["b"])


@pytest.mark.parametrize("seed", range(6))
def test_contents_change_hands(seed):
    """Random growth and reordering of two groups beside plain lists of what each request holds."""
    rng = np.random.default_rng(seed)
    cache = _cache(pages=60)
    names = [[f"{g}{b}" for b in range(3)] for g in range(2)]
    for g, group in enumerate(names):
        cache.admit(group[0])
        _write(cache, group[0], int(rng.integers(1, 11)), g + 1)
        cache.fork(group[0], group[1:])
    stamp = 10
    for _ in range(25):
        for group in names:
            for name in group:
                stamp += 1
                _write(cache, name, cache.length(name) + 1, stamp)
        parents = [[int(p) for p in rng.integers(0, 3, 3)] for _ in names]
        held = {name: _content(cache, name) for group in names for name in group}
        cache.reorder(names, parents)
        cache.check_invariants()
        for group, source in zip(names, parents):
            for name, parent in zip(group, source):
                assert _content(cache, name) == held[group[parent]]
        if cache.length("00") > 40:
            break
    for group in names:
        for name in group:
            cache.release(name)
    cache.check_invariants()
    assert cache.num_free_pages() == 60


def test_reorderings_that_are_refused():
    cache = _cache()
    for name, n in (("a", 5), ("b", 5), ("c", 6), ("d", 5)):
        cache.admit(name)
        _write(cache, name, n, 1)
    for groups, parents in (([["a", "c"]], [[0, 0]]), ([["a", "b"]], [[0, 2]]), ([["a", "b"]], [[0]]),
                            ([["a", "b"], ["b", "d"]], [[0, 0], [0, 0]]), ([["a", "b"], ["d"]], [[0, 0], [0]]),
                            ([["a", "b"]], [[0, -1]]), ([["a", "b"]], [[0, 0], [0, 0]])):
        with pytest.raises(ValueError):
            cache.reorder(groups, parents)
    with pytest.raises(KeyError):
        cache.reorder([["a", "x"]], [[0, 0]])
    cache.check_invariants()


def test_shared_prefixes():
    cache = _cache(slots=8)
    for i, name in enumerate("abcd"):
        cache.admit(name)
        _write(cache, name, 9 + i, i)
    assert cache.shared_prefixes(list("abcd")) is None
    cache.fork("a", ["a1", "a2"])
    cache.fork("c", ["c1"])
    assert cache.shared_prefixes(["a", "a1", "a2", "b", "c", "c1", "d"]) == ([3, 1, 2, 1], [8, 0, 8, 0])
    assert cache.shared_prefixes(["a", "b", "a1"]) is None
    assert cache.shared_prefixes(["b"]) is None
    for stamp, name in enumerate(("a", "a1", "a2"), 20):
        _write(cache, name, 16, stamp)
    cache.reorder([["a", "a1", "a2"]], [[0, 0, 2]])
    assert cache.shared_prefixes(["a", "a1"]) == ([2], [16])
    assert cache.shared_prefixes(["a", "a1", "a2"]) == ([3], [8])


# ------------------------------------------------------------------------------- the choice
def test_the_choice_of_beams():
    search = _Search([1], ["x", "y", "z"], [[5], [6], [7]], [-1.0, -2.0, -3.0])
    parents, tokens = choose(search, [(-1.5, 1, 9), (-1.6, 0, 2), (-1.7, 1, 2), (-1.8, 0, 8),
                                      (-1.9, 2, 2), (-2.0, 1, 4)], 3, 2, 1.0)
    # both ends are among the first three; beam 1 keeps its place, beam 0 its own, place 2 takes from 1
    assert (parents, tokens) == ([0, 1, 1], [8, 9, 4])
    assert search.tokens == [[5, 8], [6, 9], [6, 4]] and search.scores == [-1.8, -1.5, -2.0]
    assert [(h.token_ids, round(h.score, 6)) for h in search.finished] == [([5, 2], -0.8), ([6, 2], -0.85)]
    parents, tokens = choose(search, [(-4.0, 2, 3)], 3, 2, 1.0)
    assert parents == [0, 1, 2] and search.scores == [-math.inf, -math.inf, -4.0]


def test_when_a_search_is_done():
    search = _Search([1], ["x", "y"], [[5], [6]], [-1.0, -2.0])
    assert not is_done(search, 2, 1.0)
    search.finished = [Hypothesis([2], -0.5), Hypothesis([3], -1.2)]
    assert not is_done(search, 2, 1.0)
    search.finished.append(Hypothesis([3], -1.0))
    assert is_done(search, 2, 1.0)
    search.scores = [-math.inf, -math.inf]
    search.finished = []
    assert is_done(search, 2, 1.0)


class _ToyRunner:
    """Steps over a cache that holds each position's token, read back through the block tables, and a
    running state: logits are a fixed random function of the sequence that the cache really holds."""

    device = torch.device("cpu")

    def __init__(self, cache, vocabulary, seed):
        self.cache, self.vocabulary, self.seed, self.most = cache, vocabulary, seed, 0

    def step(self, entries):
        rows = []
        self.cache.reserve([(e.request_id, self.cache.length(e.request_id) + len(e.tokens))
                            if self.cache.has(e.request_id) else
                            (self.cache.admit(e.request_id) and e.request_id or e.request_id, len(e.tokens))
                            for e in entries])
        self.most = max(self.most, len(entries))
        for e in entries:
            old = self.cache.length(e.request_id)
            for i, token in enumerate(e.tokens):
                pos = old + i
                for group in self.cache.paged:
                    page = group.tables[e.request_id][pos // self.cache.page_size]
                    assert group.pool.holders(page) == 1, "a shared page is written"
                    group.k[:, page, :, pos % self.cache.page_size] = float(token)
                for sgroup in self.cache.states:
                    sgroup.state[:, self.cache.slot(e.request_id)] += (pos + 1) * token
            self.cache.commit(e.request_id, old + len(e.tokens))
            self.cache.check_invariants()
            ids = self.sequence(e.request_id)
            rows += [toy_logits(ids[: old + w + 1], self.vocabulary, self.seed) for w in e.want]
        return torch.stack(rows) if rows else torch.zeros(0, self.vocabulary)

    def sequence(self, name):
        group = self.cache.paged[0]
        ids = [int(group.k[0, group.tables[name][p // self.cache.page_size], 0, p % self.cache.page_size, 0])
               for p in range(self.cache.length(name))]
        for sgroup in self.cache.states:
            want = sum((p + 1) * t for p, t in enumerate(ids))
            assert float(sgroup.state[0, self.cache.slot(name)].flatten()[0]) == want
        return ids

    def check_status(self):
        pass


def toy_logits(ids, vocabulary, seed):
    g = torch.Generator().manual_seed(seed + sum((i + 1) * (t + 3) * 7919 for i, t in enumerate(ids)) % 10 ** 9)
    return torch.randn(vocabulary, generator=g) * 2


class _PlainSelector:
    def __init__(self, device, groups, take):
        pass

    def select(self, logits, scores, take):
        beams, out = len(scores[0]), []
        for g, row in enumerate(scores):
            total = torch.log_softmax(logits[g * beams: (g + 1) * beams].double(), 1) + torch.tensor(
                row, dtype=torch.float64)[:, None]
            order = total.flatten().sort(descending=True, stable=True).indices[:take].tolist()
            v = logits.shape[1]
            out.append([(float(total.flatten()[i]), i // v, i % v) for i in order
                        if float(total.flatten()[i]) > -math.inf])
        return out


def plain_search(logits_of, prompt, beams, most, eos, penalty):
    """Every sequence by itself; the rules of ``engine.beam`` in their plainest form."""
    running, done = [(0.0, [])], []
    for step in range(most):
        cands = []
        for score, tokens in running:
            logp = torch.log_softmax(logits_of(prompt + tokens).double(), 0)
            cands += [(score + float(logp[t]), tokens + [t]) for t in range(len(logp))]
        cands.sort(key=lambda c: -c[0])
        cands = cands[: 2 * beams]
        done += [(s / len(t) ** penalty, t) for s, t in cands[:beams] if t[-1] == eos]
        running = [(s, t) for s, t in cands if t[-1] != eos][:beams]
        if step + 1 == most or not running or (
                len(done) >= beams and sorted(d[0] for d in done)[-beams]
                >= running[0][0] / (step + 1) ** penalty):
            break
    done += [(s / len(t) ** penalty, t) for s, t in running]
    return sorted(done, key=lambda d: -d[0])[:beams]


@pytest.mark.parametrize("beams,most,eos,penalty", [(1, 6, 3, 1.0), (2, 9, 3, 1.0), (3, 12, -1, 0.0),
                                                    (4, 10, 3, 0.6), (4, 1, 3, 1.0), (3, 14, 0, 2.0)])
@pytest.mark.parametrize("lengths", [[1], [4, 9, 3], [7, 8, 5, 6, 2]])
def test_a_whole_search(beams, most, eos, penalty, lengths, monkeypatch):
    monkeypatch.setattr(beam_module, "BeamSelector", _PlainSelector)
    rng = np.random.default_rng(beams)
    prompts = [[int(t) for t in rng.integers(0, 11, n)] for n in lengths]
    cache = _cache(pages=50, slots=9, specs=[PagedKVSpec(1, 1), StateSpec((2,))])
    cache.poison = False
    runner = _ToyRunner(cache, 11, 17)
    search = BeamSearch(runner, cache, beams, 4, penalty)
    got = search.run(prompts, most, eos, "t")
    assert cache.num_free_pages() == 50 and not cache.live
    assert runner.most <= 9
    for prompt, found in zip(prompts, got):
        want = plain_search(lambda ids: toy_logits(ids, 11, 17), prompt, beams, most, eos, penalty)
        assert [h.token_ids for h in found] == [t for _, t in want]
        assert np.allclose([h.score for h in found], [s for s, _ in want], rtol=0, atol=1e-9)


def test_searches_that_are_refused():
    cache = _cache(pages=6, slots=4)
    runner = _ToyRunner(cache, 11, 1)
    for beams in (0, 33, 5, 2.0, True and -1):
        with pytest.raises(ValueError):
            BeamSearch(runner, cache, beams, 8)
    with pytest.raises(ValueError, match="length_penalty"):
        BeamSearch(runner, cache, 2, 8, float("nan"))


def test_a_prompt_that_cannot_fit_is_refused(monkeypatch):
    monkeypatch.setattr(beam_module, "BeamSelector", _PlainSelector)
    cache = _cache(pages=6, slots=4)
    search = BeamSearch(_ToyRunner(cache, 11, 1), cache, 4, 8)
    with pytest.raises(ValueError, match="pages"):
        search.run([[1] * 9], 8, -1, "t")
    assert not cache.live


@pytest.mark.parametrize("beams,budget,groups", [(3, 8, 2), (3, 5, 1), (2, 2, 1), (1, 4, 4)])
def test_a_step_keeps_to_the_token_budget(beams, budget, groups, monkeypatch):
    monkeypatch.setattr(beam_module, "BeamSelector", _PlainSelector)
    steps = []

    class Runner(_ToyRunner):
        def step(self, entries):
            steps.append(sum(len(e.tokens) for e in entries))
            return super().step(entries)

    cache = _cache(pages=60, slots=9, specs=[PagedKVSpec(1, 1), StateSpec((2,))])
    cache.poison = False
    prompts = [[1, 2, 3, 4, 5, 6, 7, 8, 9], [4, 4], [9, 1, 2, 0], [5]]
    search = BeamSearch(Runner(cache, 11, 17), cache, beams, budget)
    assert search.groups == groups
    found = search.run(prompts, 6, -1, "t")
    assert max(steps) <= budget and beams * groups in steps
    for prompt, got in zip(prompts, found):
        want = plain_search(lambda ids: toy_logits(ids, 11, 17), prompt, beams, 6, -1, 1.0)
        assert [h.token_ids for h in got] == [t for _, t in want]


def test_more_beams_than_a_step_has_tokens_are_refused():
    cache = _cache(pages=6, slots=8)
    with pytest.raises(ValueError, match="max_batch_tokens"):
        BeamSearch(_ToyRunner(cache, 11, 1), cache, 5, 4)


@pytest.mark.parametrize("penalty", [math.inf, -math.inf, 1e5, -1e5, 1e308, 10 ** 400])
def test_length_penalties_beyond_the_number_range_are_refused(penalty, monkeypatch):
    """A score is divided by the length to that power, which has to be a number above 0."""
    monkeypatch.setattr(beam_module, "BeamSelector", _PlainSelector)
    cache = _cache(pages=50, slots=4, specs=[PagedKVSpec(1, 1), StateSpec((2,))])
    cache.poison = False
    with pytest.raises(ValueError, match="length_penalty"):
        BeamSearch(_ToyRunner(cache, 11, 1), cache, 2, 8, penalty).run([[1, 2]], 5, 3, "t")
    assert not cache.live
    found = BeamSearch(_ToyRunner(cache, 11, 1), cache, 2, 8, -3).run([[1, 2]], 5, 3, "t")
    assert len(found[0]) == 2
