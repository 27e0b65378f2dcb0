"""Beam search through the entry points against a search over the plain implementations, which keeps every
sequence by itself: the Llama decoder with its beams' prefixes shared and not, and the architectures
whose beams also carry recurrent states, windows, latents and routed experts."""

import os
import subprocess
import sys

import pytest
import torch

import plain_llama
import tiny_configs
from test_beam_search import plain_search

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# Scores are sums of log probabilities of float32 logits that differ by up to 2e-5 of their size (the
# tests' bound for two orders of float32 sums): 12 tokens, twice that a token (its logit and the
# normaliser), logits of up to 5.
SCORE_TOL = 12 * 2 * 2e-5 * 5


def _engine(folder, dtype, **options):
    from distengine_b200 import Engine, EngineConfig
    return Engine(folder, EngineConfig(dtype=dtype, **options))


def _score(logits_of, prompt, tokens, penalty):
    total = 0.0
    for i, token in enumerate(tokens):
        total += float(torch.log_softmax(logits_of(prompt + tokens[:i]).double(), 0)[token])
    return total / len(tokens) ** penalty


def _check(found, logits_of, prompt, beams, most, eos, penalty, tol=SCORE_TOL):
    """The same hypotheses in the same order but where two are nearly equal; each with its own score."""
    want = plain_search(logits_of, prompt, beams, most, eos, penalty)
    assert len(found) == len(want)
    for h, (score, tokens) in zip(found, want):
        assert abs(h.score - _score(logits_of, prompt, h.token_ids, penalty)) <= tol
        assert abs(h.score - score) <= tol, (h, score, tokens)
        if h.token_ids != tokens:
            assert sum(abs(s - score) <= 2 * tol for s, _ in want) > 1, (h, score, tokens)


def _llama(name, model_root, dtype=torch.float32):
    folder = tiny_configs.make_folder(name, model_root)
    config, weights = plain_llama.load_model_folder(folder)
    memo = {}

    def logits_of(ids):
        key = tuple(ids)
        if key not in memo:
            memo[key] = plain_llama.plain_forward(config, weights, ids, dtype, rows=[len(ids) - 1])[-1]
        return memo[key]

    return folder, logits_of


@pytest.mark.parametrize("name", ["tiny_a", "tiny_c", "tiny_d", "tiny_e"])
@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("beams,eos,penalty", [(4, -1, 1.0), (2, 7, 0.5)])
def test_llama(name, share, beams, eos, penalty, model_root, monkeypatch):
    from distengine_b200.kernels import attention, shared_prefix
    calls = []
    plain_run = shared_prefix.SharedPrefixAttention.run
    monkeypatch.setattr(attention, "SHARED_SAVES", 0 if share else 1 << 60)
    monkeypatch.setattr(shared_prefix.SharedPrefixAttention, "run",
                        lambda self, *a, **k: (calls.append(1), plain_run(self, *a, **k)))
    folder, logits_of = _llama(name, model_root)
    spec = tiny_configs.ALL[name]
    engine = _engine(folder, "float32", block_size=spec["page_size"], num_blocks=64,
                     decode_batch_size=9)
    prompts = [tiny_configs.prompt_tokens(name, n, n) for n in (45, 70, 3)]
    for found, prompt in zip(engine.beam_search(prompts, 9, beams, eos, penalty), prompts):
        _check(found, logits_of, prompt, beams, 9, eos, penalty)
    assert bool(calls) == share
    engine.cache.check_invariants()
    assert engine.cache.num_free_pages() == 64 and not engine.cache.live


@pytest.mark.parametrize("name", ["tiny_d", "tiny_e"])
def test_llama_in_bfloat16(name, model_root, monkeypatch):
    """Shared or not, the scores are those of the tokens: off by the bfloat16 logits' bound a token."""
    from distengine_b200.kernels import attention
    folder, logits_of = _llama(name, model_root, torch.bfloat16)
    prompt = tiny_configs.prompt_tokens(name, 70, 3)
    for saves in (0, 1 << 60):
        monkeypatch.setattr(attention, "SHARED_SAVES", saves)
        engine = _engine(folder, "bfloat16", block_size=16, num_blocks=64, decode_batch_size=16)
        found = engine.beam_search([prompt], 8, 5)[0]
        scale = logits_of(prompt).abs().max().item()
        assert len(found) == 5
        for h in found:
            assert len(h.token_ids) == 8
            # (a mean over the tokens: no further off than one of them, its logit and the normaliser)
            assert abs(h.score - _score(logits_of, prompt, h.token_ids, 1.0)) <= 2 * 4e-2 * scale


@pytest.mark.parametrize("name", ["tiny_d", "tiny_e"])
@pytest.mark.parametrize("beams", [5, 12])
@pytest.mark.parametrize("share", [True, False])
def test_bfloat16_step_by_step(name, beams, share, model_root, monkeypatch):
    """Every row of logits of a search is that of the sequence that its beam stands for, and the search over
    these rows is the plain one: so the beams' contents, the keys that they share and the choice are all as
    they should be.  (12 beams of three query heads a kv head: more than 32 rows behind the shared keys.)"""
    from distengine_b200.kernels import attention
    from gpu_helpers import BF16_MAX_REL
    monkeypatch.setattr(attention, "SHARED_SAVES", 0 if share else 1 << 60)
    folder, logits_of = _llama(name, model_root, torch.bfloat16)
    prompt = tiny_configs.prompt_tokens(name, 70, 3)
    engine = _engine(folder, "bfloat16", block_size=16, num_blocks=64, decode_batch_size=16)
    held, rows, shared_steps = {}, {}, []
    step, fork, reorder = engine.runner.step, engine.cache.fork, engine.cache.reorder

    def follow_step(entries):
        logits = step(entries)
        at = 0
        for e in entries:
            held[e.request_id] = held.get(e.request_id, []) + e.tokens
            for _ in e.want:
                rows.setdefault(tuple(held[e.request_id]), logits[at].float().cpu())
                at += 1
        shared_steps.append(any("/shared/" in key for key in engine.runner.last_arrays))
        return logits

    def follow_fork(request_id, copies):
        held.update({name: list(held[request_id]) for name in copies})
        return fork(request_id, copies)

    def follow_reorder(groups, parents):
        for names, source in zip(groups, parents):
            held.update(dict(zip(names, [held[names[p]] for p in source])))
        return reorder(groups, parents)

    monkeypatch.setattr(engine.runner, "step", follow_step)
    monkeypatch.setattr(engine.cache, "fork", follow_fork)
    monkeypatch.setattr(engine.cache, "reorder", follow_reorder)
    found = engine.beam_search([prompt], 8, beams)[0]
    assert shared_steps == [False] + [share] * 7
    # the contents: within the bfloat16 bound of their own sequence's logits, beyond it of the others'
    # (nearly any: rows of two sequences that end alike may be as near)
    plain = {ids: logits_of(list(ids)) for ids in rows}
    apart = []
    for ids, row in rows.items():
        for other, want in plain.items():
            off = (row - want).abs().max().item() / want.abs().max().item()
            if other == ids:
                assert off <= BF16_MAX_REL, (len(ids), off)
            elif len(other) == len(ids):
                apart.append(off > BF16_MAX_REL)
    assert sum(apart) >= 0.9 * len(apart) > 0
    # the choice: scores go on from step to step as float32 (half a step of 2^-24), each total off by up to
    # 2e-6 (the fast sums) before it is rounded
    want = plain_search(lambda ids: rows[tuple(ids)], prompt, beams, 8, -1, 1.0)
    assert [h.token_ids for h in found] == [tokens for _, tokens in want]
    for h, (score, tokens) in zip(found, want):
        assert abs(h.score - score) <= 8 * (2e-6 + 2.0 ** -24 * abs(score * len(tokens)))


def _architecture(name, root):
    """(folder, last logits of a sequence, a prompt) of a small model of each architecture."""
    import importlib
    module = {"vomo_a": "vomotar", "sebi_a": "sebilorn", "vap_d": "vapelix", "biz_b": "bizetar",
              "pur_b": "puripel", "sif_b": "sifasun"}[name]
    plain = importlib.import_module(f"plain_{module}")
    configs = importlib.import_module(f"{module}_configs")
    folder, weights = configs.make_folder(name, root)
    config = configs.ALL[name]
    if module in ("vomotar", "sebilorn", "sifasun"):
        return folder, lambda ids: plain.forward(config, weights, ids)[-1], configs
    return folder, lambda ids: plain.forward(ids, weights, config)[-1], configs


@pytest.mark.parametrize("name", ["vomo_a", "sebi_a", "vap_d", "biz_b", "pur_b", "sif_b"])
def test_other_architectures(name, model_root):
    folder, logits_of, configs = _architecture(name, model_root)
    engine = _engine(folder, "float32", block_size=16, num_blocks=32, decode_batch_size=6,
                     max_model_len=96)
    prompts = [configs.tokens(name, n) for n in (37, 16)]
    memo = {}

    def last(ids):
        if tuple(ids) not in memo:
            memo[tuple(ids)] = logits_of(ids)
        return memo[tuple(ids)]

    for found, prompt in zip(engine.beam_search(prompts, 6, 3), prompts):
        _check(found, last, prompt, 3, 6, -1, 1.0)
    engine.cache.check_invariants()


def test_one_beam_is_greedy(model_root):
    folder, _ = _llama("tiny_a", model_root)
    engine = _engine(folder, "float32", block_size=16, num_blocks=32, decode_batch_size=4)
    prompt = tiny_configs.prompt_tokens("tiny_a", 20, 1)
    assert engine.beam_search([prompt], 8, 1)[0][0].token_ids == engine.generate([prompt], 8)[0]


def test_graphs_change_nothing(model_root, monkeypatch):
    from distengine_b200.kernels import attention
    monkeypatch.setattr(attention, "SHARED_SAVES", 0)
    folder, _ = _llama("tiny_d", model_root)
    prompt = tiny_configs.prompt_tokens("tiny_d", 70, 2)
    found = []
    for graphs in (True, False):
        engine = _engine(folder, "bfloat16", block_size=16, num_blocks=64, decode_batch_size=8,
                         use_graphs=graphs)
        found.append(engine.beam_search([prompt], 24, 4)[0])
        assert (engine.runner.graph_replays > 0) == graphs
    assert [h.token_ids for h in found[0]] == [h.token_ids for h in found[1]]
    assert [h.score for h in found[0]] == [h.score for h in found[1]]


def test_a_move_that_could_not_be_made_raises(model_root):
    """What the cache's own moves on the device report goes to the word that the engine looks at."""
    from distengine_b200.engine.step import KernelStatusError, StepEntry
    folder, _ = _llama("tiny_a", model_root)
    engine = _engine(folder, "float32", block_size=16, num_blocks=16, decode_batch_size=4)
    prompt = tiny_configs.prompt_tokens("tiny_a", 10, 1)
    engine.runner.step([StepEntry("a", prompt, [9])])
    engine.cache.fork("a", ["b"])
    engine.runner.check_status()
    engine.cache._move([["a", "a"]], [[1, 0]])            # (no caller can ask for this)
    with pytest.raises(KernelStatusError, match="status 5"):
        engine.runner.check_status()
    engine.runner.check_status()
    engine.cache.release("a"), engine.cache.release("b")
    assert len(engine.beam_search([prompt], 3, 2)[0]) == 2


def test_entry_points_and_refusals(model_root):
    from distengine_b200 import generate_beam
    folder, _ = _llama("tiny_a", model_root)
    engine = _engine(folder, "float32", block_size=16, num_blocks=8, decode_batch_size=4)
    prompt = tiny_configs.prompt_tokens("tiny_a", 10, 1)
    best = engine.beam_search([prompt], 5, 3)[0][0]
    out = generate_beam(engine, torch.tensor([prompt]), 5, -1, 3)
    assert out.tolist() == [prompt + best.token_ids]
    for call in (lambda: engine.beam_search([prompt], 5, 5), lambda: engine.beam_search([prompt], 0, 2),
                 lambda: engine.beam_search([[]], 5, 2), lambda: engine.beam_search([[256]], 5, 2),
                 lambda: engine.beam_search([prompt], 200, 2), lambda: engine.beam_search([prompt], 60, 4),
                 lambda: engine.beam_search([prompt], 5, 2, length_penalty=float("nan"))):
        with pytest.raises(ValueError):
            call()
    engine.submit("r", prompt, 4, -1)
    with pytest.raises(RuntimeError, match="pending"):
        engine.beam_search([prompt], 5, 2)
    while engine.has_pending():
        engine.step()
    assert engine.beam_search([prompt], 5, 3)[0][0].token_ids == best.token_ids


def test_the_command_line(model_root):
    folder, _ = _llama("tiny_a", model_root)
    prompt = tiny_configs.prompt_tokens("tiny_a", 10, 1)
    engine = _engine(folder, "float32", block_size=16, num_blocks=16, decode_batch_size=4)
    best = engine.beam_search([prompt], 5, 3)[0][0]
    done = subprocess.run(
        [sys.executable, "-m", "distengine_b200", "generate", "--model", folder, "--prompt-ids",
         " ".join(map(str, prompt)), "--max-new-tokens", "5", "--beams", "3", "--dtype", "float32",
         "--num-blocks", "16", "--decode-batch-size", "4"], cwd=ROOT, capture_output=True, text=True,
        timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    assert f"Generated token IDs: {best.token_ids}" in done.stdout and "Score:" in done.stdout
