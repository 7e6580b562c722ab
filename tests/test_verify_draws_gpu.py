"""What replaces a refused draft does not depend on how the draft was drawn: drafts of the framework's own sampler."""
import numpy as np
import pytest
import torch

from helpers import TINY, make_model_folder, random_tokens
from llm_inference_lab_b200.engine.engine import Engine, Entry
from llm_inference_lab_b200.kernels import ops

pytestmark = pytest.mark.gpu

P, Q = np.array([0.2, 0.5, 0.3, 0.0]), np.array([0.75, 0.05, 0.15, 0.05])


def frequencies(p, q, seeds_of_drafts, certain=False, **how):
    """Frequencies of the first token and of acceptance over 4 x 30,000 requests of one draft, drawn by `sample`."""
    n, total, taken = 30000, np.zeros(len(p)), 0
    log = lambda x, rows: torch.from_numpy(np.where(x > 0, np.log(np.maximum(x, 1e-30)), -np.inf).astype(np.float32)).cuda().repeat(rows, 1)  # noqa: E731
    ones, positions = torch.ones(n, device="cuda"), torch.full((n,), 77, dtype=torch.int32, device="cuda")
    starts = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda")
    probs = None if certain else torch.from_numpy(q.astype(np.float32)).cuda().repeat(2 * n, 1)
    for turn in range(4):
        seeds = torch.arange(n, dtype=torch.int32, device="cuda") + turn * n
        drafts = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
        drafts[::2] = ops.sample(log(q, n), ones, seeds_of_drafts(seeds), positions).int()
        tokens, counts = ops.verify_drafts(log(p, 2 * n), drafts, starts, probs, ones, seeds, positions, **how)
        total += np.bincount(tokens[::2].cpu().numpy(), minlength=len(p))
        taken += int((counts == 2).sum())
    ops.take_device_errors()
    return total / (4 * n), taken / (4 * n), 4 * n


def within(seen, p, n):
    # five standard deviations of a frequency of n draws
    return (np.abs(seen - p) <= 5 * np.sqrt(p * (1 - p) / n)).all()


def test_drafts_of_the_sampler_with_the_same_seeds():
    seen, taken, n = frequencies(P, Q, lambda seeds: seeds, fresh=True)
    assert within(seen, P, n), seen
    assert abs(taken - np.minimum(P, Q).sum()) <= 5 * 0.5 / n ** 0.5


@pytest.mark.parametrize("fresh", [False, True])
def test_drafts_of_the_sampler_with_other_seeds(fresh):
    seen, taken, n = frequencies(P, Q, lambda seeds: seeds ^ 0x5BD1E995, fresh=fresh)
    assert within(seen, P, n), seen
    assert abs(taken - np.minimum(P, Q).sum()) <= 5 * 0.5 / n ** 0.5


def test_sampled_drafts_given_as_certain():
    """Judged as if nothing else could have been drafted: accepted with p of them, and replaced by the rest of p all the same."""
    seen, taken, n = frequencies(P, Q, lambda seeds: seeds, certain=True, fresh=True)
    assert within(seen, P, n), seen
    assert abs(taken - (P * Q).sum()) <= 5 * 0.5 / n ** 0.5


def test_only_what_replaces_a_refused_draft_is_drawn_anew():
    """Acceptance, and the draw behind the last draft (that of a request without drafts too), are as they were."""
    rng = np.random.default_rng(5)
    rows, vocab = 400, 3000
    logits = torch.from_numpy((rng.standard_normal((rows, vocab)) * 2).astype(np.float32)).cuda()
    probs = torch.softmax(logits + torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32)).cuda() * 0.5, dim=-1)
    drafts = torch.multinomial(probs, 1, generator=torch.Generator("cuda").manual_seed(6))[:, 0].int()
    starts = torch.arange(0, rows + 1, 4, dtype=torch.int32, device="cuda")
    starts[1] = 1                                   # a request without drafts, and one of six
    n = starts.numel() - 1
    t, seeds = torch.full((n,), 0.8, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    old, old_counts = ops.verify_drafts(logits, drafts, starts, probs, t, seeds, seeds)
    new, counts = ops.verify_drafts(logits, drafts, starts, probs, t, seeds, seeds, fresh=True)
    ops.take_device_errors()
    assert torch.equal(counts, old_counts)
    sizes = starts[1:] - starts[:-1]
    ends = (starts[:-1] + counts - 1).long()
    refused = counts < sizes
    assert refused.any() and not refused.all()
    same = torch.ones(rows, dtype=torch.bool, device="cuda")
    same[ends[refused]] = False
    assert torch.equal(old[same], new[same]) and (old[~same] != new[~same]).float().mean() > 0.5
    # greedy requests draw nothing
    for temperature in (None, torch.zeros(n, device="cuda")):
        args = (None, None, None) if temperature is None else (temperature, seeds, seeds)
        assert all(torch.equal(a, b) for a, b in zip(ops.verify_drafts(logits, drafts, starts, probs, *args),
                                                     ops.verify_drafts(logits, drafts, starts, probs, *args, fresh=True)))


def test_an_engines_drafted_step_draws_anew(tmp_path, monkeypatch):
    """`verify_step` over drafts that its own sampler would draw for the seed: the replacements are those of `fresh`."""
    cfg, opt = TINY["A"]
    rng = np.random.default_rng(9)
    n = 16
    folder = make_model_folder(str(tmp_path), cfg, opt["seed"], "bfloat16")
    engine = Engine(folder, "bf16", page_size=opt["page_size"], max_tokens=2048, max_requests=n)
    prompts = [random_tokens(rng, 5, cfg["vocab_size"]) for _ in range(n)]
    engine.step([Entry(r, p[:-1]) for r, p in enumerate(prompts)])
    drafts = [random_tokens(rng, 2, cfg["vocab_size"]) for _ in range(n)]
    seen = {}
    real = ops.verify_drafts

    def keep(logits, *args, **how):
        seen["args"] = (logits.clone(), *args)
        return real(logits, *args, **how)
    monkeypatch.setattr(ops, "verify_drafts", keep)
    told = engine.verify_step([(r, prompts[r][-1], drafts[r]) for r in range(n)], [1.0] * n, list(range(n)))
    results = []
    for fresh in (True, False):
        tokens, counts = (t.tolist() for t in real(*seen["args"], fresh=fresh))
        results.append([tokens[3 * r: 3 * r + counts[r]] for r in range(n)])
    assert told == results[0] != results[1]
