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


@pytest.mark.parametrize("offset, temperature", [(0.0, 1.0), (150.0, 0.75), (-300.0, 1.3)])
def test_replacements_where_the_drafts_probabilities_are_near_the_targets(offset, temperature):
    """w = p - q cancels: a draw may go to another token than in exact arithmetic only within the error of 32-bit probabilities.

    logit / T has an error of |logit / T| 2^-23 (two roundings), so has the largest one, and the exponential one of 2^-22 of its
    argument's size; sums, quotients and logarithms a few 2^-23, 2^-20 in all.  p's error reaches w as it is, w's weight by p / w."""
    from q8_helpers import mix32, mix32_all, uniform
    rng = np.random.default_rng(10)
    n, vocab = 200, 4000
    logits = (rng.standard_normal((2 * n, vocab)) * 2 + offset).astype(np.float32)
    x = logits.astype(np.float64) / temperature
    top = x.max(axis=-1, keepdims=True)
    p = np.exp(x - top)
    p /= p.sum(axis=-1, keepdims=True)
    q = (p * (1 + 2.0 ** -9 * rng.standard_normal(p.shape))).astype(np.float32)
    drafts = np.array([rng.choice(vocab, p=r / r.sum()) for r in p])
    drafted = np.arange(2 * n), drafts
    q[drafted] = np.minimum(4 * p[drafted], 0.9)
    starts, seeds = np.arange(0, 2 * n + 1, 2), np.arange(n)
    to = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to(t).cuda()  # noqa: E731
    tokens, counts = (t.cpu().numpy() for t in ops.verify_drafts(
        to(logits, torch.float32), to(drafts, torch.int32), to(starts, torch.int32), to(q, torch.float32),
        torch.full((n,), temperature, device="cuda"), to(seeds, torch.int32), torch.full((n,), 9, dtype=torch.int32, device="cuda")))
    ops.take_device_errors()
    t32 = float(np.float32(temperature))
    error = (np.abs(x).max() * 2 * 2.0 ** -23 + (top - x) * 2.0 ** -22 + 2.0 ** -20) * p + abs(t32 - temperature) / t32 * (top - x) * p
    refused = 0
    for b in range(n):
        row = 2 * b
        key = mix32(mix32(b ^ 0x9E3779B9) ^ 9)
        u, x0 = uniform(mix32(key ^ 0xFFFFFFFF)), drafts[row]
        if abs(u * q[row, x0] - p[row, x0]) < 1e-3 * p[row, x0]:
            continue
        assert (counts[b] == 2) == (u * q[row, x0] < p[row, x0])
        if counts[b] == 2:
            continue
        refused += 1
        wait = -np.log(uniform(mix32_all(key + np.arange(vocab, dtype=np.uint64) * np.uint64(0x85EBCA6B))))
        w = np.maximum(p[row] - q[row].astype(np.float64), 0.0)
        low, high = (w - error[row]) / wait, (w + error[row]) / wait
        assert high[tokens[row]] * (1 + 2.0 ** -20) >= low.max()
    assert refused > n // 2
