"""Drafted tokens judged and replaced, against the definition in 64 bits: the same tokens, and the target's distribution."""
import numpy as np
import pytest
import torch

from llm_inference_lab_b200.kernels import ops
from q8_helpers import verify

pytestmark = pytest.mark.gpu


def near(rng, logits, temperature, sharp=0.5):
    e = (logits + rng.standard_normal(logits.shape) * sharp) / temperature
    e = np.exp(e - e.max(axis=-1, keepdims=True))
    return (e / e.sum(axis=-1, keepdims=True)).astype(np.float32)


def run(logits, drafts, starts, probs=None, temperature=None, seeds=None, positions=None, stride=0):
    to = lambda x, t: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(t).cuda()  # noqa: E731
    x = to(logits, torch.float32)
    q = to(probs, torch.float32)
    if stride:      # rows further apart, off their boundaries
        wide = [None if t is None else torch.zeros((t.shape[0], t.shape[1] + stride), device="cuda") for t in (x, q)]
        for w, t in zip(wide, (x, q)):
            if t is not None:
                w[:, 1: 1 + t.shape[1]] = t
        x, q = (None if w is None else w[:, 1: 1 + logits.shape[1]] for w in wide)
    seeds = None if seeds is None else np.asarray(seeds, np.int64).astype(np.int32)
    out = ops.verify_drafts(x, to(drafts, torch.int32), to(starts, torch.int32), q, to(temperature, torch.float32),
                            to(seeds, torch.int32), to(positions, torch.int32))
    ops.take_device_errors()
    return [t.cpu().numpy().astype(np.int64) for t in out]


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 8192, 8193, 20001, 151936])
@pytest.mark.parametrize("counts", [[1], [5], [3, 1, 0, 9, 2], [2] * 20])
@pytest.mark.parametrize("how", ["probs", "certain", "greedy", "mixed"])
def test_tokens(vocab, counts, how):
    rng = np.random.default_rng(vocab + len(counts))
    starts = np.concatenate(([0], np.cumsum(counts)))
    rows, B = int(starts[-1]), len(counts)
    logits = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    temperature = {"greedy": None, "mixed": np.where(np.arange(B) % 2, 0.0, 0.9)}.get(how, rng.uniform(0.5, 1.5, B))
    temperature = None if temperature is None else np.asarray(temperature, np.float32)
    probs = near(rng, logits, 0.9) if how in ("probs", "mixed") else None
    drafts = np.array([rng.choice(vocab, p=r.astype(np.float64) / r.astype(np.float64).sum()) for r in (probs if probs is not None else near(rng, logits, 0.4))],
                      np.int64).reshape(rows)
    if how in ("greedy", "mixed"):
        drafts = np.where(rng.random(rows) < 0.7, logits.argmax(axis=-1) if rows else drafts, drafts)
    seeds, positions = rng.integers(0, 2 ** 31, B), rng.integers(1, 5000, B)
    tokens, got_counts = run(logits, drafts, starts, probs, temperature, seeds, positions, stride=5 if vocab == 20001 else 0)
    want, want_counts, gap = verify(logits, drafts, starts, probs, temperature, seeds, positions)
    assert gap > 2.0 ** -19, "the inputs hold a comparison that 32 bits cannot settle"
    assert np.array_equal(tokens, want) and np.array_equal(got_counts, want_counts)


def test_drafts_that_are_no_tokens_are_refused():
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((4, 50)).astype(np.float32)
    for drafts in ([-1, 0, 0, 0], [50, 0, 0, 0], [2 ** 31 - 1, 0, 0, 0]):
        for temperature in (None, np.array([1.0], np.float32)):
            tokens, counts = run(logits, np.array(drafts), [0, 4], None, temperature, [3], [9])
            want, _, _ = verify(logits, drafts, [0, 4], None, temperature, [3], [9])
            assert counts[0] == 1 and np.array_equal(tokens, want) and tokens[1:].tolist() == [-1] * 3


def test_numbers_that_are_none():
    """A NaN never wins and takes no weight; masks of the type's lowest value and of -inf leave the rest; a row of NaN says so."""
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((6, 300)).astype(np.float32)
    logits[0, 5] = np.nan
    logits[1, 10:] = -np.inf
    logits[2, 10:] = np.finfo(np.float32).min
    logits[3, :] = np.nan
    logits[4, :] = -np.inf
    logits[4, 7] = 0.0
    starts = np.arange(7)
    for temperature in (None, np.ones(6, np.float32)):
        tokens, counts = run(logits, np.zeros(6), starts, None, temperature, range(6), range(6))
        keep = [0, 1, 2, 4, 5]
        want = np.array([verify(logits[[i]], [0], [0, 1], None, None if temperature is None else temperature[:1], [i], [i])[0][0] for i in keep])
        assert np.array_equal(tokens[keep], want) and tokens[3] == 2 ** 31 - 1 and (counts == 1).all()
        assert tokens[1] < 10 and tokens[2] < 10 and tokens[4] == 7
    logits = np.zeros((1, 9), np.float32)      # ties go to the lowest index
    assert run(logits, [0], [0, 1])[0][0] == 0
    # the draft's own probabilities equal the target's: nothing is left over, and nothing is refused
    p = np.full((2, 8), 0.125, np.float32)
    tokens, counts = run(np.zeros((2, 8), np.float32), [3, 0], [0, 2], p, np.ones(1, np.float32), [1], [1])
    assert counts[0] == 2 and tokens[0] == 3


def test_a_draw_is_the_samplers_own():
    """Without drafts a request's token is what `sample` draws for the same seed and position."""
    rng = np.random.default_rng(3)
    logits = torch.from_numpy((rng.standard_normal((40, 5000)) * 2).astype(np.float32)).cuda()
    t = torch.full((40,), 0.7, device="cuda")
    seeds, positions = (torch.from_numpy(rng.integers(0, 2 ** 31, 40).astype(np.int32)).cuda() for _ in range(2))
    tokens, counts = ops.verify_drafts(logits, torch.zeros(40, dtype=torch.int32, device="cuda"), torch.arange(41, dtype=torch.int32, device="cuda"),
                                       None, t, seeds, positions)
    assert torch.equal(tokens, ops.sample(logits, t, seeds, positions)) and (counts == 1).all()


def test_emitted_tokens_have_the_targets_distribution():
    """40,000 requests with one draft each, drawn from another distribution: the first token's frequencies are p's."""
    rng = np.random.default_rng(4)
    vocab, n = 6, 20000
    p, q = np.array([0.4, 0.25, 0.2, 0.1, 0.05, 0.0]), np.array([0.05, 0.1, 0.15, 0.3, 0.3, 0.1])
    logits = np.where(p > 0, np.log(np.maximum(p, 1e-30)), -np.inf).astype(np.float32)[None].repeat(2 * n, axis=0)
    total = np.zeros(vocab)
    for turn in range(2):
        drafts = np.zeros(2 * n, np.int64)
        drafts[::2] = rng.choice(vocab, n, p=q)
        tokens, counts = run(logits, drafts, np.arange(0, 2 * n + 1, 2), np.tile(q.astype(np.float32), (2 * n, 1)), np.ones(n, np.float32),
                             np.arange(n) + turn * n, np.full(n, 77))
        total += np.bincount(tokens[::2], minlength=vocab)
        assert abs((counts == 2).mean() - np.minimum(p, q).sum()) < 5 * 0.5 / n ** 0.5
    # five standard deviations of a frequency of 2 n draws
    assert (np.abs(total / (2 * n) - p) <= 5 * np.sqrt(p * (1 - p) / (2 * n))).all()


def test_starts_outside_the_logits_are_reported():
    logits = torch.zeros((4, 10), device="cuda")
    drafts = torch.zeros(4, dtype=torch.int32, device="cuda")
    for starts in ([0, 5], [3, 2], [-1, 2]):
        _, counts = ops.verify_drafts(logits, drafts, torch.tensor(starts, dtype=torch.int32, device="cuda"))
        assert int(counts[0]) == 0
        with pytest.raises(ops.KernelError, match="outside the batch"):
            ops.take_device_errors()


def test_graphs_and_streams_do_not_meet():
    """Two captured calls and an eager one side by side: each has its own scratch."""
    rng = np.random.default_rng(5)
    xs = [torch.from_numpy((rng.standard_normal((30, 9000)) * 2).astype(np.float32)).cuda() for _ in range(2)]
    starts = torch.arange(0, 31, 5, dtype=torch.int32, device="cuda")
    drafts = torch.zeros(30, dtype=torch.int32, device="cuda")
    t, seeds = torch.ones(6, device="cuda"), torch.arange(6, dtype=torch.int32, device="cuda")
    call = lambda x: ops.verify_drafts(x, drafts, starts, None, t, seeds, seeds)  # noqa: E731
    graphs = []
    for x in xs:
        call(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(x)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for x in xs:
        x.neg_()
    want = [call(x) for x in xs]
    for _ in range(5):
        for s, (g, _) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        again = [call(x) for x in xs]
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for w, a, (_, o) in zip(want, again, graphs):
            assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(w, a, o))
