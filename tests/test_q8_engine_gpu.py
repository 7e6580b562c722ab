"""An engine whose cache is in 8 bits, and steps over drafted tokens: store, attention, reading back and verification together."""
import contextlib

import numpy as np
import pytest
import torch

from helpers import TINY, make_model_folder, random_tokens
from llm_inference_lab_b200.engine.engine import Engine, Entry, InvalidInput
from llm_inference_lab_b200.engine.llm import LLM
from llm_inference_lab_b200.kernels import ops
from llm_inference_lab_b200.sampling import SamplingConfig
from q8_helpers import attention, encode

pytestmark = pytest.mark.gpu
_folders = {}


def folder_of(tmp_path_factory, name, dtype="bfloat16"):
    if (name, dtype) not in _folders:
        cfg, opt = TINY[name]
        _folders[(name, dtype)] = make_model_folder(str(tmp_path_factory.mktemp(f"q8{name}{dtype}")), cfg, opt["seed"], dtype)
    return _folders[(name, dtype)]


def plain_store(qkv, table, rotary_dim, slots, pages, n_q, n_kv, head_dim, bias=None):
    x = qkv.double()
    if qkv.dim() == 3:
        x = x.sum(dim=0)
        x = (x if bias is None else x + bias.double()).to(torch.bfloat16).double()
    x, half = x.view(-1, n_q + 2 * n_kv, head_dim), rotary_dim // 2
    if rotary_dim:
        c, s = table.double()[:, None].unbind(-1)
        lo, hi = x[:, : n_q + n_kv, :half].clone(), x[:, : n_q + n_kv, half: rotary_dim].clone()
        x[:, : n_q + n_kv, :half], x[:, : n_q + n_kv, half: rotary_dim] = lo * c - hi * s, hi * c + lo * s
    ps = pages.k.shape[2]
    for t, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        for codes, scale, rows in ((pages.k, pages.k_scale, x[t, n_q: n_q + n_kv]), (pages.v, pages.v_scale, x[t, n_q + n_kv:])):
            new, byte = encode(rows.cpu().numpy())
            codes.view(torch.uint8)[slot // ps, :, slot % ps] = torch.from_numpy(new).cuda()
            scale[slot // ps, :, slot % ps] = torch.from_numpy(byte).cuda()
    return x[:, :n_q].reshape(x.shape[0], -1).to(torch.bfloat16)


class Held:
    """A step's requests as `q8_helpers.attention` takes them."""

    def __init__(self, q_start, kv_len, pos0, block_table, n_requests, q_lens, page_size):
        self.rows, self.starts, self.page_size = list(q_lens), q_start.cpu().numpy(), page_size
        self.past, self.held = pos0.cpu().numpy()[:n_requests].tolist(), kv_len.cpu().numpy()[:n_requests].tolist()
        self.table, self.tokens = block_table.cpu().numpy(), int(self.starts[n_requests])


@contextlib.contextmanager
def every_call_checked(monkeypatch, seen):
    """Every store's bytes against the definition's, every attention's rows against the definition within its bound, on the very
    arguments that the model's layers give them."""
    store, attend = ops.rope_kv_store_q8, ops.attention_q8

    def checked_store(qkv, table, rotary_dim, slots, pages, n_q, n_kv, head_dim, bias=None):
        copy = ops.QuantPages(*(t.clone() for t in pages))
        want = plain_store(qkv.clone(), table, rotary_dim, slots, copy, n_q, n_kv, head_dim, bias)
        q = store(qkv, table, rotary_dim, slots, pages, n_q, n_kv, head_dim, bias)
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(pages, copy))
        # the rotation in 32 bits (under 2^-21 of the largest number that enters it) and one rounding to bfloat16, on either side
        assert ((q.double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 2.0 ** -20 * qkv.abs().max()).all()
        seen.append("store")
        return q

    def checked_attend(q, pages, q_start, kv_len, pos0, block_table, n_requests, q_lens, max_kv_len, n_q, n_kv, head_dim, window, scale):
        out = attend(q, pages, q_start, kv_len, pos0, block_table, n_requests, q_lens, max_kv_len, n_q, n_kv, head_dim, window, scale)
        held = Held(q_start, kv_len, pos0, block_table, n_requests, q_lens, pages.k.shape[2])
        codes_of_p = head_dim in (64, 128) and pages.k.shape[2] in (8, 16, 32, 64, 128)
        want, bound = attention(q, pages, held, n_q, n_kv, head_dim, window, scale, codes_of_p)
        off = np.abs(out.double().cpu().numpy()[: held.tokens] - want[: held.tokens])
        assert (off <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all()
        seen.append("attention")
        return out

    with monkeypatch.context() as m:
        m.setattr(ops, "rope_kv_store_q8", checked_store)
        m.setattr(ops, "attention_q8", checked_attend)
        yield


@pytest.mark.parametrize("name", ["A", "C", "D", "F", "G"])
def test_every_layer_of_every_step(tmp_path_factory, monkeypatch, name):
    """Whole prompts, portions beside single tokens, windows, heads of 16, 48, 64, 80 and 128."""
    cfg, opt = TINY[name]
    rng = np.random.default_rng(3)
    steps = [[(0, 37), (1, 5)], [(0, 1), (1, 30)], [(0, 9), (1, 1), (2, 70)], [(0, 1), (1, 1), (2, 1)]]
    engine = Engine(folder_of(tmp_path_factory, name), "bf16", page_size=opt["page_size"], max_tokens=512, max_requests=4, cache_dtype="e4m3")
    assert all(v.k is None and v.pages8 is not None for v in engine.views)
    seen = []
    with every_call_checked(monkeypatch, seen):
        for step in steps:
            logits = engine.step([Entry(r, random_tokens(rng, n, cfg["vocab_size"]), range(n)) for r, n in step])
            assert torch.isfinite(logits).all()
    ops.take_device_errors()
    assert seen == ["store", "attention"] * (len(steps) * cfg["num_hidden_layers"])


@pytest.mark.parametrize("name", ["F", "G"])
def test_generation_from_graphs_and_eagerly(tmp_path_factory, monkeypatch, name):
    """Requests that come and go, portions of prompts, every call checked; then decode steps from graphs.  A graph is captured for a
    bucket of lengths, an eager step for its own: with the keys split alike both are the same kernels on the same numbers, and the
    same tokens."""
    cfg, opt = TINY[name]
    folder = folder_of(tmp_path_factory, name)
    rng = np.random.default_rng(4)
    prompts = [random_tokens(rng, n, cfg["vocab_size"]) for n in (5, 90, 33, 1, 61)]
    make = lambda graph: LLM(folder, "bf16", page_size=opt["page_size"], kv_tokens=1024, max_requests=3, max_batch_tokens=64,  # noqa: E731
                             cuda_graph=graph, cache_dtype="e4m3")
    seen = []
    with every_call_checked(monkeypatch, seen):
        llm = make(False)
        results = llm.generate(prompts, SamplingConfig(max_new_tokens=6, ignore_eos=True))
    ops.take_device_errors()
    assert llm.engine.cache.live_requests == 0 and all(len(r.tokens) == 6 for r in results) and "attention" in seen
    monkeypatch.setattr(ops, "q8_few_splits", lambda *_: 1)
    for batch in (prompts[:1], prompts[1:3]):
        tokens = []
        for graph in (False, True):
            llm = make(graph)
            tokens.append([r.tokens for r in llm.generate(batch, SamplingConfig(max_new_tokens=20, ignore_eos=True))])
            assert not graph or llm.graphs.replays > 10
        assert tokens[0] == tokens[1]
    ops.take_device_errors()


def test_cached_rows(tmp_path_factory):
    """The first layer's keys and values of an 8-bit and a 16-bit cache differ by what rounding to 8 and 16 bits allows."""
    cfg, opt = TINY["G"]
    prompt = random_tokens(np.random.default_rng(5), 40, cfg["vocab_size"])
    rows = []
    for how in ("auto", "e4m3"):
        engine = Engine(folder_of(tmp_path_factory, "G"), "bf16", page_size=opt["page_size"], max_tokens=256, max_requests=2, cache_dtype=how)
        engine.step([Entry(7, prompt[:25])])
        engine.step([Entry(7, prompt[25:])])
        rows.append([t.double().cpu().numpy() for t in engine.cached_rows(7)])
        assert rows[-1][0].shape == (40, cfg["num_key_value_heads"], cfg["head_dim"])
    for a, b in zip(*rows):
        # half a step of 8 bits, at least 2^-10 of a scale of at most 2^-7 of the row's largest; half a step of 16 bits for the
        # other cache, and (keys) of the projection's rounding, which a product of other shape may do otherwise
        top = np.abs(a).max(axis=-1, keepdims=True)
        assert (np.abs(a - b) <= (2.0 ** -4 + 2 * 2.0 ** -8) * np.abs(a) + (2.0 ** -17 + 2 * 2.0 ** -8) * top).all()
        assert np.abs(a - b).max() > 0


def test_rows_that_a_window_has_left_are_zeros(tmp_path_factory):
    cfg, opt = TINY["C"]
    engine = Engine(folder_of(tmp_path_factory, "C"), "bf16", page_size=opt["page_size"], max_tokens=256, max_requests=2, cache_dtype="e4m3")
    engine.step([Entry(1, random_tokens(np.random.default_rng(6), 60, cfg["vocab_size"]))])
    seen = [(engine.cached_rows(1, i)[0] != 0).any(dim=-1).any(dim=-1).cpu().numpy() for i in range(len(engine.views))]
    windows = [v.need.window for v in engine.views]
    assert 0 in windows and max(windows) > 0
    for rows, window in zip(seen, windows):
        assert rows.all() if window == 0 else rows[60 - window:].all() and not rows[: 60 - window - 2 * opt["page_size"]].any()


@pytest.mark.parametrize("dtype, cache", [("f32", "auto"), ("bf16", "auto"), ("bf16", "e4m3")])
def test_drafts_change_nothing_but_the_number_of_steps(tmp_path_factory, dtype, cache):
    """Greedy tokens with right, wrong and no drafts.  The 32-bit engine does not depend on how a sequence is cut: its tokens are
    those of `generate`.  In 16 bits a token may be another where two logits are as near as the cut's roundings (0.09 of their size,
    as for the engine's other cuts); over a cache in 8 bits, whose codes amplify them, what was accepted and what is held is looked at."""
    cfg, opt = TINY["F"]
    folder = folder_of(tmp_path_factory, "F", "float32" if dtype == "f32" else "bfloat16")
    rng = np.random.default_rng(7)
    prompts = [random_tokens(rng, n, cfg["vocab_size"]) for n in (6, 40, 17)]
    llm = LLM(folder, dtype, page_size=opt["page_size"], kv_tokens=512, max_requests=4, cache_dtype=cache)
    want = [r.tokens for r in llm.generate(prompts, SamplingConfig(max_new_tokens=12, ignore_eos=True))]
    engine = Engine(folder, dtype, page_size=opt["page_size"], max_tokens=512, max_requests=4, cache_dtype=cache)
    logits = engine.step([Entry(i, p, [len(p) - 1]) for i, p in enumerate(prompts)])
    made = [[int(t)] for t in logits.argmax(dim=-1)]
    free = engine.free_pages()
    while min(len(m) for m in made) < 12:
        entries = []
        for i, m in enumerate(made):
            drafts = want[i][len(m): len(m) + int(rng.integers(0, 5))]      # right ones
            if drafts and rng.random() < 0.5:
                drafts[int(rng.integers(0, len(drafts)))] = int(rng.integers(0, cfg["vocab_size"]))      # one of them wrong, as a rule
            entries.append((i, m[-1], drafts))
        for m, e, new in zip(made, entries, engine.verify_step(entries)):
            assert 1 <= len(new) <= len(e[2]) + 1 and new[:-1] == list(e[2])[: len(new) - 1]
            m += new
        for i, (p, m) in enumerate(zip(prompts, made)):
            assert engine.length(i) == len(p) + len(m) - 1      # the last token is not in the cache yet
    ops.take_device_errors()
    if dtype == "f32":
        assert [m[:12] for m in made] == want
    elif cache == "auto":
        check = Engine(folder, dtype, page_size=opt["page_size"], max_tokens=512, max_requests=4, cache_dtype=cache)
        for i, (p, m) in enumerate(zip(prompts, made)):
            rows = check.step([Entry(i, p + m[:-1], range(len(p) - 1, len(p) + len(m) - 1))]).cpu().numpy()
            assert all(row.max() - row[t] <= 0.09 * np.abs(row).max() for row, t in zip(rows, m))
    for i in range(3):
        engine.close(i)
    assert engine.free_pages()[0] == engine.num_pages and free[0] < engine.num_pages


def test_sampled_drafts(tmp_path_factory):
    """At a temperature a seed and a position decide a draw: without drafts the sampler's own token, with certain drafts of it too
    (a refused draft is one that the draw would not have been; an accepted one may differ from what it would have drawn)."""
    cfg, opt = TINY["A"]
    folder = folder_of(tmp_path_factory, "A", "float32")
    prompt = random_tokens(np.random.default_rng(8), 9, cfg["vocab_size"])
    engine = Engine(folder, "f32", page_size=opt["page_size"], max_tokens=256, max_requests=4)
    llm = LLM(folder, "f32", page_size=opt["page_size"], kv_tokens=256, max_requests=4)
    want = llm.generate([prompt], SamplingConfig(max_new_tokens=6, do_sample=True, temperature=0.9, seed=11, ignore_eos=True))[0].tokens
    engine.step([Entry(0, prompt[:-1])])
    last, made = prompt[-1], []
    for _ in range(6):
        made += engine.verify_step([(0, last, [])], [0.9], [11])[0]
        last = made[-1]
    assert made == want
    vocab = cfg["vocab_size"]
    probs = torch.full((3, vocab), 1.0 / vocab, device="cuda")
    new = engine.verify_step([(0, last, [3, 5])], [0.9], [11], draft_probs=probs)[0]
    assert 1 <= len(new) <= 3 and all(0 <= t < vocab for t in new)


def test_refusals(tmp_path_factory):
    cfg, opt = TINY["A"]
    folder = folder_of(tmp_path_factory, "A", "float32")
    with pytest.raises(ValueError, match="bfloat16 engine"):
        Engine(folder, "f32", max_tokens=64, max_requests=2, cache_dtype="e4m3")
    with pytest.raises(ValueError, match="unknown cache_dtype"):
        Engine(folder, "bf16", max_tokens=64, max_requests=2, cache_dtype="fp8")
    engine = Engine(folder, "bf16", page_size=opt["page_size"], max_tokens=64, max_requests=2)
    for entries, temperatures, seeds, says in (([(0, 1, [cfg["vocab_size"]])], None, None, "token id"), ([], None, None, "at least one"),
                                               ([(0, 1, []), (0, 2, [])], None, None, "twice"), ([(0, 1, [2])], [1.0], None, "a temperature and a seed")):
        with pytest.raises(InvalidInput, match=says):
            engine.verify_step(entries, temperatures, seeds)
    assert not engine.has(0)


def test_models_that_do_not_take_it_are_refused(tmp_path_factory):
    from sogulix_helpers import SMALL, SPREAD
    cfg, opt = SMALL["A"]
    folder = make_model_folder(str(tmp_path_factory.mktemp("q8sogulix")), cfg, opt["seed"], "bfloat16", std=0.08, scales=SPREAD)
    with pytest.raises(ValueError, match="does not take its cache in 8 bits"):
        Engine(folder, "bf16", page_size=opt["page_size"], max_tokens=64, max_requests=2, cache_dtype="e4m3")
    engine = Engine(folder, "bf16", page_size=opt["page_size"], max_tokens=64, max_requests=2)
    with pytest.raises(InvalidInput, match="fixed-size state"):
        engine.verify_step([(0, 1, [2])])


def test_drafted_steps_from_step_graphs(tmp_path_factory, monkeypatch):
    """Steps over drafted tokens whose shape repeats are captured and replayed: the eager engine's tokens, greedy and drawn."""
    cfg, opt = TINY["G"]
    folder = folder_of(tmp_path_factory, "G")
    monkeypatch.setattr(ops, "q8_few_splits", lambda *_: 1)      # (a captured step is one for a bucket of lengths)
    monkeypatch.setattr(ops, "q8_rows_splits", lambda *_: 1)
    told = []
    for graphs in (False, True):
        rng = np.random.default_rng(6)
        engine = Engine(folder, "bf16", page_size=opt["page_size"], max_tokens=1024, max_requests=4, cache_dtype="e4m3")
        if graphs:
            engine.enable_step_graphs()
        prompts = [random_tokens(rng, n, cfg["vocab_size"]) for n in (40, 7)]
        engine.step([Entry(r, p, [len(p) - 1]) for r, p in enumerate(prompts)])
        held, out = [3, 5], []
        for i in range(12):
            drafts = [random_tokens(rng, 3, cfg["vocab_size"]) for _ in range(2)]
            drawn = ([0.9, 0.7], [11, 12]) if i % 3 == 2 else (None, None)
            new = engine.verify_step([(r, held[r], drafts[r]) for r in range(2)], *drawn)
            held = [t[-1] for t in new]
            out.append(new)
        assert not graphs or engine.graph_replays >= 8
        told.append((out, [engine.length(r) for r in range(2)]))
        ops.take_device_errors()
    assert told[0] == told[1]
