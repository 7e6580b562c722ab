"""Attention over the 8-bit cache where values are nothing, batches are mixed, host and device disagree, and scratch is scarce."""
import numpy as np
import pytest
import torch

from llm_inference_lab_b200.kernels import ops
from q8_helpers import Batch, attention, random_pages
from test_attention_q8_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e", [0, 10, 20, 30])
@pytest.mark.parametrize("rows, past", [([1], [3000]), ([5], [3000]), ([140], [2000])])
@pytest.mark.parametrize("d", [64, 128])
def test_keys_whose_values_are_nothing_keep_their_weight(rows, past, d, e):
    """Most values are rows of zeros, every 61st is of scale 2^e: the zeros' keys belong to the softmax's sum all the same."""
    rng = np.random.default_rng(21)

    def values(pages, batch):
        keep = torch.zeros(tuple(pages.v_scale.shape), dtype=torch.bool, device="cuda")
        for j in range(0, batch.held[0], 61):
            keep[int(batch.table[0, j // batch.page_size]), :, j % batch.page_size] = True
        pages.v.view(torch.uint8)[~keep] = 0
        pages.v_scale[~keep] = 127
        pages.v_scale[keep] = 127 + e
    check(rng, rows, past, 4, 2, d, 16, change=values, tail=0)


@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("splits", [1, 4, 20])
def test_tiles_of_nothing_keep_their_weight(monkeypatch, rows, splits):
    """Whole tiles of keys whose values are zeros, 2^-18 of the largest weight each and thousands of them: 1.5 % of the sum."""
    monkeypatch.setattr(ops, "q8_few_splits", lambda *_: splits)
    rng = np.random.default_rng(22)
    d, n_q, page, past = 64, 2, 16, 4090
    batch = Batch(rng, [rows], [past], page)
    pages = random_pages(ops, rng, batch.num_pages, 1, page, d, spread=0.0)
    first = batch.table[0, : 4096 // page].astype(np.int64)[: -8]      # all but the last tile
    pages.k[:] = 0.0
    pages.k_scale[:] = 127
    pages.v.view(torch.uint8)[first] = 0
    pages.v_scale[first] = 127
    pages.v_scale[batch.table[0, 4096 // page - 8:].astype(np.int64)] = 131
    last = batch.table[0, 4096 // page - 8].astype(np.int64)
    pages.k[last, 0, 0, 0] = 1.0                                       # one key of the last tile has nearly all the weight
    q = np.zeros((rows, n_q * d))
    q[:, ::d] = 12.5 * d ** 0.5                                        # e^12.5 = 2^18.03
    x = torch.from_numpy(q.astype(np.float32)).cuda().to(torch.bfloat16)
    out = ops.attention_q8(x, pages, *batch.args(), n_q, 1, d, 0, d ** -0.5).double().cpu().numpy()
    ops.take_device_errors()
    want, bound = attention(x, pages, batch, n_q, 1, d, 0, d ** -0.5, True)
    assert (np.abs(out - want) <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all()
    # the values of the last tile as if the others' keys were not there: 1.5 % off, and farther than what is allowed
    away = np.abs(want) * 0.014 > bound + 2.0 ** -8 * (np.abs(want) + bound)
    assert away.any()


def test_long_portions_that_see_no_key_at_all():
    """Every request's length is nothing: zeros, whatever the kernel."""
    batch = Batch(np.random.default_rng(23), [150, 1, 130], [0, 0, 0], 16, lengths=[0, 0, 0])
    pages = random_pages(ops, np.random.default_rng(23), 2, 2, 16, 64)
    x = torch.ones((batch.tokens, 4 * 64), dtype=torch.bfloat16, device="cuda")
    out = ops.attention_q8(x, pages, *batch.args(), 4, 2, 64, 0, 0.125, out=torch.full_like(x, 7.0))
    ops.take_device_errors()
    assert (out == 0).all()


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("d", [64, 128])
def test_a_portion_that_the_host_has_not_counted_is_left_alone(monkeypatch, splits, d):
    """Told one portion of 200 rows and a single token, the device has two of 200: the second is reported and its rows stay."""
    monkeypatch.setattr(ops, "q8_rows_splits", lambda ctas, keys: splits)
    rng = np.random.default_rng(25)
    batch = Batch(rng, [200, 200], [30, 40], 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, d)
    q_start, kv_len, pos0, table, *_ = batch.args()
    q = torch.from_numpy(rng.standard_normal((400, 4 * d)).astype(np.float32)).cuda().to(torch.bfloat16)
    want = ops.attention_q8(q, pages, q_start, kv_len, pos0, table, 2, [200, 200], 240, 4, 2, d, 0, d ** -0.5)
    out = torch.full_like(q, 7.0)
    ops.attention_q8(q, pages, q_start, kv_len, pos0, table, 2, [200, 1], 240, 4, 2, d, 0, d ** -0.5, out=out)
    with pytest.raises(ops.KernelError, match="row"):
        ops.take_device_errors()
    assert torch.equal(out[:200], want[:200]) and (out[200:] == 7.0).all()


@pytest.mark.parametrize("told, rows", [([1, 1], [1, 130]), ([5, 5, 5], [5, 60, 5]), ([1], [400])])
@pytest.mark.parametrize("d", [64, 128])
def test_a_request_longer_than_any_that_was_told_is_reported(told, rows, d):
    """The host's counts need the kernel for few rows alone; on the device one request has more than that kernel takes."""
    rng = np.random.default_rng(26)
    batch = Batch(rng, rows, [9] * len(rows), 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, d)
    q_start, kv_len, pos0, table, *_ = batch.args()
    q = torch.ones((batch.tokens, 4 * d), dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, torch.nan)      # (no result of these inputs is one)
    ops.attention_q8(q, pages, q_start, kv_len, pos0, table, len(told), told, 500, 4, 2, d, 0, d ** -0.5, out=out)
    with pytest.raises(ops.KernelError, match="row"):
        ops.take_device_errors()
    b = rows.index(max(rows))
    untouched = torch.isnan(out)
    own = slice(batch.starts[b], batch.starts[b + 1])
    assert untouched[own].all() and int(untouched.sum()) == untouched[own].numel()


@pytest.mark.parametrize("told, rows", [([200], [1]), ([150, 200], [3, 160]), ([200, 0], [0, 2]), ([200, 1], [130, 1])])
def test_requests_shorter_than_told_are_attended(told, rows):
    rng = np.random.default_rng(27)
    batch = Batch(rng, rows, [70] * len(rows), 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, 64)
    q_start, kv_len, pos0, table, _, _, most = batch.args()
    q = torch.from_numpy(rng.standard_normal((sum(told), 4 * 64)).astype(np.float32)).cuda().to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    ops.attention_q8(q, pages, q_start, kv_len, pos0, table, len(told), told, most, 4, 2, 64, 0, 0.125, out=out)
    ops.take_device_errors()
    got = out[: batch.tokens].double().cpu().numpy()
    want, bound = attention(q[: batch.tokens], pages, batch, 4, 2, 64, 0, 0.125, True)
    assert (np.abs(got - want) <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all() and (out[batch.tokens:] == 7.0).all()


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("rows", [
    [200] + [1] * 40, [1] * 40 + [200], [1] * 35 + [200, 0, 1, 150, 1, 1, 300] + [1] * 33, [150, 200, 5], [1, 130, 130], [0, 130, 0, 2, 0, 140, 0]])
@pytest.mark.parametrize("d", [64, 128])
def test_portions_among_many_single_tokens(monkeypatch, splits, rows, d):
    """First, last, in between and alone: every portion finds its keys, whatever stands beside it."""
    monkeypatch.setattr(ops, "q8_rows_splits", lambda ctas, keys: splits)
    rng = np.random.default_rng(28)
    past = [int(p) for p in rng.integers(0, 300, len(rows))]
    check(rng, rows, past, 4, 2, d, 16)
    monkeypatch.setattr(ops, "Q8_WIDE_BYTES", 1)
    check(rng, rows, past, 4, 2, d, 16, window=90)


@pytest.mark.parametrize("told, rows, lost", [
    ([1, 200, 1, 1], [1, 1, 200, 1], 2),            # the portion is another request's, behind the run
    ([200, 1, 200, 1], [200, 150, 200, 1], 2),      # three in the run where two were told: the last has no place
    ([1, 200, 1, 200], [150, 200, 1, 1], 0)])       # in front of the run
def test_portions_where_none_was_told_are_reported(told, rows, lost):
    rng = np.random.default_rng(29)
    batch = Batch(rng, rows, [20] * 4, 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, 64)
    q_start, kv_len, pos0, table, *_ = batch.args()
    q = torch.ones((max(sum(told), batch.tokens), 4 * 64), dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, torch.nan)
    ops.attention_q8(q, pages, q_start, kv_len, pos0, table, 4, told, 220, 4, 2, 64, 0, 0.125, out=out)
    with pytest.raises(ops.KernelError, match="row"):
        ops.take_device_errors()
    untouched = torch.isnan(out[: batch.tokens])
    own = untouched[batch.starts[lost]: batch.starts[lost + 1]]
    assert own.all() and int(untouched.sum()) == own.numel()


@pytest.mark.parametrize("splits", [1, 2])
def test_portions_told_and_not_there(monkeypatch, splits):
    """Two portions were told; the first has no rows on the device: the second finds its own keys."""
    monkeypatch.setattr(ops, "q8_rows_splits", lambda ctas, keys: splits)
    rng = np.random.default_rng(30)
    batch = Batch(rng, [0, 150, 140], [70, 300, 5], 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, 64)
    q_start, kv_len, pos0, table, _, _, most = batch.args()
    q = torch.from_numpy(rng.standard_normal((600, 4 * 64)).astype(np.float32)).cuda().to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    ops.attention_q8(q, pages, q_start, kv_len, pos0, table, 3, [200, 200, 200], most, 4, 2, 64, 0, 0.125, out=out)
    ops.take_device_errors()
    got = out[: batch.tokens].double().cpu().numpy()
    want, bound = attention(q[: batch.tokens], pages, batch, 4, 2, 64, 0, 0.125, True)
    assert (np.abs(got - want) <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all() and (out[batch.tokens:] == 7.0).all()


def test_scratch_of_splits_counts_too(monkeypatch):
    """One long portion beside many short ones: keys, values and the splits' results stay within the bound together."""
    rng = np.random.default_rng(24)
    monkeypatch.setattr(ops, "q8_rows_splits", lambda ctas, keys: 2)
    n_q, d, page = 1, 128, 16
    batch = Batch(rng, [2048] + [100] * 30, [0] * 31, page)
    pages = random_pages(ops, rng, batch.num_pages, 1, page, d)
    x = torch.randn((batch.tokens, n_q * d), device="cuda").to(torch.bfloat16)
    args = batch.args()
    together = ops.attention_q8(x, pages, *args, n_q, 1, d, 0, d ** -0.5)
    # 31 requests of 17 tiles of keys and values, 34.6 MB, with 31 x 16 tiles x 2 splits' results 66 MB more
    monkeypatch.setattr(ops, "Q8_WIDE_BYTES", 40 << 20)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    apart = ops.attention_q8(x, pages, *args, n_q, 1, d, 0, d ** -0.5)
    taken = torch.cuda.max_memory_allocated() - before
    ops.take_device_errors()
    assert torch.equal(together, apart)
    assert taken <= (40 << 20) + apart.nbytes + 2 ** 20


@pytest.mark.parametrize("rows, past, n_q, n_kv, d", [
    ([1, 1], [300, 4], 100, 2, 64),              # 50 query heads a kv head: two tiles of rows for one token
    ([1], [3000], 160, 1, 64), ([2, 1], [90, 700], 60, 1, 128), ([1, 1, 1], [10, 0, 150], 130, 1, 128)])
@pytest.mark.parametrize("window", [0, 70])
def test_more_rows_than_a_tile_of_the_few_rows_kernel(rows, past, n_q, n_kv, d, window):
    check(np.random.default_rng(31), rows, past, n_q, n_kv, d, 16, window=window)


@pytest.mark.parametrize("rows, past", [([70], [40]), ([33, 5, 1], [0, 600, 90]), ([140, 1], [300, 3])])
@pytest.mark.parametrize("d, shift", [(64, 2), (64, 4), (128, 6)])
def test_queries_off_their_boundaries_take_any_number_of_rows(rows, past, d, shift):
    """Queries 4, 8 or 12 bytes off a boundary of 16 are the few-rows kernel's, however many rows they have."""
    rng = np.random.default_rng(32)
    n_q, n_kv, page = 6, 2, 16
    batch = Batch(rng, rows, past, page)
    pages = random_pages(ops, rng, batch.num_pages, n_kv, page, d)
    wide = torch.zeros((batch.tokens, n_q * d + 8), dtype=torch.bfloat16, device="cuda")
    q = wide[:, shift: shift + n_q * d]
    q.copy_(torch.from_numpy(rng.standard_normal((batch.tokens, n_q * d)).astype(np.float32)))
    out = torch.full((batch.tokens, n_q * d + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.attention_q8(q, pages, *batch.args(), n_q, n_kv, d, 0, d ** -0.5, out=out[:, 1: 1 + n_q * d])
    ops.take_device_errors()
    assert (out[:, 0] == 7.0).all() and (out[:, 1 + n_q * d:] == 7.0).all()
    got = out[:, 1: 1 + n_q * d].double().cpu().numpy()
    want, bound = attention(q, pages, batch, n_q, n_kv, d, 0, d ** -0.5, True)
    assert (np.abs(got - want) <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all()


def test_the_first_call_may_be_a_captured_one(monkeypatch):
    """How many clusters find room is asked for within a capture too; a replay twice and an eager call leave the same bits."""
    monkeypatch.setattr(ops, "_q8_places", {})
    rng = np.random.default_rng(33)
    batch = Batch(rng, [5, 5, 200, 1], [900, 30, 0, 2000], 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, 128)
    q = torch.from_numpy(rng.standard_normal((batch.tokens, 14 * 128)).astype(np.float32)).cuda().to(torch.bfloat16)
    args = batch.args()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attention_q8(q, pages, *args, 14, 2, 128, 0, 128 ** -0.5)
    assert ops._q8_places and all(n > 0 for found in ops._q8_places.values() for n in found[1:])
    seen = []
    for _ in range(2):
        out.zero_()
        graph.replay()
        seen.append(out.clone())
    eager = ops.attention_q8(q, pages, *args, 14, 2, 128, 0, 128 ** -0.5)
    ops.take_device_errors()
    assert torch.equal(seen[0], seen[1]) and torch.equal(seen[0], eager)
