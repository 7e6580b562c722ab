"""Attention over the 8-bit cache against the definition in 64 bits: tensor-core kernels and the one on the ordinary units."""
import numpy as np
import pytest
import torch

from llm_inference_lab_b200.kernels import ops
from q8_helpers import Batch, attention, random_pages

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def on_tensor_cores(dtype, d, page):
    return dtype == torch.bfloat16 and d in (64, 128) and page in (8, 16, 32, 64, 128)


def check(rng, rows, past, n_q, n_kv, d, page, window=0, dtype=torch.bfloat16, lengths=None, q=None, change=None, spread=0.7, tail=3):
    """Runs a batch and checks every row; `tail` rows behind the last request have to stay as they were."""
    batch = Batch(rng, rows, past, page, lengths=lengths)
    pages = random_pages(ops, rng, batch.num_pages, n_kv, page, d, spread=spread)
    if change is not None:
        change(pages, batch)
    if q is None:
        q = rng.standard_normal((batch.tokens + tail, n_q * d)) * np.exp(rng.standard_normal((batch.tokens + tail, 1)))
    q = torch.from_numpy(np.asarray(q, np.float32)).cuda().to(dtype)
    scale = d ** -0.5
    out = torch.full((batch.tokens + tail, n_q * d), 7.0, dtype=dtype, device="cuda")
    ops.attention_q8(q, pages, *batch.args(), n_q, n_kv, d, window, scale, out=out)
    ops.take_device_errors()
    assert (out[batch.tokens:] == 7.0).all()
    got = out[: batch.tokens].double().cpu().numpy()
    want, bound = attention(q[: batch.tokens], pages, batch, n_q, n_kv, d, window, scale, on_tensor_cores(dtype, d, page))
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    over = np.abs(got - want)[fine] - bound[fine] - HALF[dtype] * (np.abs(want)[fine] + bound[fine])
    assert over.size == 0 or over.max() <= 0, f"off by {np.abs(got - want)[fine].max():.3g}, {over.max():.3g} more than the bound"
    return got, want


SHAPES = [
    ([1], [0]), ([1], [127]), ([1], [128]), ([1] * 5, [0, 3, 300, 17, 128]),                # single tokens, lengths from one on
    ([5], [0]), ([3, 1, 8], [700, 5, 40]), ([2] * 6, [129, 0, 64, 255, 1, 400]),            # drafted tokens
    ([40, 1], [0, 60]), ([130], [3]), ([0, 7, 0, 1], [0, 90, 0, 12]), ([300, 5], [0, 700]),  # portions, requests without rows
]


@pytest.mark.parametrize("rows, past", SHAPES)
@pytest.mark.parametrize("n_q, n_kv, d, page", [(14, 2, 64, 16), (8, 2, 128, 32), (20, 1, 64, 8), (3, 3, 128, 128)])
def test_tensor_cores(rows, past, n_q, n_kv, d, page):
    check(np.random.default_rng(len(rows) + d + page), rows, past, n_q, n_kv, d, page)


@pytest.mark.parametrize("rows, past", [([1, 1, 4], [0, 200, 33]), ([70, 0], [10, 0])])
@pytest.mark.parametrize("n_q, n_kv, d, page, dtype", [
    (4, 2, 64, 16, torch.float32), (3, 1, 128, 24, torch.bfloat16), (2, 2, 33, 5, torch.bfloat16), (6, 2, 256, 16, torch.float32),
    (2, 1, 80, 64, torch.bfloat16), (5, 5, 1, 1, torch.float32)])
def test_ordinary_units(rows, past, n_q, n_kv, d, page, dtype):
    check(np.random.default_rng(d), rows, past, n_q, n_kv, d, page, dtype=dtype)


@pytest.mark.parametrize("window", [1, 5, 128, 130, -1, -64, -100])
@pytest.mark.parametrize("rows, past", [([1, 1, 1], [0, 500, 131]), ([6, 3], [400, 60]), ([150], [200])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_windows_and_chunks(window, rows, past, dtype):
    def given_back(pages, batch):
        # pages that no row's window reaches have been given back: nothing may be read from them
        for b, (r, p) in enumerate(zip(batch.rows, batch.past)):
            first = max(0, p - window + 1) if window > 0 else p // -window * -window
            batch.table[b, : first // batch.page_size] = -1
    rng = np.random.default_rng(abs(window))
    if dtype == torch.bfloat16:
        check(rng, rows, past, 6, 2, 64, 16, window=window, change=given_back)
    check(rng, rows, past, 4, 2, 128, 16, window=window, dtype=dtype, change=given_back)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_see_nothing_are_zero(dtype):
    """Lengths that end before a row's window, and lengths of nothing."""
    got, want = check(np.random.default_rng(1), [3, 4, 1, 2], [0, 300, 0, 40], 4, 2, 64, 16, window=20, dtype=dtype, lengths=[0, 150, 0, 42])
    assert (got[:8] == 0).all() and (got[8:] != 0).any()


def poison(pages, batch, b, position, what):
    """The key's or value's row at a request's position, in every kv head, is no number."""
    page, at = batch.table[b, position // batch.page_size], position % batch.page_size
    getattr(pages, what + "_scale")[page, :, at] = 255
    getattr(pages, what)[page, :, at] = 0.0


@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_are_no_numbers_reach_those_that_see_them(what, dtype):
    """Request 0's rows before position 44 do not see the NaN there; request 1's window has left it."""
    got, _ = check(np.random.default_rng(2), [8, 1, 1], [40, 300, 9], 4, 2, 64, 16, window=50, dtype=dtype,
                   change=lambda p, b: (poison(p, b, 0, 44, what), poison(p, b, 1, 240, what)))
    assert not np.isnan(got[:4]).any() and np.isnan(got[4:8]).all() and not np.isnan(got[8:]).any()


@pytest.mark.parametrize("d", [64, 128])
def test_what_lies_behind_the_last_key_does_not_matter(d):
    """Codes that are no numbers, and scales that are none, behind the end of a page's rows and on spare pages."""
    def stale(pages, batch):
        used = np.zeros((batch.num_pages, batch.page_size), bool)
        for b, n in enumerate(batch.held):
            for j in range(n):
                used[batch.table[b, j // batch.page_size], j % batch.page_size] = True
        rest = torch.from_numpy(~used).cuda()[:, None, :].expand(-1, pages.k.shape[1], -1)
        for codes, scale in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
            codes.view(torch.uint8)[rest] = 0x7F
            scale[rest] = 255
    for rows, past in (([1, 1], [2, 140]), ([5, 3], [20, 131]), ([70], [3])):
        got, _ = check(np.random.default_rng(5), rows, past, 8, 2, d, 16, change=stale)
        assert not np.isnan(got).any()


def test_queries_that_are_no_numbers_stay_in_their_rows():
    rng = np.random.default_rng(6)
    q = rng.standard_normal((9, 4 * 64))
    q[2, 64 + 5], q[7, 3] = np.nan, np.inf
    batch = Batch(rng, [5, 1], [30, 200], 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, 64)
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.from_numpy(q[:6].astype(np.float32)).cuda().to(dtype)
        out = ops.attention_q8(x, pages, *batch.args(), 4, 2, 64, 0, 0.125).view(6, 4, 64)
        nan = torch.isnan(out).all(dim=-1)
        assert nan[2, 1] and int(torch.isnan(out).any(dim=-1).sum()) == 1 == int(nan.sum())


@pytest.mark.parametrize("rows", [1, 5, 150])
@pytest.mark.parametrize("d", [64, 128])
def test_long_tail_behind_one_dominant_key(rows, d):
    """The first key holds nearly all weight, and its value is nothing: what comes out is the tail's alone, keys of 2^-19 each."""
    rng = np.random.default_rng(7)
    n_q, n_kv, page, past = 2, 1, 16, 2500
    batch = Batch(rng, [rows], [past], page)
    pages = random_pages(ops, rng, batch.num_pages, n_kv, page, d, spread=0.0)
    first = batch.table[0, 0]
    pages.k[:] = 0.0
    pages.k_scale[:] = 127
    pages.k[first, :, 0, 0] = 1.0
    pages.v[first, :, 0] = 0.0
    pages.v_scale[first, :, 0] = 127
    q = np.zeros((rows, n_q * d))
    q[:, ::d] = 13.0 * d ** 0.5      # e^13 = 2^18.8
    x = torch.from_numpy(q.astype(np.float32)).cuda().to(torch.bfloat16)
    out = ops.attention_q8(x, pages, *batch.args(), n_q, n_kv, d, 0, d ** -0.5).double().cpu().numpy()
    want, bound = attention(x, pages, batch, n_q, n_kv, d, 0, d ** -0.5, True)
    assert (np.abs(out - want) <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all()
    # the bound's term for codes is largest in the first tile; the tail as a whole has to be there
    assert np.linalg.norm(out - want) < 0.01 * np.linalg.norm(want)


@pytest.mark.parametrize("rows, past", [([1], [700]), ([4], [300]), ([140], [0])])
def test_values_and_queries_of_very_different_sizes(rows, past):
    """Values and queries over 2^30: p' goes by the value's scale, q by its row's."""
    rng = np.random.default_rng(8)
    q = rng.standard_normal((sum(rows), 6 * 64)) * 2.0 ** rng.integers(-30, 3, (sum(rows), 6)).repeat(64, axis=1)
    def wide(pages, batch):
        pages.v_scale[:] = torch.from_numpy(rng.integers(107, 137, tuple(pages.v_scale.shape)).astype(np.uint8)).cuda()
    check(rng, rows, past, 6, 2, 64, 16, q=q, change=wide, tail=0)


def test_rows_of_a_wider_projection_and_odd_places():
    """q as columns of the fused projection, out with rows of its own distance, rows off every boundary."""
    rng = np.random.default_rng(10)
    batch = Batch(rng, [3, 1], [50, 9], 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, 64)
    x = torch.from_numpy(rng.standard_normal((4, 6 * 64)).astype(np.float32)).cuda().to(torch.bfloat16)
    want = ops.attention_q8(x, pages, *batch.args(), 6, 2, 64, 0, 0.125)
    for shift, width in ((0, 10 * 64), (1, 6 * 64 + 3), (2, 6 * 64 + 2), (3, 6 * 64 + 4)):
        wide = torch.zeros((4, width + 4), dtype=torch.bfloat16, device="cuda")
        wide[:, shift: shift + 6 * 64] = x
        out = torch.zeros((4, width + 4), dtype=torch.bfloat16, device="cuda")
        view = out[:, shift: shift + 6 * 64]
        ops.attention_q8(wide[:, shift: shift + 6 * 64], pages, *batch.args(), 6, 2, 64, 0, 0.125, out=view)
        # (rows off a boundary of four bytes run on the ordinary units)
        assert (view.float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()
        out[:, shift: shift + 6 * 64] = 0
        assert (out == 0).all()


@pytest.mark.parametrize("bad", [-1, 10 ** 6])
@pytest.mark.parametrize("rows, dtype", [([1], torch.bfloat16), ([5], torch.bfloat16), ([140], torch.bfloat16), ([2], torch.float32)])
def test_pages_outside_the_pool_are_reported(bad, rows, dtype):
    rng = np.random.default_rng(11)
    batch = Batch(rng, rows, [100], 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, 64)
    batch.table[0, 3] = bad
    ops.attention_q8(torch.ones((sum(rows), 256), dtype=dtype, device="cuda"), pages, *batch.args(), 4, 2, 64, 0, 0.125)
    with pytest.raises(ops.KernelError, match="outside the pool"):
        ops.take_device_errors()


def test_streams_and_graphs():
    """On a stream of its own, and two captured calls replayed in turn with other inputs: the eager results' bits."""
    rng = np.random.default_rng(12)
    kinds = [Batch(rng, [1, 1], [600, 40], 16), Batch(rng, [4, 2], [300, 700], 16), Batch(rng, [200], [10], 16)]
    pages = [random_pages(ops, rng, b.num_pages, 2, 16, 64) for b in kinds]
    xs = [torch.randn((b.tokens, 14 * 64), device="cuda").to(torch.bfloat16) for b in kinds]
    args = [b.args() for b in kinds]
    call = lambda i: ops.attention_q8(xs[i], pages[i], *args[i], 14, 2, 64, 0, 0.125)  # noqa: E731
    eager = [call(i) for i in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        moved = [call(i) for i in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, moved))
    graphs = []
    for i in range(3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(i)
        graphs.append((g, out))
    for round_ in range(2):
        for x in xs:
            x.mul_(-0.5)
        eager = [call(i) for i in range(3)]
        for g, _ in graphs:
            g.replay()
        assert all(torch.equal(a, out) for a, (_, out) in zip(eager, graphs))


def test_two_ways_agree_on_stored_rows():
    """Stored, attended and read back together: the attention's rows are those of the read-back keys and values."""
    rng = np.random.default_rng(13)
    n_q, n_kv, d, page = 14, 2, 64, 16
    for rows, past in (([6], [0]), ([1], [70]), ([150], [0])):
        total = rows[0] + past[0]
        batch = Batch(rng, rows, past, page)
        pages = ops.quant_pages(batch.num_pages, n_kv, page, d, "cuda")
        qkv = torch.randn((total, (n_q + 2 * n_kv) * d), device="cuda").to(torch.bfloat16)
        angle = torch.rand((total, d // 2), device="cuda") * 6
        table = torch.stack((angle.cos(), angle.sin()), dim=-1).contiguous()
        slots = torch.tensor([batch.table[0, j // page] * page + j % page for j in range(total)], dtype=torch.int32, device="cuda")
        q = ops.rope_kv_store_q8(qkv, table, d, slots, pages, n_q, n_kv, d)[past[0]:]
        out = ops.attention_q8(q, pages, *batch.args(), n_q, n_kv, d, 0, d ** -0.5).double().view(rows[0], n_kv, -1, d)
        k, v = (t.double() for t in ops.kv_load_q8(pages, slots))
        s = torch.einsum("tkgd,jkd->tkgj", q.double().view(rows[0], n_kv, -1, d), k) * d ** -0.5
        hidden = torch.arange(total, device="cuda") > torch.arange(past[0], total, device="cuda")[:, None]
        p = torch.softmax(s.masked_fill(hidden[:, None, None], -torch.inf), dim=-1)
        want = torch.einsum("tkgj,jkd->tkgd", p, v)
        # p's two codes (2^-8 and a sixteenth of that for their floor in a tile), the result's rounding
        slack = 2.0 ** -8 * 1.1 * torch.einsum("tkgj,jkd->tkgd", p, v.abs()) + 2.0 ** -8 * want.abs() + 2.0 ** -12 * v.abs().max()
        assert ((out - want).abs() <= slack).all()


def test_long_portions_in_several_launches(monkeypatch):
    """Scratch for one long request at a time: the bits of a launch over all of them."""
    rng = np.random.default_rng(14)
    batch = Batch(rng, [150, 1, 200, 0, 7, 140], [30, 300, 0, 5, 60, 500], 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, 64)
    x = torch.randn((batch.tokens, 8 * 64), device="cuda").to(torch.bfloat16)
    call = lambda: ops.attention_q8(x, pages, *batch.args(), 8, 2, 64, 0, 0.125)  # noqa: E731
    together = call()
    monkeypatch.setattr(ops, "Q8_WIDE_BYTES", 1)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    apart = call()
    taken = torch.cuda.max_memory_allocated() - before
    ops.take_device_errors()
    assert torch.equal(together, apart)
    one = 2 * (640 // 128 + 1) * 128 * 64 * 4          # kv heads, 640 keys and a tile, keys and values in bfloat16
    assert taken <= one + apart.nbytes + 2 ** 21       # (the splits of the few rows and the batch's numbers: far below 2 MB)


def test_a_long_portion_beside_a_single_token_takes_no_place_for_splits():
    """Many splits of one row's keys: their results are counted in rows of such requests, not in rows of the batch."""
    rng = np.random.default_rng(15)
    n_q, n_kv, d, page = 8, 2, 64, 16
    batch = Batch(rng, [1, 1500], [20000, 0], page)
    pages = random_pages(ops, rng, batch.num_pages, n_kv, page, d)
    args = batch.args()
    splits = ops.q8_few_splits(n_kv * 1, 16, 20001)
    assert splits > 16
    x = torch.randn((batch.tokens, n_q * d), device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = ops.attention_q8(x, pages, *args, n_q, n_kv, d, 0, d ** -0.5)
    taken = torch.cuda.max_memory_allocated() - before
    ops.take_device_errors()
    wide = n_kv * (20096 // 128 + 1) * 128 * d * 4
    # and where the portion's keys are split too, each of its tiles of 128 rows leaves (d + 2) 32-bit numbers a row and split
    tiles = n_kv * -(-1500 * (n_q // n_kv) // 128)
    parts = ops.q8_rows_splits(tiles, 20001)
    shares = tiles * parts * 128 * (d + 2) * 4 if parts > 1 else 0
    assert taken <= out.nbytes + wide + shares + 2 * n_q * splits * (d + 2) * 4 + 2 ** 20
    alone = ops.attention_q8(x[:1], pages, args[0][:2].contiguous(), args[1][:1], args[2][:1], args[3][:1], 1, [1], 20001, n_q, n_kv, d, 0, d ** -0.5)
    assert torch.equal(out[:1], alone)


@pytest.mark.parametrize("told, rows, keys, most", [
    (1, 5, 5, 5), (5, 9, 9, 9),                      # more rows than the host's count, and than q has
    (200, 300, 300, 300), (200, 200, 900, 300),      # portions: more rows, and more keys than `max_kv_len`
])
def test_requests_beyond_what_the_host_said_are_reported(told, rows, keys, most):
    rng = np.random.default_rng(16)
    batch = Batch(rng, [rows], [keys - rows], 16)
    pages = random_pages(ops, rng, batch.num_pages, 2, 16, 64)
    q_start, kv_len, pos0, table, *_ = batch.args()
    q = torch.ones((told, 4 * 64), dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 7.0)
    ops.attention_q8(q, pages, q_start, kv_len, pos0, table, 1, [told], most, 4, 2, 64, 0, 0.125, out=out)
    with pytest.raises(ops.KernelError, match="row"):
        ops.take_device_errors()
    assert (out == 7.0).all()


@pytest.mark.parametrize("splits", [2, 3, 7])
@pytest.mark.parametrize("rows, past, window", [([150], [700], 0), ([150, 1, 140, 0, 300], [30, 9, 1500, 0, 0], 0), ([200], [900], 130), ([140, 160], [0, 500], -100)])
@pytest.mark.parametrize("d", [64, 128])
def test_keys_of_many_rows_in_splits(monkeypatch, splits, rows, past, window, d):
    """More splits than some rows have tiles, and rows of which a split sees nothing; long rows also one request at a time."""
    monkeypatch.setattr(ops, "q8_rows_splits", lambda ctas, keys: splits)
    check(np.random.default_rng(17), rows, past, 4, 2, d, 16, window=window)
    monkeypatch.setattr(ops, "Q8_WIDE_BYTES", 1)
    check(np.random.default_rng(17), rows, past, 4, 2, d, 16, window=window)


@pytest.mark.parametrize("what", ["k", "v"])
def test_rows_that_are_no_numbers_in_splits(monkeypatch, what):
    monkeypatch.setattr(ops, "q8_rows_splits", lambda ctas, keys: 3)
    got, _ = check(np.random.default_rng(18), [150], [400], 4, 2, 64, 16, change=lambda pages, batch: poison(pages, batch, 0, 480, what))
    assert np.isnan(got).any() and not np.isnan(got).all()


def test_rows_that_see_nothing_are_zero_in_splits(monkeypatch):
    monkeypatch.setattr(ops, "q8_rows_splits", lambda ctas, keys: 2)
    got, _ = check(np.random.default_rng(19), [150, 140], [10, 20], 4, 2, 64, 16, lengths=[0, 160])
    assert (got[:150] == 0).all()


def test_a_portion_behind_a_long_context_is_split():
    assert ops.q8_rows_splits(2 * 4, 6000) > 1
    check(np.random.default_rng(20), [140], [5860], 6, 2, 64, 64)
