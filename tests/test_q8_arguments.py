"""What the operators of the 8-bit cache and of drafted tokens refuse, and their choices of launches: no GPU needed."""
import numpy as np
import pytest
import torch

from llm_inference_lab_b200.kernels import ops
from q8_helpers import decode, encode

KERNEL_ERROR = ops.KernelError


def pages(n_kv=2, page=16, d=64, count=4):
    return ops.quant_pages(count, n_kv, page, d, "cpu")


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def store(**change):
    a = dict(qkv=torch.zeros((3, 10 * 64), dtype=torch.bfloat16), table=torch.zeros((3, 32, 2)), rotary_dim=64, slots=ints(0, 1, -1),
             pages=pages(), n_q=6, n_kv=2, head_dim=64)
    a.update(change)
    return ops.rope_kv_store_q8(**a)


@pytest.mark.parametrize("change, says", [
    (dict(), "must be CUDA tensors"),
    (dict(qkv=torch.zeros((3, 9 * 64), dtype=torch.bfloat16)), "rows of 640"),
    (dict(qkv=torch.zeros((3, 10 * 64), dtype=torch.float16)), "unsupported storage type"),
    (dict(qkv=torch.zeros((2, 3, 10 * 64), dtype=torch.bfloat16)), "partial products are contiguous float32"),
    (dict(qkv=torch.zeros((640,), dtype=torch.bfloat16)), "rows or partial products"),
    (dict(bias=torch.zeros((640,), dtype=torch.bfloat16)), "goes with partial products"),
    (dict(table=torch.zeros((2, 32, 2))), "a table"),
    (dict(table=None), "a table"),
    (dict(rotary_dim=66), "rotary_dim"),
    (dict(rotary_dim=31), "rotary_dim"),
    (dict(slots=ints(0, 1)), "slots"),
    (dict(slots=torch.zeros((3,), dtype=torch.int64)), "slots"),
    (dict(pages=pages(d=32)), "are not"),
    (dict(pages=pages()._replace(k=torch.zeros((4, 2, 16, 64), dtype=torch.uint8))), "float8_e4m3fn"),
    (dict(pages=pages()._replace(v_scale=torch.zeros((4, 2, 8), dtype=torch.uint8))), "uint8"),
])
def test_store_refuses(change, says):
    with pytest.raises(KERNEL_ERROR, match=says):
        store(**change)


@pytest.mark.parametrize("change, says", [
    (dict(), "must be CUDA tensors"),
    (dict(slots=ints()[:, None]), "one row of slots"),
    (dict(slots=torch.zeros((3,))), "slots"),
    (dict(dtype=torch.float16), "unsupported storage type"),
    (dict(pages=pages()._replace(k=torch.zeros((4, 2), dtype=torch.float8_e4m3fn))), "are not"),
])
def test_load_refuses(change, says):
    a = dict(pages=pages(), slots=ints(3, 1), dtype=torch.bfloat16)
    a.update(change)
    with pytest.raises(KERNEL_ERROR, match=says):
        ops.kv_load_q8(**a)


@pytest.mark.parametrize("change, says", [
    (dict(), "must be CUDA tensors"),
    (dict(q=torch.zeros((3, 6 * 32), dtype=torch.bfloat16)), "q of 384"),
    (dict(q=torch.zeros((3, 6 * 64), dtype=torch.float16)), "unsupported storage type"),
    (dict(n_q=5, q=torch.zeros((3, 5 * 64), dtype=torch.bfloat16)), "over 2 kv heads"),
    (dict(q_start=ints(0, 2)), "q_start"),
    (dict(kv_len=torch.zeros((2,))), "kv_len"),
    (dict(pos0=ints(0)), "pos0"),
    (dict(block_table=ints(0, 1)), "block table"),
    (dict(block_table=torch.zeros((1, 3), dtype=torch.int32)), "block table"),
    (dict(q_lens=[3]), "row counts"),
    (dict(scale=0.0), "scale"),
    (dict(out=torch.zeros((3, 6 * 64))), "out as q"),
    (dict(pages=pages(n_kv=3)), "are not"),
])
def test_attention_refuses(change, says):
    a = dict(q=torch.zeros((3, 6 * 64), dtype=torch.bfloat16), pages=pages(), q_start=ints(0, 2, 3), kv_len=ints(2, 1), pos0=ints(0, 0),
             block_table=torch.zeros((2, 3), dtype=torch.int32), n_requests=2, q_lens=[2, 1], max_kv_len=2, n_q=6, n_kv=2, head_dim=64,
             window=0, scale=0.125)
    a.update(change)
    with pytest.raises(KERNEL_ERROR, match=says):
        ops.attention_q8(**a)


@pytest.mark.parametrize("change, says", [
    (dict(), "must be CUDA tensors"),
    (dict(logits=torch.zeros((5, 11), dtype=torch.bfloat16)), "logits are float32"),
    (dict(logits=torch.zeros((11, 5)).T), "logits are float32"),
    (dict(drafts=ints(1, 2)), "drafts"),
    (dict(starts=torch.zeros((3,), dtype=torch.int64)), "starts"),
    (dict(draft_probs=torch.zeros((4, 11))), "draft_probs"),
    (dict(temperature=torch.ones((2,))), "needs seeds and positions"),
    (dict(temperature=torch.ones((1,)), seeds=ints(1, 2), positions=ints(1, 2)), "temperature per request"),
    (dict(temperature=torch.ones((2,)), seeds=ints(1), positions=ints(1, 2)), "seeds"),
    (dict(logits=torch.zeros((65536, 1)), drafts=torch.zeros((65536,), dtype=torch.int32)), "65535"),
])
def test_verify_refuses(change, says):
    a = dict(logits=torch.zeros((5, 11)), drafts=ints(1, 2, 3, 4, 5), starts=ints(0, 2, 5))
    a.update(change)
    with pytest.raises(KERNEL_ERROR, match=says):
        ops.verify_drafts(**a)


def test_codes_of_the_yardstick():
    """Numbers that codes stand for come back; halfway between two codes goes to the even one; borders of the scale."""
    assert decode(*encode(np.array([[448.0, -448.0, 2.0 ** -9, 0.0]]))).tolist() == [[448.0, -448.0, 2.0 ** -9, 0.0]]
    assert encode(np.array([448.0]))[1] == 127 and encode(np.array([448.5]))[1] == 128 and encode(np.array([224.0]))[1] == 126
    assert encode(np.zeros(3))[1] == 127 and encode(np.array([1.0, np.inf]))[1] == 255 and encode(np.array([1e-40]))[1] == 17
    codes = encode(np.array([448.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10]))[0]
    assert decode(codes[None], np.array([127]))[0].tolist() == [448.0, 16.0, 20.0, 0.0, 2.0 ** -8]
    there = torch.arange(256, dtype=torch.int16).to(torch.uint8)
    value = there.view(torch.float8_e4m3fn).double().numpy()
    keep = ~np.isnan(value)
    assert (decode(there.numpy()[:, None], np.full(256, 127))[keep, 0] == value[keep]).all() and keep.sum() == 254


@pytest.mark.parametrize("ctas, keys", [(1, 1), (1, 128), (1, 100000), (16, 530), (128, 4096), (5000, 4096), (37, 129)])
def test_splits_leave_no_cta_without_room_or_keys(ctas, keys):
    for width, held in ((16, 3), (32, 2), (48, 1)):      # CTAs that a multiprocessor holds
        splits = ops.q8_few_splits(ctas, width, keys)
        assert 1 <= splits <= -(-keys // 128)
        assert splits == 1 or splits * ctas <= held * ops.sm_count()


@pytest.mark.parametrize("rows", [1, 7, 16, 17, 32, 33, 48, 49, 1000])
def test_widths_are_built(rows):
    assert ops.q8_few_width(rows) in (16, 32, 48) and (rows > 48 or ops.q8_few_width(rows) >= rows)


@pytest.mark.parametrize("change, says", [
    (dict(q_lens=[3, 1]), "row counts within the 3 rows"),
    (dict(q_lens=[4, -1]), "row counts within the 3 rows"),
    (dict(n_q=0, q=torch.zeros((3, 0), dtype=torch.bfloat16)), "0 query heads"),
])
def test_attention_refuses_rows_and_heads_that_are_not_there(change, says):
    a = dict(q=torch.zeros((3, 6 * 64), dtype=torch.bfloat16), pages=pages(), q_start=ints(0, 2, 3), kv_len=ints(2, 1), pos0=ints(0, 0),
             block_table=torch.zeros((2, 3), dtype=torch.int32), n_requests=2, q_lens=[2, 1], max_kv_len=2, n_q=6, n_kv=2, head_dim=64,
             window=0, scale=0.125)
    a.update(change)
    with pytest.raises(KERNEL_ERROR, match=says):
        ops.attention_q8(**a)


@pytest.mark.parametrize("q_lens", [[200], [1, 200, 1], [200, 300, 1, 0, 129, 500, 2], [129] * 7])
@pytest.mark.parametrize("at_once", [1, 2, 3])
def test_runs_of_long_requests_cover_each_request_once(q_lens, at_once):
    runs = ops._spans_of_many(q_lens, 128, at_once)
    assert [b for first, end, _ in runs for b in range(first, end)] == list(range(len(q_lens)))
    for first, end, held in runs:
        assert held == sum(n > 128 for n in q_lens[first:end]) and 1 <= held <= at_once


@pytest.mark.parametrize("head_dim, taken", [(256, True), (272, False)])
def test_engine_refuses_heads_that_no_kernel_takes(head_dim, taken):
    from types import SimpleNamespace as Some

    from llm_inference_lab_b200.engine.engine import Engine
    from llm_inference_lab_b200.parts.spec import PagedKV
    model = Some(order=[Some(layer=0, cache=0)], blocks=[Some(mixer=Some(quantised_cache=True))])
    plan = Some(needs=[PagedKV(n_kv_heads=1, head_dim=head_dim)])
    check = lambda: Engine._check_quantised(Some(dtype=torch.bfloat16), model, plan)  # noqa: E731
    if taken:
        check()
    else:
        with pytest.raises(ValueError, match="heads of 272"):
            check()


@pytest.mark.parametrize("ctas, keys, splits", [(1, 1, 1), (1, 767, 2), (1, 640, 1), (4, 4100, 11), (4, 100000, 74), (68, 20000, 4), (112, 8500, 1),
                                                (56, 8500, 2), (132, 20600, 2), (149, 20600, 1), (500, 100000, 1), (0, 300, 1)])
def test_splits_of_many_rows_find_room_and_keys(monkeypatch, ctas, keys, splits):
    monkeypatch.setattr(ops, "sm_count", lambda: 148)
    assert ops.q8_rows_splits(ctas, keys) == splits
