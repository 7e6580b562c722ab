"""How attention of few rows over the 8-bit cache shares keys out: rules on the host, no GPU."""
import pytest

from llm_inference_lab_b200.kernels import ops

# a B200's clusters of 1 .. 8 CTAs, a CTA a multiprocessor
ALONE = [0, 148, 74, 45, 33, 26, 22, 15, 15]


def places(monkeypatch, width):
    class Library:
        @staticmethod
        def lab_attention_q8_few_clusters(width, size):
            return ALONE[size]
    monkeypatch.setattr(ops, "lib", lambda *_: Library)
    monkeypatch.setattr(ops, "_q8_places", {})
    return ops._q8_few_places(0, 128, width)


def test_clusters_that_find_room(monkeypatch):
    assert places(monkeypatch, 48)[1:] == ALONE[1:]
    assert places(monkeypatch, 32)[8] == 33 and places(monkeypatch, 32)[6] == 44      # four multiprocessors hold eight CTAs
    assert places(monkeypatch, 16)[8] == 45 and places(monkeypatch, 16)[1] == 444


@pytest.mark.parametrize("ctas, width, keys, splits", [
    (12, 48, 2000, 8), (16, 48, 2000, 6), (24, 48, 2000, 5), (32, 48, 6000, 4), (36, 48, 6000, 3), (100, 48, 6000, 1),      # drafts of 7B heads
    (32, 32, 1700, 8), (34, 32, 6000, 6), (48, 32, 6000, 5), (32, 16, 4096, 8), (52, 16, 6000, 6), (72, 16, 6000, 5), (128, 16, 4096, 3),
    (4, 16, 2000, 8), (4, 16, 4096, 32), (4, 16, 100000, 111), (16, 16, 4096, 8), (16, 16, 8000, 27), (16, 16, 100, 1),
    (4, 48, 2000, 8), (4, 48, 6000, 37), (8, 48, 8000, 8), (8, 48, 12000, 18), (2, 32, 4096, 32), (16, 32, 8000, 8), (16, 32, 40000, 18),
    (16, 48, 40000, 9), (1000, 16, 40000, 1), (0, 16, 0, 1)])
def test_splits_by_what_finds_room_and_pays(monkeypatch, ctas, width, keys, splits):
    monkeypatch.setattr(ops, "sm_count", lambda: 148)
    assert ops.q8_few_splits(ctas, width, keys, places(monkeypatch, width)) == splits


@pytest.mark.parametrize("head_dim, requests, keys, rows", [
    (128, 1, 300, 128), (128, 1, 60000, 128), (128, 2, 300, 96), (128, 40, 16000, 96), (64, 1, 300, 48), (64, 1, 2000, 96), (64, 2, 60000, 48)])
def test_rows_that_a_request_alone_may_have(head_dim, requests, keys, rows):
    assert ops.q8_few_rows(head_dim, requests, keys) == rows
