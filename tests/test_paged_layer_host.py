"""No-GPU checks of the paged cache's Python layer and of what a cache that is written has to look like."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

from tessera_amd import lane, paged
from test_paged_host import attend, handle, read, write


class Host:
    """Stands in for a device array."""
    fail_at = None
    made = 0

    def __init__(self, a):
        self.a, self.shape, self.ndim, self.address = a, a.shape, a.ndim, 1 << 24
        self.dtype = {"int64": "i64", "int32": "i32", "float16": "f16"}[a.dtype.name]

    @classmethod
    def from_host(cls, a):
        cls.made += 1
        if cls.made == cls.fail_at:
            raise RuntimeError("malloc: device operation failed")
        return cls(np.ascontiguousarray(a))


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(paged, "DeviceArray", Host)
    monkeypatch.setattr(Host, "fail_at", None)
    monkeypatch.setattr(Host, "made", 0)
    return Host


def small(**change):
    return SimpleNamespace(**{**dict(num_pages=6, page_size=4, num_kv_heads=2, head_dim=64, dtype="f16", handle=handle()), **change})


@pytest.mark.parametrize("tokens", (2, 4))
def test_queries_and_batch_have_as_many_tokens(host, monkeypatch, tokens):
    """Rows of O behind the batch's tokens would be an earlier result's memory, rows that are not there the last sequences'."""
    monkeypatch.setattr(paged, "_result", lambda shape, dtype: pytest.fail("a result was made"))
    cache = small()
    batch = paged.SequencePages(cache).extend({"a": 2, "b": 1})
    with pytest.raises(ValueError, match="3"):
        paged.paged_attention(Host(np.zeros((tokens, 4, 64), np.float16)), cache, batch)
    with pytest.raises(ValueError, match="3"):
        paged.paged_attention_fused_qkv(Host(np.zeros((tokens, 8 * 64), np.float16)), 4, cache, batch)


def test_a_batch_without_slots_is_not_compared(host, monkeypatch):
    """A caller's own batch of fewer rows than were written (the last token of each sequence) leaves the slots out."""
    class Reached(Exception):
        pass

    def result(shape, dtype):
        raise Reached
    monkeypatch.setattr(paged, "_result", result)
    cache = small()
    step = paged.SequencePages(cache).extend({"a": 2, "b": 1})
    last = paged.PagedBatch(None, step.page_table, Host(np.asarray([0, 1, 2], np.int32)), step.kv_lens, 1, 2)
    with pytest.raises(Reached):
        paged.paged_attention(Host(np.zeros((2, 4, 64), np.float16)), cache, last)


@pytest.mark.parametrize("at", (1, 2, 3, 4))
def test_a_step_whose_arrays_cannot_be_made_takes_nothing(host, at):
    pages = paged.SequencePages(small())
    pages.extend({"a": 3})
    before = (pages.free_pages, list(pages._free), pages.slots("a").tolist(), pages.length("a"), pages.length("b"))
    host.fail_at = host.made + at
    with pytest.raises(RuntimeError):
        pages.extend({"a": 9, "b": 2, "c": 0})
    assert (pages.free_pages, list(pages._free), pages.slots("a").tolist(), pages.length("a"), pages.length("b")) == before
    assert set(pages._pages) == {"a"} and set(pages._length) == {"a"}
    batch = pages.extend({"a": 9, "b": 2})
    assert pages.length("a") == 12 and pages.length("b") == 2 and len(set(batch.slots.a.tolist())) == 11


def test_slots_are_those_of_tokens_that_are_there(host):
    """Beyond a sequence's end lie slots of its last page that hold nothing of it."""
    pages = paged.SequencePages(small())
    pages.extend({"a": 5})
    assert len(pages.slots("a")) == 5 and len(pages.slots("a", 2, 4)) == 2 and len(pages.slots("a", 5)) == 0 and len(pages.slots("nobody")) == 0
    for first, last in ((0, 6), (0, 9), (-1, None), (6, None), (3, 2), (0, -1)):
        with pytest.raises(IndexError):
            pages.slots("a", first, last)
    with pytest.raises(IndexError):
        pages.slots("nobody", 0, 1)


CODES = dict(format=1, k_scale=1 << 22, v_scale=1 << 23)


@pytest.mark.parametrize("change", [
    dict(k_strides=(64, 64, 64)), dict(v_strides=(64, 64, 64)), dict(k_strides=(2048, 64, 64)), dict(v_strides=(1024, 128, 64)),
    dict(k_strides=(64, 128, 1024)), dict(k_strides=(128, 128, 64), page_size=1, num_pages=4, num_heads=3),
    dict(**CODES, scale_strides=(1, 1, 1)), dict(**CODES, scale_strides=(16, 2, 1)), dict(**CODES, k_strides=(1024, 128, 64))], ids=str)
def test_rows_on_top_of_each_other_are_not_written(change):
    """Two slots or heads of one cache in the same memory: what a write leaves there would depend on the order of its waves."""
    assert write(handle(**change)) == lane.BAD_SHAPE


@pytest.mark.parametrize("change", [
    dict(), dict(k_strides=(2048, 64, 1024)), dict(k_strides=(128, 256, 64)), dict(v_strides=(64, 256, 128), k_strides=(4096, 256, 128)),
    dict(num_pages=1, k_strides=(0, 128, 64)), dict(num_heads=1, k_strides=(1024, 64, 0)), dict(page_size=1, k_strides=(128, 8, 64)),
    dict(**CODES), dict(**CODES, scale_strides=(1, 4, 2)), dict(**CODES, scale_strides=(64, 4, 1))], ids=str)
def test_caches_of_any_order_and_with_gaps_are_written(change):
    if lane.available():
        pytest.skip("made-up addresses: only where there is no device to use them on")
    c = handle(**change)
    assert write(c) == read(c) == attend(c, max_kv=2, max_q=2, total=2) == lane.NO_DEVICE


def test_caches_that_are_only_read_may_share_rows():
    if lane.available():
        pytest.skip("made-up addresses: only where there is no device to use them on")
    assert read(handle(k_strides=(64, 64, 64))) == attend(handle(k_strides=(64, 64, 64))) == lane.NO_DEVICE
