"""Paged caches whose K, V and scales lie in orders and strides of their own, codes and scales beyond 32-bit offsets, and steps without a token."""
import ctypes

import numpy as np
import pytest

import tessera_oracle as orc
from test_gpu_paged import FORMATS, Cache, from_bits, hold, i64, make, reference, to_bits

pytestmark = pytest.mark.gpu


def placed(lane, a, order, gap):
    """A [pages, page, heads, ...] array on the device with its first three dimensions in `order` (outermost first) and `gap`
    rows left out behind each innermost run.  Returns the buffer, its element strides and a function that reads it back."""
    width = int(np.prod(a.shape[3:], dtype=np.int64))
    dims = [a.shape[i] for i in order]
    strides = [0, 0, 0]
    strides[order[2]] = width
    strides[order[1]] = width * (dims[2] + gap)
    strides[order[0]] = strides[order[1]] * dims[1]
    whole = np.full((dims[0], dims[1], dims[2] + gap, width), 0x7b, a.dtype)
    whole[:, :, :dims[2]] = a.reshape(a.shape[:3] + (width,)).transpose(order + (3,))
    buf = lane.DeviceBuffer.from_host(whole)

    def back():
        got = buf.download(whole.shape, a.dtype)
        assert np.all(got[:, :, dims[2]:] == whole[:, :, dims[2]:])          # nothing is written between the rows
        return got[:, :, :dims[2]].transpose(tuple(np.argsort(order)) + (3,)).reshape(a.shape)
    return buf, strides, back


def device(lane, c, k_order, v_order, s_order, gap=0):
    pages, page, heads, D = c.dims
    k, v = (placed(lane, a, o, gap) for a, o in ((c.k, k_order), (c.v, v_order)))
    ks, vs = (placed(lane, a, s_order, gap) for a in (c.ks, c.vs))
    scaled = c.fmt != "storage"
    handle = lane.KVCache(k=k[0].ptr, v=v[0].ptr, k_scale=ks[0].ptr if scaled else None, v_scale=vs[0].ptr if scaled else None, k_strides=tuple(k[1]),
                          v_strides=tuple(v[1]), scale_strides=tuple(ks[1]) if scaled else (0, 0, 0), num_pages=pages, page_size=page, num_heads=heads,
                          head_dim=D, format=FORMATS.index(c.fmt))
    return handle, (k, v, ks, vs)


ORDERS = [((0, 1, 2), (0, 2, 1), (2, 0, 1), 0), ((2, 0, 1), (0, 1, 2), (0, 1, 2), 3), ((1, 0, 2), (2, 1, 0), (1, 2, 0), 1), ((0, 2, 1), (0, 2, 1), (0, 1, 2), 2)]


@pytest.mark.parametrize("fmt,dtype", [("storage", "bf16"), ("storage", "f16"), ("i8", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("orders", ORDERS, ids=str)
@pytest.mark.parametrize("new,kv,D", [([1, 1, 3], [300, 2000, 9], 64), ([120, 40], [300, 900], 128), ([1, 50], [70, 50], 80)])
def test_orders_of_their_own(lane, fmt, dtype, orders, new, kv, D):
    """Attention, and what a write leaves and a read finds, with K, V and the scales each in another order, rows and scales with gaps."""
    lib, hq, hkv = lane.load(), 4, 2
    c, table, slots, q = make(lane, new, kv, hq=hq, hkv=hkv, D=D, page=16, fmt=fmt, dtype=dtype, seed=41)
    handle, parts = device(lane, c, *orders)
    total = sum(new)
    bufs = [lane.DeviceBuffer.from_host(a) for a in (q, table, np.concatenate([[0], np.cumsum(new)]).astype(np.int32), np.asarray(kv, np.int32))]
    O, L = lane.DeviceBuffer(total * hq * D * 4), lane.DeviceBuffer(total * hq * 4)
    lane.check(getattr(lib, f"tessera_gfx950_paged_attention_{dtype}_dev")(
        ctypes.byref(handle), bufs[0].ptr, O.ptr, L.ptr, i64((hq * D, D) * 2), bufs[1].ptr, table.shape[1], bufs[2].ptr, bufs[3].ptr, len(kv), hq, total, max(new),
        max(kv), D ** -0.5, 1, 0, 0.0, 0, None), "paged_attention")
    lane.synchronize()
    hold(O.download((total, hq, D), np.float32), L.download((total, hq), np.float32), reference(c, slots, q, new, kv, hq), c, kv=max(kv))
    rng = np.random.default_rng(6)
    T = 37
    to = rng.permutation(c.dims[0] * 16)[:T].astype(np.int64)
    k, v = (rng.standard_normal((T, hkv, D)).astype(np.float32) for _ in range(2))
    d = [lane.DeviceBuffer.from_host(a) for a in (to_bits(k, dtype), to_bits(v, dtype), to)]
    back = [lane.DeviceBuffer(T * hkv * D * 2) for _ in range(2)]
    st = i64((hkv * D, D) * 2)
    lane.check(getattr(lib, f"tessera_gfx950_kv_cache_write_{dtype}_dev")(ctypes.byref(handle), d[0].ptr, d[1].ptr, st, d[2].ptr, T, None), "write")
    lane.check(getattr(lib, f"tessera_gfx950_kv_cache_read_{dtype}_dev")(ctypes.byref(handle), d[2].ptr, back[0].ptr, back[1].ptr, st, T, None), "read")
    lane.synchronize()
    c.put(to, k, v)
    table8 = orc.e4m3_decode_table()
    for i, host in enumerate((c.k, c.v, c.ks, c.vs)):
        if i >= 2 and fmt == "storage":
            continue
        got = parts[i][2]()
        if fmt == "e4m3" and i < 2:                            # (a negative zero is a zero)
            got, host = table8[got], table8[host]
        assert np.array_equal(got, host, equal_nan=True)
    for buf, want in zip(back, c.values(to)):
        got = from_bits(buf.download((T, hkv, D), np.uint16), dtype)
        assert np.all(np.abs(got - want) <= np.abs(want) * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -10) + 2.0 ** -24)


@pytest.mark.parametrize("fmt", ("i8", "e4m3"))
def test_codes_and_scales_past_32_bits(lane, fmt):
    """Codes more than 4 GiB and scales more than 2^31 elements (8 GiB) into their arrays, by the strides of the pages."""
    lib, heads, D, page, pages = lane.load(), 2, 64, 16, 4
    k_page, s_page = (1 << 31) - 4096, 1 << 30                  # bytes; elements
    k, v = lane.DeviceBuffer(3 * k_page + page * heads * D), lane.DeviceBuffer(3 * k_page + page * heads * D)
    ks, vs = lane.DeviceBuffer(3 * s_page * 4 + page * heads * 4), lane.DeviceBuffer(3 * s_page * 4 + page * heads * 4)
    handle = lane.KVCache(k=k.ptr, v=v.ptr, k_scale=ks.ptr, v_scale=vs.ptr, k_strides=(k_page, heads * D, D), v_strides=(k_page, heads * D, D),
                          scale_strides=(s_page, heads, 1), num_pages=pages, page_size=page, num_heads=heads, head_dim=D, format=FORMATS.index(fmt))
    rng = np.random.default_rng(0)
    new, kv, hq = [1, 20], [30, 32], 4
    table = np.asarray([[3, 2], [1, 0]], np.int32)
    small = Cache(lane, pages, page, heads, D, fmt, "bf16")
    q = to_bits(rng.standard_normal((21, hq, D)), "bf16")
    slots, strides = [], i64((heads * D, D) * 2)
    for b in range(2):
        j = np.arange(kv[b])
        slots.append(table[b, j // page].astype(np.int64) * page + j % page)
        kk, vv = (rng.standard_normal((kv[b], heads, D)).astype(np.float32) for _ in range(2))
        small.put(slots[b], kk, vv)
        bufs = [lane.DeviceBuffer.from_host(a) for a in (to_bits(kk, "bf16"), to_bits(vv, "bf16"), slots[b])]
        lane.check(lib.tessera_gfx950_kv_cache_write_bf16_dev(ctypes.byref(handle), bufs[0].ptr, bufs[1].ptr, strides, bufs[2].ptr, kv[b], None), "write")
        back = lane.DeviceBuffer(kv[b] * heads * D * 2), lane.DeviceBuffer(kv[b] * heads * D * 2)
        lane.check(lib.tessera_gfx950_kv_cache_read_bf16_dev(ctypes.byref(handle), bufs[2].ptr, back[0].ptr, back[1].ptr, strides, kv[b], None), "read")
        lane.synchronize()
        for buf, want in zip(back, small.values(slots[b])):
            got = from_bits(buf.download((kv[b], heads, D), np.uint16), "bf16")
            assert np.all(np.abs(got - want) <= np.abs(want) * 2.0 ** -8)
    bufs = [lane.DeviceBuffer.from_host(a) for a in (q, table, np.asarray([0, 1, 21], np.int32), np.asarray(kv, np.int32))]
    for rows, max_q in ((slice(0, 21), 20), (slice(0, 1), 1)):  # tiles, few rows
        B, T = (2, 21) if max_q > 1 else (1, 1)
        for group in (hq, heads * 64):
            qs = q if group == hq else to_bits(rng.standard_normal((21, group, D)), "bf16")
            dq = lane.DeviceBuffer.from_host(qs)
            O, L = lane.DeviceBuffer(T * group * D * 4), lane.DeviceBuffer(T * group * 4)
            lane.check(lib.tessera_gfx950_paged_attention_bf16_dev(
                ctypes.byref(handle), dq.ptr, O.ptr, L.ptr, i64((group * D, D) * 2), bufs[1].ptr, 2, bufs[2].ptr, bufs[3].ptr, B, group, T, max_q, 32, D ** -0.5, 1, 0,
                0.0, 0, None), "paged_attention")
            lane.synchronize()
            ref = reference(small, slots[:B], qs[rows], new[:B], kv[:B], group)
            hold(O.download((T, group, D), np.float32), L.download((T, group), np.float32), ref, small)


@pytest.mark.parametrize("quant", (None, "e4m3"))
def test_steps_without_a_token(lane, quant):
    """No sequence, and sequences that get nothing: arrays of no element, results of none, and the cache as it was."""
    from tessera_amd import paged
    from tessera_amd.resident import DeviceArray
    cache = paged.PagedKVCache(4, 16, 2, 64, dtype="f16", quant=quant)
    pages = paged.SequencePages(cache)
    for step in ({}, {"a": 0}, {"a": 3}, {"a": 0, "b": 0}):
        batch = pages.extend(step)
        T = sum(step.values())
        k = DeviceArray.from_host(np.ones((T, 2, 64), np.float16))
        cache.write(k, k, batch.slots)
        o, lse = paged.paged_attention(DeviceArray.from_host(np.ones((T, 4, 64), np.float16)), cache, batch, return_lse=True, out="f32")
        assert o.to_host().shape == (T, 4, 64) and lse.to_host().shape == (T, 4)
        assert np.all(np.abs(o.to_host() - 1) <= 2.0 ** -3)
        got = cache.read(DeviceArray.from_host(pages.slots("a")))[0].to_host()
        assert got.shape == (pages.length("a"), 2, 64) and np.all(np.abs(got - 1) <= 2.0 ** -3)


def test_more_tokens_than_one_launch_has_rows(lane):
    """A buffer of 2^24 and more rows of Q, of which the sequence has a few: the merge of its shares is launched over all of them."""
    lib, D, kv, total = lane.load(), 16, 9000, (1 << 24) + 40
    c, table, slots, q = make(lane, [2], [kv], hq=1, hkv=1, D=D, page=64, fmt="storage", dtype="bf16", seed=43)
    handle = c.upload()
    Q, O = lane.DeviceBuffer(total * D * 2), lane.DeviceBuffer(total * D * 2)
    for first in (0, total - 2):                                # its rows at the buffer's start, and at its end
        lane.check(lib.tessera_gfx950_memcpy_h2d(Q.ptr + first * D * 2, q.ctypes.data, q.nbytes), "memcpy_h2d")
        bufs = [lane.DeviceBuffer.from_host(a) for a in (table, np.asarray([first, first + 2], np.int32), np.asarray([kv], np.int32))]
        lane.check(lib.tessera_gfx950_paged_attention_bf16_dev(
            ctypes.byref(handle), Q.ptr, O.ptr, None, i64((D, D) * 2), bufs[0].ptr, table.shape[1], bufs[1].ptr, bufs[2].ptr, 1, 1, total, 2, kv, D ** -0.5, 1, 0, 0.0, 1,
            None), "paged_attention")
        lane.synchronize()
        got = np.empty((2, 1, D), np.uint16)
        lane.check(lib.tessera_gfx950_memcpy_d2h(got.ctypes.data, O.ptr + first * D * 2, got.nbytes), "memcpy_d2h")
        ref = reference(c, slots, q, [2], [kv], 1)
        hold(from_bits(got, "bf16"), ref[1].astype(np.float32), ref, c, 1, kv=kv)
