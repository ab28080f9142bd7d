"""Paged attention recorded into graphs: one eager call with arguments as large makes room for every smaller one, whichever kernels,
splits and merges the two take."""
import ctypes

import numpy as np
import pytest

from test_gpu_paged import attend, hold, i64, make, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    L = ctypes.CDLL("libamdhip64.so", mode=ctypes.RTLD_LOCAL)
    p, pp = ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)
    for name, args in {"hipStreamCreate": [pp], "hipStreamSynchronize": [p], "hipStreamDestroy": [p], "hipStreamBeginCapture": [p, ctypes.c_int],
                       "hipStreamEndCapture": [p, pp], "hipGraphInstantiate": [pp, p, p, p, ctypes.c_size_t], "hipGraphLaunch": [p, p],
                       "hipGraphExecDestroy": [p], "hipGraphDestroy": [p]}.items():
        getattr(L, name).argtypes = args
    return L


class Call:
    """One attention call over a cache of its own."""

    def __init__(self, lane, new, kv, hq, hkv, D, fmt="storage", dtype="bf16", window=0, seed=0):
        self.lane, self.new, self.kv, self.hq, self.window = lane, new, kv, hq, window
        self.c, self.table, self.slots, self.q = make(lane, new, kv, hq=hq, hkv=hkv, D=D, page=16, fmt=fmt, dtype=dtype, seed=seed)
        self.handle = self.c.upload()
        self.pages = self.c.bufs                            # (an upload for another call replaces the cache's own reference)
        self.bufs = [lane.DeviceBuffer.from_host(a) for a in (self.q, self.table, np.concatenate([[0], np.cumsum(new)]).astype(np.int32),
                                                              np.asarray(kv, np.int32))]
        total = sum(new)
        self.O, self.L = lane.DeviceBuffer(total * hq * D * 4), lane.DeviceBuffer(total * hq * 4)

    def __call__(self, s):
        D, b, total = self.c.dims[3], self.bufs, sum(self.new)
        fn = getattr(self.lane.load(), f"tessera_gfx950_paged_attention_{self.c.dtype}_dev")
        return fn(ctypes.byref(self.handle), b[0].ptr, self.O.ptr, self.L.ptr, i64((self.hq * D, D) * 2), b[1].ptr, self.table.shape[1], b[2].ptr, b[3].ptr,
                  len(self.kv), self.hq, total, max(self.new), max(self.kv), D ** -0.5, 1, self.window, 0.0, 0, s)

    def clear(self):
        self.O.zero(), self.L.zero()

    def results(self):
        D, total = self.c.dims[3], sum(self.new)
        return self.O.download((total, self.hq, D), np.float32), self.L.download((total, self.hq), np.float32)

    def eager_results(self):
        return attend(self.lane, self.c, self.table, self.q, self.new, self.kv, self.hq, window=self.window)


# what the stream has run eagerly, and what is recorded behind it: (new, kv, window) of the same heads and head dimension
PAIRS = {
    "a batch of 64, then one": (8, 8, 128, [1] * 64, [512] * 64, [([1], [512], 0), ([1] * 3, [512, 7, 400], 0), ([1], [40], 0)]),
    "a merge of many shares, then of few": (8, 1, 128, [1], [131072], [([1], [1000], 0), ([1], [3000], 0), ([1], [100000], 0)]),
    "an uncut chunk, then single tokens": (8, 2, 128, [512], [512], [([1], [512], 0), ([3], [500], 0), ([40], [512], 0), ([130], [512], 0)]),
    "chunks, then fewer and shorter ones": (8, 2, 64, [300, 300, 1], [3000, 700, 1], [([300, 1], [3000, 50], 0), ([70], [3000], 0), ([299], [2999], 0)]),
    "a chunk, then mixtures": (8, 2, 128, [200, 200, 200, 200], [4000] * 4, [([200, 1, 1, 1], [900, 4000, 4000, 1], 0), ([1, 1, 4], [4000, 3, 2000], 0)]),
    "a window, then none of the keys cut": (4, 2, 64, [1] * 8, [4000] * 8, [([1] * 5, [3000] * 5, 100), ([1] * 2, [4000, 4000], 2000)]),
    "a speculative step, then single tokens": (8, 2, 64, [8, 8], [6000, 6000], [([1, 8], [6000, 9], 0), ([1], [6000], 0), ([5, 2], [700, 600], 0)]),
}


@pytest.mark.parametrize("mode", (0, 2), ids=("global", "relaxed"))
@pytest.mark.parametrize("fmt", ("storage", "e4m3"))
@pytest.mark.parametrize("name", PAIRS)
def test_smaller_calls_record_behind_a_larger_one(lane, hip, name, fmt, mode):
    hq, hkv, D, new, kv, after = PAIRS[name]
    large = Call(lane, new, kv, hq, hkv, D, fmt)
    calls = [Call(lane, n, k, hq, hkv, D, fmt, window=w, seed=i + 1) for i, (n, k, w) in enumerate(after)]
    want = [c.eager_results() for c in calls]
    p = ctypes.c_void_p
    s, graphs, exes = p(), [], []
    assert hip.hipStreamCreate(ctypes.byref(s)) == 0
    try:
        lane.check(large(s), "paged_attention")
        assert hip.hipStreamSynchronize(s) == 0
        for call in calls:
            graph, exe = p(), p()
            assert hip.hipStreamBeginCapture(s, mode) == 0
            rc = call(s)
            assert hip.hipStreamEndCapture(s, ctypes.byref(graph)) == 0 and graph.value
            graphs.append(graph)
            assert rc == lane.OK
            assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
            exes.append(exe)
        for _ in range(3):
            for call, exe, ref in zip(calls, exes, want):
                call.clear()
                lane.check(large(s), "paged_attention")    # eager work between the replays
                assert hip.hipStreamSynchronize(s) == 0
                assert hip.hipGraphLaunch(exe, s) == 0
                assert hip.hipStreamSynchronize(s) == 0
                for got, w in zip(call.results(), ref):
                    assert np.array_equal(got, w)
    finally:
        for exe in exes:
            hip.hipGraphExecDestroy(exe)
        for graph in graphs:
            hip.hipGraphDestroy(graph)
        hip.hipStreamSynchronize(s)
        lane.load().tessera_gfx950_stream_release(s)
        hip.hipStreamDestroy(s)


@pytest.mark.parametrize("window", (0, 700))
def test_a_split_walk_records_without_a_workspace(lane, hip, window):
    """A chunk whose walk an eager call splits, first met inside a capture: recorded whole, and right."""
    call = Call(lane, [100], [4000], 8, 2, 64, "i8", "f16", window=window)
    p = ctypes.c_void_p
    s, graph, exe = p(), p(), p()
    assert hip.hipStreamCreate(ctypes.byref(s)) == 0
    try:
        lane.synchronize()
        assert hip.hipStreamBeginCapture(s, 0) == 0
        rc = call(s)
        assert hip.hipStreamEndCapture(s, ctypes.byref(graph)) == 0 and graph.value
        assert rc == lane.OK
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        ref = reference(call.c, call.slots, call.q, call.new, call.kv, call.hq, window=window)
        first = None
        for _ in range(3):
            call.clear()
            lane.synchronize()
            assert hip.hipGraphLaunch(exe, s) == 0
            assert hip.hipStreamSynchronize(s) == 0
            o, lse = call.results()
            hold(o, lse, ref, call.c, kv=4000)
            assert first is None or np.array_equal(o, first)
            first = o
    finally:
        if exe.value:
            hip.hipGraphExecDestroy(exe)
        if graph.value:
            hip.hipGraphDestroy(graph)
        hip.hipStreamSynchronize(s)
        lane.load().tessera_gfx950_stream_release(s)
        hip.hipStreamDestroy(s)
