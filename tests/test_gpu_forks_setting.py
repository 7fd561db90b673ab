"""nm_stack_share under qg_prefix_least_saving: a step that is replayed shares by the setting of the call, as an eager one does."""
import threading

import numpy as np
import pytest

from nebula_amd import qg
from nebula_amd.qg import Device, call
from spec_oracle import F16, Batch
from test_gpu_forks_step import forked_cache
from test_gpu_spec_step import HD, HK, LAYERS, WIDTH, make_stack, stack_parts  # noqa: F401

pytestmark = pytest.mark.gpu
NEVER = 1 << 60


def test_replays_follow_the_setting(stack_parts):  # noqa: F811
    h, lib = qg.host(), qg.lib()
    cache = forked_cache(np.random.default_rng(7), [600], [0, 0, 0], typ=F16, layers=LAYERS, kv_heads=HK, page=16, dim=HD, spare=40, table_pages=50)
    batch = Batch([2, 1, 3, 1])
    n = lib.qg_kv_workspace_bytes(cache.ref)
    ws, status = Device(np.zeros(n, np.uint8)), Device(np.zeros(cache.B, np.int32))
    call("kv_reserve", cache.ref, batch.ref, status.p, ws.p, n)
    assert (status.get() == 0).all()
    h0 = np.random.default_rng(4).standard_normal((7, WIDTH)).astype(np.float32)
    stack = make_stack(stack_parts, cache, 17)
    src = Device(h0)

    def step(least, graph):
        lib.qg_prefix_least_saving(least)
        hidden = h.nm_stack_hidden(stack)
        call("copy", hidden, src.p, h0.nbytes)
        assert h.nm_stack_verify(stack, batch.ref, graph) == 0, h.nm_last_error()
        call("sync")
        assert lib.qg_prefix_least_saving(least) == least  # left as it was
        got = np.empty_like(h0)
        call("read", got.ctypes.data, hidden, got.nbytes)
        return got

    before = lib.qg_prefix_least_saving(0)
    try:
        assert h.nm_stack_share(stack, 1) == 0, h.nm_last_error()
        want = {least: step(least, 0) for least in (0, NEVER)}
        assert not np.array_equal(want[0], want[NEVER])  # the last bits say whether pages were shared
        for least in (0, NEVER, NEVER, 0, NEVER, 0, 0):
            assert np.array_equal(step(least, 1), want[least]), least
        # another thread has a setting of its own
        lib.qg_prefix_least_saving(0)
        got = []
        t = threading.Thread(target=lambda: got.append(step(NEVER, 1)))
        t.start()
        t.join()
        assert np.array_equal(got[0], want[NEVER])
        assert np.array_equal(step(0, 1), want[0])
        # not shared at all: the setting does not matter
        assert h.nm_stack_share(stack, 0) == 0
        assert np.array_equal(step(0, 1), step(NEVER, 1))
    finally:
        lib.qg_prefix_least_saving(before)
        call("sync")
        h.nm_stack_destroy(stack)
