"""core.Buffer, which takes blocks of the pool and gives them back natively (csrc/py/graph.cpp), against the pool's own methods.  The
driver is a stand-in that counts; nothing touches a device."""
import gc
import sys
import threading

import numpy as np
import pytest

from jittor_amd import _lib as L
from jittor_amd import core


class _Driver:
    def __init__(self):
        self.live, self.next = {}, 1 << 20

    def alloc(self, size):
        self.next += 1 << 32
        self.live[self.next] = size
        return self.next

    def free(self, ptr):
        del self.live[ptr]


@pytest.fixture
def driver(monkeypatch):
    d = _Driver()
    monkeypatch.setattr(L, "alloc", d.alloc)
    monkeypatch.setattr(L, "free", d.free)
    monkeypatch.setattr(L, "_device", 0)
    monkeypatch.setattr(core, "pool", core._Pool())
    yield d
    gc.collect()


def _cached(pool):
    return sorted((p, size) for size, lst in pool.free_blocks.items() for p in lst)


@pytest.mark.parametrize("n", [0, 1, 256, 257, 512, 513, 4096, 5000, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, (5 << 20) + 3])
def test_sizes_are_the_pools(driver, n):
    b = core.Buffer(n)
    assert b.size == core._Pool._round(n) == driver.live[b.ptr]
    ptr, size = b.ptr, b.size
    del b
    assert _cached(core.pool) == [(ptr, size)] and core.pool.cached_bytes == size
    b = core.Buffer(n)
    assert b.ptr == ptr and not core.pool.free_blocks and core.pool.cached_bytes == 0 and len(driver.live) == 1


def test_the_size_used_last_is_given_up_last(driver):
    core.pool.limit = 3000
    held = {n: core.Buffer(n) for n in (256, 512, 1024)}
    for n in (256, 512, 1024):
        del held[n]
    del n
    a = [core.Buffer(256)]
    a.clear()                                              # 256 is the size used last now
    assert list(core.pool.free_blocks) == [512, 1024, 256]
    big = [core.Buffer(2048)]
    big.clear()                                            # past the limit: the pool makes room, 512 and 1024 first
    assert list(core.pool.free_blocks) == [256, 2048] and core.pool.cached_bytes == 2304 == sum(driver.live.values())


def test_a_pool_with_methods_of_its_own_is_asked(driver, monkeypatch):
    seen = []
    monkeypatch.setattr(core.pool, "alloc", lambda n: (seen.append(("alloc", n)), (77, 256))[1])
    monkeypatch.setattr(core.pool, "free", lambda p, n: seen.append(("free", p, n)))
    b = core.Buffer(3)
    del b
    assert seen == [("alloc", 3), ("free", 77, 256)]


def test_without_a_device_blocks_are_dropped(driver, monkeypatch):
    b = core.Buffer(3)
    monkeypatch.setattr(L, "_device", None)
    del b
    assert not core.pool.free_blocks


def test_a_block_that_comes_back_in_the_middle_of_the_pools_bookkeeping_waits(driver):
    late, first = [core.Buffer(256)], core.Buffer(512)

    class Collecting(dict):
        def pop(self, *args):
            late.clear()
            return dict.pop(self, *args)

    second = core.Buffer(512)
    del first
    core.pool.free_blocks = Collecting(core.pool.free_blocks)
    del second                                             # not a plain table: the pool's own method, inside which `late` comes back
    assert sorted(size for size, lst in core.pool.free_blocks.items() for _ in lst) == [256, 512, 512] and core.pool.cached_bytes == 1280


def test_failures_are_the_pools(driver, monkeypatch):
    def refuse(size):
        raise L.MjtError(-4, "no memory")
    monkeypatch.setattr(L, "alloc", refuse)
    with pytest.raises(L.MjtError):
        core.Buffer(100)
    with pytest.raises(TypeError):
        core.Buffer()
    with pytest.raises(TypeError):
        core.Buffer("x")


@pytest.mark.parametrize("limit", [1 << 40, 5000])
def test_threads_that_make_and_drop_buffers(driver, limit):
    core.pool.limit = limit
    every, failed = sys.getswitchinterval(), []
    sys.setswitchinterval(1e-6)

    def work(seed):
        rng = np.random.default_rng(seed)
        held = []
        try:
            for k, size in enumerate(rng.choice([256, 512, 1024, 4096], 6000)):
                if k % 7 == 0:
                    held.append(core.pool.alloc(int(size)))        # the pool's methods in between
                else:
                    held.append(core.Buffer(int(size)))
                if len(held) > 3:
                    old = held.pop(0)
                    if isinstance(old, tuple):
                        core.pool.free(*old)
                    del old
            for old in held:
                if isinstance(old, tuple):
                    core.pool.free(*old)
        except Exception as e:                             # shown by the assertion below
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    try:
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(every)
    gc.collect()
    assert not failed, failed[:3]
    cached = _cached(core.pool)
    assert len({p for p, _ in cached}) == len(cached) and dict(cached) == driver.live
    assert core.pool.cached_bytes == sum(size for _, size in cached) <= limit and all(core.pool.free_blocks.values())
