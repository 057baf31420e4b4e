"""Compiles the kernels of the GPU tests while they run.

Most of a GPU test's time is the run-time compiler's, one kernel after the other (0.2 s each, some 4000 in all).  A run of many GPU tests
therefore starts helpers, each with every n-th chunk of the same tests in compile-only mode: results are zeros, assertions are off, and
what is left of a test are its kernels, which land in the cache on disk that the run itself looks into.  A helper that fails costs the run nothing
but time."""
import ctypes
import os
import signal
import subprocess
import sys
import tempfile

import numpy as np

HELPERS, CHUNK, FEWEST = 10, 8, 100
_lists = []
_VARIABLE = "MJT_TESTS_AHEAD"                                # "number of the helper/helpers/file with the names of the tests"


def is_helper():
    return _VARIABLE in os.environ


def start(items, root):
    """Helpers for a run of these tests; none where the run is short, has no GPU, or keeps no cache."""
    names = [t.nodeid for t in items if t.get_closest_marker("gpu")]
    n = min(HELPERS, len(os.sched_getaffinity(0)) - 2)
    if is_helper() or len(names) < FEWEST or n < 1 or not os.path.exists("/dev/kfd") or os.environ.get("MJT_NO_DISK_CACHE"):
        return []
    with tempfile.NamedTemporaryFile("w", suffix=".txt", delete=False) as f:
        f.write("\n".join(names))
    _lists.append(f.name)
    env = dict(os.environ, OMP_NUM_THREADS="1", OPENBLAS_NUM_THREADS="1", HIP_VISIBLE_DEVICES="-1")      # (no helper sees a device)
    env.pop("PYTEST_ADDOPTS", None)
    command = [sys.executable, "-O", "-m", "pytest", "--assert=plain", "-p", "no:cacheprovider", "-q", "-m", "gpu", os.path.join(root, "tests")]
    return [subprocess.Popen(command, cwd=root, env=dict(env, **{_VARIABLE: "%d/%d/%s" % (i, n, f.name)}), stdin=subprocess.DEVNULL, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
            for i in range(n)]


def stop(helpers):
    for p in helpers:
        p.kill()
    for p in helpers:
        p.wait()
    while _lists:
        os.unlink(_lists.pop())


def become_helper():
    """Compile-only mode, and nothing that reads a result or a device."""
    ctypes.CDLL(None).prctl(1, signal.SIGKILL)              # PR_SET_PDEATHSIG: not longer than the run itself
    from jittor_amd import _lib as L
    L.init(-1)
    at = [1 << 40]

    def alloc(n):
        at[0] += 1 << 33
        return at[0]

    class Event:
        def record(self):
            return self

        def elapsed_ms_since(self, start):
            return 1.0

    L.alloc, L.free, L.h2d, L.d2h, L.sync, L.Event = alloc, lambda p: None, lambda p, a: None, lambda p, shape, dtype: np.zeros(shape, dtype), lambda: None, Event
    L.check, L.init, L.shutdown = lambda rc: rc, lambda device=0: L.load(), lambda: None
    for name in ("assert_allclose", "assert_array_equal", "assert_equal", "assert_almost_equal", "assert_array_almost_equal", "assert_array_less"):
        setattr(np.testing, name, lambda *a, **k: None)


def share(items):
    """The helper's tests, in the run's order."""
    i, n, path = os.environ[_VARIABLE].split("/", 2)
    with open(path) as f:
        names = f.read().split("\n")
    place = {name: k for k, name in enumerate(names)}
    mine = [t for t in items if place.get(t.nodeid, -1) // CHUNK % int(n) == int(i) and t.nodeid in place]
    return sorted(mine, key=lambda t: place[t.nodeid])
