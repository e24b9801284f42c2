"""A wait of the cache for the device leaves Python's other threads running."""
import threading
import time

import pytest
import torch

from test_gpu_kv4 import filled

pytestmark = pytest.mark.gpu


def test_freeing_a_cache_lets_other_threads_run(pkg):
    """free() and the end of a cache's life wait for the device; a thread of Python's goes on meanwhile."""
    for end in ("free", "del"):
        cache, _, _, _ = filled(pkg, 1, 20, 2, 64, 1)
        torch.cuda.synchronize()
        stamps, stop = [], threading.Event()

        def watch():
            while not stop.is_set():
                stamps.append(time.perf_counter())
                time.sleep(0.002)

        thread = threading.Thread(target=watch)
        thread.start()
        torch.cuda._sleep(800_000_000)  # cycles: 0.4 s and more
        begin = time.perf_counter()
        if end == "free":
            cache.free()
        del cache
        done = time.perf_counter()
        stop.set()
        thread.join()
        torch.cuda.synchronize()
        assert done - begin > 0.2
        assert sum(begin < s < done for s in stamps) > 20
