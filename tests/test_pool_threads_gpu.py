"""Page pools of different sizes used by several host threads at once."""
import ctypes
import threading

import pytest
import torch

from ananta_ocr_b200 import _lib as L
from ananta_ocr_b200.page_pool import PagePool

pytestmark = pytest.mark.gpu


def test_pools_of_two_sizes_in_two_threads():
    """The kernels' shared memory goes by the pool's size (25 and 164 KB for
    ``free``): a call on a small pool must not lower the limit that a call of
    another thread on a large one is about to launch under."""
    failures, lib = [], L.load()

    def work(pages, rows, stream):
        with torch.cuda.stream(stream):
            pool = PagePool(pages, rows, 4, 16)
            some = torch.arange(rows, dtype=torch.int32, device="cuda")
            args = pool._args(None, some.data_ptr(), 0, 0, 1)
            at, st = ctypes.byref(args), stream.cuda_stream
            start.wait()
            for _ in range(20_000):
                rc = lib.dash_pages_free(at, st)           # row 0, which holds nothing
                if rc != L.DASH_OK:
                    failures.append((pages, rc, L.last_error()))
                    break
            stream.synchronize()
            if pool.n_free.item() != pages:
                failures.append((pages, "n_free"))

    start = threading.Barrier(2)
    threads = [threading.Thread(target=work, args=(p, r, torch.cuda.Stream()))
               for p, r in ((100_000, 2), (1 << 19, 8192))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failures, failures
