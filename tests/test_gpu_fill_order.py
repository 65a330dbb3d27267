"""GPU: fills that are only noted, with two threads: the next call of either thread enqueues them, and no thread's call goes
ahead of its own fill."""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F32 = np.float32


def test_fills_of_one_thread_are_not_enqueued_behind_its_calls(hip):
    # noted fills of both threads go out with the next call of either; each thread's calls overwrite what it filled
    before = hip.fusing
    hip.set_fusing(False)
    wrong, start = [], threading.Barrier(2)

    def work(n):
        a, b = hip.create_from_numpy(np.full((7, 9), n + 2.0, F32)), hip.create_from_numpy(np.full((7, 9), 0.5, F32))
        start.wait()
        for k in range(400):
            out = hip.empty((7, 9))
            hip.fill(out, 5.0)
            hip.mult_tt(a, b, out)
            if not (out.get() == (n + 2.0) * 0.5).all():
                wrong.append((n, k))

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(100)
    hip.set_fusing(before)
    assert not wrong, wrong[:5]
