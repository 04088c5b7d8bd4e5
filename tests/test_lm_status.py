"""The status words' host side (CPU only)."""

import threading
import time


def test_threads_share_one_set_of_status_words(monkeypatch):
    """First calls of several threads at once get the same words: a launch holds their
    address for good, so words that only one thread knows would be lost."""
    from prlstm_b200 import _lib

    class Slow:
        def __init__(self):
            time.sleep(0.05)

    monkeypatch.setattr(_lib, "HostStatus", Slow)
    monkeypatch.setattr(_lib, "_host_status", {})
    go, got = threading.Barrier(8), []

    def first():
        go.wait()
        got.append(_lib.host_status(0))

    threads = [threading.Thread(target=first) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 8 and all(s is got[0] for s in got) and _lib._host_status[0] is got[0]
