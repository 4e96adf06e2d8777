"""Errors of calls from several threads."""
import threading


def test_each_thread_has_its_own_error():
    import dcamd
    L = dcamd.Lib()
    first, second, got = threading.Event(), threading.Event(), []

    def one():
        assert L.L.dc_act_forward_device(9, 1, 4, 8, None, 8, None, 0, None, 8, None, None, None) == -2
        first.set()
        assert second.wait(20)
        got.append(L.err())

    def other():
        assert first.wait(20)
        assert L.L.dc_kv_status(None, None, 0) == -2
        got.append(L.err())
        second.set()

    threads = [threading.Thread(target=f) for f in (one, other)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 2 and "status" in got[0] and "activation: unknown kind" in got[1], got
