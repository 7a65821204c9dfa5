"""When the residual tower's Python layers order the store's stream with torch's, without a device: the calls they make."""
import pytest


@pytest.fixture
def calls(monkeypatch):
    from ps_amd import api, native as N
    made = []

    class Lib:
        def ps_store_order(self, h, stream, store_first):
            made.append(("order", stream, store_first))
            return self.order_rc

        def ps_last_error(self):
            return b"refused"
        order_rc = 0
    lib = Lib()
    monkeypatch.setattr(N, "lib", lambda: lib)

    class Tensor:
        def __init__(self, stream):
            at[0] = stream                     # the one that its framework works on from here
    at = [None]
    monkeypatch.setattr(api, "_STREAM_OF", {Tensor: lambda device: at[0] if device == 3 else -1})

    class Store:
        h, device, stream = None, 3, None
    layer = api._TowerLayer(Store(), 0)

    def op(rc=0):
        def fn(h, n, *a):
            made.append(("call",) + a)
            return rc
        return fn
    return layer, lib, made, op, N, Tensor


def test_ordered_both_ways_unless_the_stream_is_shared(calls):
    layer, lib, made, op, N, T = calls
    layer._call(T(0), op(), 5)                                     # the store's own stream, torch's default one
    assert made == [("order", 0, 0), ("call", 5), ("order", 0, 1)]
    del made[:]
    layer.store.stream = 0                                         # the default stream adopted
    layer._call(T(0), op(), 5)
    layer._call(object(), op(), 6)                                 # no torch tensor: its owner's business
    assert made == [("call", 5), ("call", 6)]
    del made[:]
    layer._call(T(77), op(), 7)                                    # torch has left it
    assert made == [("order", 77, 0), ("call", 7), ("order", 77, 1)]


def test_a_refused_call_is_still_followed_by_the_join(calls):
    layer, lib, made, op, N, T = calls
    with pytest.raises(N.PsError):
        layer._call(T(9), op(N.PS_E_BAD_ARG))
    assert made == [("order", 9, 0), ("call",), ("order", 9, 1)]
    del made[:]
    lib.order_rc = N.PS_E_STATE                                    # a graph is being recorded there: nothing is enqueued
    with pytest.raises(N.PsError):
        layer._call(T(9), op())
    assert made == [("order", 9, 0)]


def test_the_adopted_handle_is_remembered(monkeypatch):
    import ctypes as C
    from ps_amd import api, native as N

    class Lib:
        def ps_store_set_stream(self, h, s):
            return 0
    monkeypatch.setattr(N, "lib", lambda: Lib())
    kv = api.KVStore.__new__(api.KVStore)
    kv.h = None
    assert kv.stream is None
    for given, kept in ((1234, 1234), (C.c_void_p(99), 99), (0, 0), (None, 0), (C.c_void_p(), 0)):
        kv.set_stream(given)
        assert kv.stream == kept
