"""The quick entries of the binding: the same function, the same refusals, and
the ctypes path for whatever they do not take."""
import ctypes

import pytest


@pytest.fixture
def quick(rnet):
    rnet.lib()
    return rnet._quick


ENTRIES = ["rnet_topk_logits_forward", "rnet_distill_topk_forward", "rnet_beam_select",
           "rnet_beam_reorder", "rnet_beam_backtrack"]
SELECT = (4096, 0, 64, 8192, None, -1, 12288, 16384, 20480, None, 0, 4, 64, None)


@pytest.mark.parametrize("name", ENTRIES)
def test_entries_take_what_ctypes_takes(rnet, quick, name):
    kinds = rnet._SIGS[name]
    args = [None if k is ctypes.c_void_p else 0.0 if k is ctypes.c_float else 0 for k in kinds]
    f, g = getattr(quick, name), getattr(rnet.lib(), name)
    rc = f(*args)
    assert rc is not NotImplemented and rc == g(*args)
    assert f(*args[:-1]) is NotImplemented and f(*args, 0) is NotImplemented
    for i, k in enumerate(kinds):
        wrong = ["x", 1.5 if k is not ctypes.c_float else "1", ctypes.c_void_p(8), b""]
        if k is ctypes.c_int:
            wrong += [None, 1 << 31, -(1 << 31) - 1]
        if k in (ctypes.c_longlong, ctypes.c_size_t):
            wrong += [None, 1 << 64]
        if k is ctypes.c_size_t:
            wrong += [-1]
        if k is ctypes.c_float:
            wrong += [None]
            assert f(*args[:i], 1, *args[i + 1:]) is not NotImplemented
        for w in wrong:
            assert f(*args[:i], w, *args[i + 1:]) is NotImplemented, (name, i, w)


def test_call_refuses_with_the_librarys_message(rnet):
    rnet.call("rnet_beam_select", *SELECT)  # no sequences: nothing to do
    with pytest.raises(rnet.RnetError, match="beam_select: null pointer"):
        rnet.call("rnet_beam_select", None, *SELECT[1:])
    with pytest.raises(rnet.RnetError, match="row pitch below vocab"):
        rnet.call("rnet_beam_select", *SELECT[:2], 63, *SELECT[3:])


def test_call_takes_other_arguments_through_ctypes(rnet):
    rnet.call("rnet_beam_select", ctypes.c_void_p(4096), *SELECT[1:])
    with pytest.raises(ctypes.ArgumentError):
        rnet.call("rnet_beam_select", SELECT[0], "f32", *SELECT[2:])
    with pytest.raises(TypeError):
        rnet.call("rnet_beam_select", *SELECT[:-1])
