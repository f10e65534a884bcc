"""The native callables of the Python mirror on a context that did not come up: their checks of arguments, borrowed
arrays and their descriptions need no GPU."""
import ctypes

import numpy as np
import pytest

import futhark_b200 as fb


@pytest.fixture(scope="module")
def bare():
    """A context object, whether or not there is a GPU; nothing of it is used but its address."""
    from futhark_b200 import build
    build.build()
    L = fb.load()
    cfg = L.futhark_context_config_new()
    ctx = L.futhark_context_new(cfg)
    fb._take_string(L.futhark_context_get_error(ctx))
    yield ctx
    L.futhark_context_free(ctx)
    L.futhark_context_config_free(cfg)


@pytest.mark.parametrize("tname", sorted(fb.ARRAY_TYPES))
def test_borrowed_arrays_describe_themselves(bare, tname):
    dtype, rank, _ = fb.ARRAY_TYPES[tname]
    f = fb._type_fns[tname]
    dims = (5, 0, 7)[:rank]
    a = f.new_raw(bare, 0x7f0000001230, *dims)
    assert f.interface(bare, a) == {"shape": dims, "typestr": np.dtype(dtype).str, "data": (0x7f0000001230, False), "version": 2}
    assert f.free(bare, a) == 0


def test_arguments_are_checked(bare):
    f = fb._type_fns["f32_2d"]
    for args in ((bare, 16, 3), (bare, 16, 3, 3, 3), (bare, 16), (bare,), ()):
        with pytest.raises(TypeError):
            f.new_raw(*args)
    with pytest.raises(TypeError):
        f.new_raw(bare, 16, 3, "4")
    with pytest.raises(OverflowError):
        f.new_raw(bare, -1, 3, 4)
    with pytest.raises(ValueError):                    # a closed context's address is 0 or None
        f.new_raw(0, 16, 3, 4)
    with pytest.raises((TypeError, ValueError)):
        f.free(bare, None)
    entry = fb._entries["vocab_xent_f16", False, fb.LOSSES, 2]
    with pytest.raises((TypeError, ValueError)):
        entry(bare, None, None, None)
    Fn = fb._native().Fn
    for bad in (("new_raw", 1), ("free",), ("nothing", 1), (1, 1), ("new_raw", 1, 4), ("free", 0)):
        with pytest.raises((TypeError, ValueError)):
            Fn(*bad)


def test_a_context_that_did_not_come_up_refuses(bare):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    a = fb._type_fns["f16_2d"].new_raw(bare, 256, 3, 4)
    t = fb._type_fns["i32_1d"].new_raw(bare, 256, 3)
    assert fb._entries["vocab_xent_f16", False, fb.LOSSES, 2](bare, a, a, t) == -1
    assert "failed to initialise" in fb._take_string(fb.load().futhark_context_get_error(bare))
    s = fb._type_fns["f32_2d"].new_raw(bare, 256, 3, 4)
    i = fb._type_fns["i32_2d"].new_raw(bare, 256, 3, 4)
    assert fb._entries["topk_distill_grad_f32", True, "", 0](bare, 1.0, s, i, s, t, t) == -1
    fb._take_string(fb.load().futhark_context_get_error(bare))
    with pytest.raises(TypeError):
        fb._entries["topk_distill_grad_f32", True, "", 0](bare, "one", s, i, s, t, t)
    for name, x in (("f16_2d", a), ("i32_1d", t), ("f32_2d", s), ("i32_2d", i)):
        assert fb._type_fns[name].free(bare, x) == 0
