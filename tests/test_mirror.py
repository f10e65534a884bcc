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


def test_loss_entry_points_check_the_types_of_arrays():
    ctx = fb.Context.__new__(fb.Context)
    ctx.ptr = None                           # a closed one: whatever passes the check of types is refused there
    wanted = {
        "entry_vocab_xent_f16": ((), ("f16_2d", "f16_2d", "i32_1d")),
        "entry_vocab_xent_grad_f16": ((), ("f16_2d", "f16_2d", "i32_1d", "f32_1d", "f32_1d", "f32_1d")),
        "entry_topk_distill": (("f16", 1.0), ("f16_2d", "i32_2d", "f32_2d")),
        "entry_topk_distill_grad": (("f32", 1.0), ("f32_2d", "i32_2d", "f32_2d", "f32_1d", "f32_1d")),
        "entry_router_balance": (("f32",), ("f32_2d", "bool_1d", "i32_2d")),
        "entry_router_balance_grad": (("f16",), ("f16_2d", "bool_1d", "i32_1d", "f32_1d", "f32_1d")),
    }

    def arrays(types):
        return [fb.Array(ctx, t, None) for t in types]

    for name, (head, types) in wanted.items():
        for i in range(len(types)):
            for other in ("f32_2d", "f16_2d", "i32_1d", "f32_1d", "f64_2d"):
                if other != types[i]:
                    with pytest.raises(TypeError, match="arrays of types"):
                        getattr(ctx, name)(*head, *arrays(types[:i] + (other,) + types[i + 1:]))
        with pytest.raises((TypeError, ValueError), match="(?!arrays of types)"):
            getattr(ctx, name)(*head, *arrays(types))


def test_a_description_belongs_to_its_caller(bare):
    ctx = fb.Context.__new__(fb.Context)
    ctx.ptr = bare
    a = fb.Array(ctx, "f32_2d", fb._type_fns["f32_2d"].new_raw(bare, 4096, 3, 5))
    d = a.__cuda_array_interface__
    want = dict(d)
    d["version"] = 3
    d.pop("shape")
    assert a.__cuda_array_interface__ == want and a.shape == (3, 5)
    a.free()
