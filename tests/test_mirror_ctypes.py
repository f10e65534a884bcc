"""The Python mirror where its native callables were not built: the library builds, and calls go through ctypes with the same
checks and results."""
import os
import sys

import numpy as np
import pytest

import futhark_b200 as fb
import test_mirror
from test_mirror import bare  # noqa: F401 (fixture)


@pytest.fixture
def without_native(monkeypatch):
    monkeypatch.setitem(sys.modules, "futhark_b200._mirror", None)       # importing it raises ImportError
    monkeypatch.delattr(fb, "_mirror", raising=False)
    monkeypatch.setattr(fb, "_mirror_module", None)
    for table in (fb._type_fns, fb._entries):
        table.clear()
    yield
    for table in (fb._type_fns, fb._entries):
        table.clear()


def test_the_library_builds_without_headers_or_compiler(monkeypatch, tmp_path, capsys):
    from futhark_b200 import build
    monkeypatch.setattr(build, "MIRROR", str(tmp_path / "_mirror.so"))
    for cc in ("false", str(tmp_path / "no-such-compiler")):
        monkeypatch.setenv("CC", cc)
        assert build.build() == build.LIB and os.path.exists(build.LIB)
        assert "ctypes" in capsys.readouterr().err
    assert not os.path.exists(build.MIRROR)


def test_calls_go_through_ctypes(without_native):
    assert fb._native().__name__ == "futhark_b200.mirror"


@pytest.mark.parametrize("tname", sorted(fb.ARRAY_TYPES))
def test_borrowed_arrays_describe_themselves(without_native, bare, tname):  # noqa: F811
    test_mirror.test_borrowed_arrays_describe_themselves(bare, tname)


def test_checks(without_native, bare):  # noqa: F811
    test_mirror.test_arguments_are_checked(bare)
    test_mirror.test_loss_entry_points_check_the_types_of_arrays()


def test_a_context_that_did_not_come_up_refuses(without_native, bare):  # noqa: F811
    test_mirror.test_a_context_that_did_not_come_up_refuses(bare)


@pytest.mark.gpu
def test_losses_and_other_calls(without_native, ctx):
    import test_gpu_losses as t
    t.check_xent(ctx, *t.xent_inputs(40, 300, 64, 1))
    t.check_distill(ctx, "f16", 2.0, *t.distill_inputs("f16", 9, 500, 4, 2))
    t.check_router(ctx, "f32", *t.router_inputs("f32", 50, 8, 2, 3), 0.1)
    t.refused(ctx, lambda: fb.vocab_xent_f16(ctx, np.zeros((2, 3)), np.zeros((4, 5)), np.zeros(2)), "invalid sizes")
    xs = np.arange(1000, dtype=np.int32)
    assert fb.reduce_i32(ctx, xs) == xs.sum() and np.array_equal(fb.scan_i32(ctx, xs), np.cumsum(xs))
    a = ctx.new("i32_1d", xs)
    b = ctx.new_raw("i32_1d", a.raw + 40, 20)
    assert np.array_equal(b.values(), xs[10:30]) and b.shape == (20,) and b.__cuda_array_interface__["data"][0] == a.raw + 40
    b.free()
    a.free()
