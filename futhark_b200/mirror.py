"""What mirror.c does, through ctypes: the callables of the Python mirror where the native ones were not built (no compiler, no
Python headers, another interpreter).  The same kinds, arguments and errors; a call takes a few microseconds longer."""
import ctypes

_P = ctypes.c_void_p
MAX_ARGS = 6


def _address(x):
    if not isinstance(x, int):
        raise TypeError("an integer is required")
    if x < 0 or x >= 1 << 64:
        raise OverflowError("an address is out of range")
    return x


class Fn:
    """A function of libfuthark_b200.so"""

    def __init__(self, kind, *rest):
        if not isinstance(kind, str) or not rest:
            raise TypeError("a kind and an address are wanted")
        wanted = {"new_raw": (2,), "free": (1,), "interface": (4,), "array": (2,), "record": range(4, 8)}
        if kind not in wanted or len(rest) not in wanted[kind]:
            raise TypeError("no function of kind %s with %d arguments" % (kind, len(rest) + 1))
        addr = _address(rest[0])
        if addr == 0:
            raise ValueError("no address")
        self.kind = kind
        if kind == "new_raw":
            self.rank = rest[1]
            if self.rank not in (1, 2, 3):
                raise TypeError("one to three dimensions")
            self.fn = ctypes.CFUNCTYPE(_P, _P, ctypes.c_uint64, *[ctypes.c_int64] * self.rank)(addr)
        elif kind == "free":
            self.fn = ctypes.CFUNCTYPE(ctypes.c_int, _P, _P)(addr)
        elif kind == "interface":
            self.fn = ctypes.CFUNCTYPE(ctypes.POINTER(ctypes.c_int64), _P, _P)(addr)
            self.raw = ctypes.CFUNCTYPE(ctypes.c_uint64, _P, _P)(_address(rest[1]))
            self.rank, self.typestr = rest[2:]
        else:
            head = [_P, ctypes.POINTER(_P)] + ([ctypes.c_float] if rest[1] else [])
            self.float_first = bool(rest[1])
            self.entries = [None] + [ctypes.CFUNCTYPE(ctypes.c_int, *head, *[_P] * n)(addr) for n in range(1, MAX_ARGS + 1)]
            if kind == "record":
                self.free = ctypes.CFUNCTYPE(ctypes.c_int, _P, _P)(_address(rest[2]))
                self.project = [ctypes.CFUNCTYPE(ctypes.c_int, _P, ctypes.POINTER(_P), _P)(_address(p)) for p in rest[3:]]

    def __call__(self, *args):
        if len(args) < 2:
            raise TypeError("a context and at least one argument are wanted")
        ctx = _address(args[0])
        if ctx == 0:
            raise ValueError("the context is closed")
        if self.kind == "new_raw":
            if len(args) - 2 != self.rank:
                raise TypeError("%d dimensions are wanted, got %d" % (self.rank, len(args) - 2))
            dims = [d.__index__() if hasattr(d, "__index__") else _address(d) for d in args[2:]]
            return self.fn(ctx, _address(args[1]), *dims) or 0
        if self.kind in ("free", "interface"):
            if len(args) != 2:
                raise TypeError("a context and an array are wanted")
            arr = _address(args[1])
            if arr == 0:
                raise ValueError("the array has been freed")
            if self.kind == "free":
                return self.fn(ctx, arr)
            return {"shape": tuple(self.fn(ctx, arr)[:self.rank]), "typestr": self.typestr, "data": (self.raw(ctx, arr), False), "version": 2}
        head, arrays = [], args[1:]
        if self.float_first:
            head, arrays = [float(arrays[0])] if not isinstance(arrays[0], str) else _not_a_number(), arrays[1:]
        if len(arrays) > MAX_ARGS:
            raise TypeError("too many arguments")
        if not arrays:
            raise TypeError("an array is wanted")
        arrays = [_address(a) for a in arrays]
        if 0 in arrays:
            raise ValueError("an array has been freed")
        out = _P()
        rc = self.entries[len(arrays)](ctx, ctypes.byref(out), *head, *arrays)
        if rc != 0:
            return -abs(rc)
        if self.kind == "array":
            return out.value or 0
        parts = [_P() for _ in self.project]
        bad = [p(ctx, ctypes.byref(x), out) for p, x in zip(self.project, parts)]
        self.free(ctx, out)
        if any(bad):
            raise MemoryError
        return tuple(x.value or 0 for x in parts)


def _not_a_number():
    raise TypeError("must be real number, not str")
