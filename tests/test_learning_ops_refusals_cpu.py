"""More refusals of the learning operators' entry points, which need no GPU."""
import ctypes
import math

from go_ai import _hip

lib = _hip.lib


def test_adamw_scalars():
    call = lambda t=1, lr=1e-3, b1=0.9, b2=0.999, opt=64, out=64: lib.goai_adamw_scalars(None, opt, t, lr, b1, b2, out)  # noqa: E731
    for bad, message in ((dict(t=0), "t = 1"), (dict(lr=-1.0), "lr"), (dict(lr=math.nan), "lr"), (dict(b1=1.0), "betas"), (dict(b2=math.nan), "betas"),
                         (dict(opt=None), "NULL"), (dict(out=None), "NULL"), (dict(), "ctx is NULL")):
        assert call(**bad) == -1 and message in lib.goai_last_error().decode(), bad


def test_adamw_skipped():
    n = ctypes.c_int64(5)
    assert lib.goai_adamw_skipped(None, None, ctypes.byref(n)) == -1 and "NULL" in lib.goai_last_error().decode()
    assert lib.goai_adamw_skipped(None, 64, None) == -1 and "NULL" in lib.goai_last_error().decode()
