"""What the paged cache's entry points refuse, before any launch: these run without a GPU."""
import pytest

A = 1 << 20        # an aligned address that is never read


@pytest.fixture()
def lib():
    from mytorch_b200 import _lib
    return _lib


def refused(call, args, text, lib):
    with pytest.raises(lib.MTError) as e:
        call(*args, None)
    assert text in str(e.value), str(e.value)


def test_tables_refusals(lib):
    bufs = [A + 256 * i for i in range(10)]
    ok = bufs + [4, 8, 16, 32, 10]
    for change, text in [({0: None}, "bad arguments"), ({9: None}, "bad arguments"), ({10: 0}, "requests"), ({10: 8193}, "requests"),
                         ({11: 0}, "positions"), ({12: 0}, "positions"), ({11: 1 << 27, 12: 16}, "positions"), ({11: 1 << 62, 12: 4}, "positions"),
                         ({13: -1}, "sizes"), ({14: -1}, "sizes"), ({14: 1 << 31}, "sizes"), ({6: bufs[0]}, "buffers of their own"),
                         ({9: bufs[4]}, "buffers of their own")]:
        refused(lib.paged_tables, [change.get(i, v) for i, v in enumerate(ok)], text, lib)


def test_release_refusals(lib):
    ok = [A + 256 * i for i in range(5)] + [4, 8, 16, 32]
    for change, text in [({0: None}, "bad arguments"), ({5: 0}, "requests"), ({5: 8193}, "requests"), ({6: 0}, "sizes"), ({7: 0}, "sizes"),
                         ({8: -1}, "sizes")]:
        refused(lib.paged_release, [change.get(i, v) for i, v in enumerate(ok)], text, lib)


def test_append_refusals(lib):
    st = lib.Strides3(0, 64, 128)
    ok = [A, A, A, A, st, st, st, A, 3, 2, 64, 16, 8, lib.F16]
    for change, text in [({0: None}, "bad arguments"), ({7: None}, "bad arguments"), ({8: -1}, "bad arguments"), ({9: 0}, "bad arguments"),
                         ({10: 0}, "bad arguments"), ({11: 0}, "2^31"), ({11: 1 << 16, 12: 1 << 15}, "2^31"), ({13: 9}, "dtype")]:
        refused(lib.paged_append, [change.get(i, v) for i, v in enumerate(ok)], text, lib)


def test_attention_refusals(lib):
    row, pages = lib.Strides3(0, 64, 256), lib.Strides3(2048, 1024, 64)
    ok = [A, A, A, A + 4096, row, pages, row, A, A, A, 2, 8, 3, 1, 4, 2, 64, 16, 8, 0.125, lib.BF16]
    for change, text in [({0: None}, "bad arguments"), ({9: None}, "bad arguments"), ({10: -1}, "bad arguments"), ({14: 3}, "multiple"),
                         ({16: 80}, "head_dim"), ({17: 0}, "positions"), ({11: 1 << 28}, "positions"), ({11: 1 << 62, 17: 4}, "positions"),
                         ({5: lib.Strides3(2048, 1024, 60)}, "16-byte"), ({5: lib.Strides3(2050, 1024, 64)}, "16-byte"), ({1: A + 2}, "16-byte"),
                         ({3: A}, "of its own"), ({19: 0.0}, "scale"), ({19: -1.0}, "scale"), ({19: float("inf")}, "scale"), ({19: float("nan")}, "scale"),
                         ({20: 5}, "dtype"), ({12: 1 << 30, 14: 4}, "rows"), ({13: -1}, "rows")]:
        refused(lib.attn_paged, [change.get(i, v) for i, v in enumerate(ok)], text, lib)


class Fake:
    """The shape and type of a device array; nothing behind it."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.ndim, self.ptr, self.code = shape, dtype, len(shape), A, {"float16": 1, "float32": 0}.get(dtype)


@pytest.fixture()
def K(monkeypatch):
    from mytorch_b200 import fused_ops
    monkeypatch.setattr(fused_ops, "_A", lambda a: a)
    monkeypatch.setattr(fused_ops, "stream", lambda: pytest.fail("reached the launch"))
    return fused_ops


def i(*shape):
    return Fake(shape, "int32")


def h(*shape):
    return Fake(shape, "float16")


def test_python_refusals(K):
    pools = h(8, 2, 16, 64), h(8, 2, 16, 64)
    attend = lambda q=h(5, 4, 64), k=pools[0], v=pools[1], t=i(3, 9), s=i(4), n=i(3), **kw: K.fused_paged_attention(q, k, v, t, s, n, **kw)
    for bad in (dict(q=h(5, 3, 64)), dict(q=h(5, 4, 32)), dict(q=h(5, 256)), dict(v=h(8, 2, 16, 32)), dict(t=i(2, 9)), dict(t=h(3, 9)),
                dict(s=i(3)), dict(n=i(3, 1)), dict(out=h(5, 2, 64)), dict(out=Fake((5, 4, 64), "float32"))):
        with pytest.raises(ValueError):
            attend(**bad)
    with pytest.raises(TypeError):
        attend(q=Fake((5, 4, 64), "float32"))
    for bad in ((h(5, 2, 64), h(4, 2, 64), i(5)), (h(5, 1, 64), h(5, 1, 64), i(5)), (h(5, 2, 64), h(5, 2, 64), i(4)), (h(5, 2, 64), h(5, 2, 64), h(5))):
        with pytest.raises(ValueError):
            K.fused_paged_append(bad[0], bad[1], *pools, bad[2])
    tables = lambda held=i(3), fresh=i(3), t=i(3, 4), free=i(9), n=i(1), **kw: K.fused_paged_tables(held, fresh, t, free, n, 16, **kw)
    for bad in (dict(fresh=i(2)), dict(t=i(2, 4)), dict(n=i(2)), dict(held=h(3)), dict(), dict(out=(i(3), i(3), i(5), i(5), i(1))),
                dict(out=(i(4), i(3), i(5), i(4), i(1))), dict(rows=6, out=(i(4), i(3), i(5), i(5), i(1)))):
        with pytest.raises(ValueError):
            tables(**bad)
    with pytest.raises(ValueError):
        K.fused_paged_release(i(3), i(3, 4), i(2), i(9), i(1), 16)
