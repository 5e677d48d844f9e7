"""Example bank, without a GPU: the C entry points refuse what their kernels were not written for before anything is launched."""
import ctypes

import pytest
import torch


def _struct(**change):
    from super_resolution_amd import _lib
    f = dict(k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096, offset=4096, centroid=4096, pages=8, heads=2, page_rows=64,
             dim=64, bits=4, kernel_id=0)
    return _lib.Bank(**{**f, **change})


def _calls(bank, **change):
    """Every entry point with plausible (never dereferenced) arguments, some of them replaced."""
    from super_resolution_amd import _lib
    lib = _lib.load()
    a = dict(table=4096, B=2, J=4, start=4096, count=4096, k=4096, v=4096, dtype=0, T=3, length=4096, q=4096, Hq=4, scale=1.0,
             out=4096, sel=4096, n_sel=4)
    a.update(change)
    st = (ctypes.c_int64 * 3)(64, 64, 64)
    ref = None if bank is None else ctypes.byref(bank)
    big = 1 << 62
    return {
        "write": lambda: lib.gpsr_bank_write(ref, a["table"], a["B"], a["J"], a["start"], a["count"], a["k"], a["v"], a["dtype"], a["T"], st, st, None),
        "read": lambda: lib.gpsr_bank_read(ref, a["table"], a["B"], a["J"], a["start"], a["count"], a["k"], a["v"], a["dtype"], a["T"], None),
        "attend": lambda: lib.gpsr_bank_attend(ref, a["table"], a["B"], a["J"], a["length"], a["q"], a["dtype"], a["T"], a["Hq"], st,
                                               a["scale"], None, a["out"], None, 4096, big, None),
        "select": lambda: lib.gpsr_bank_select(ref, a["table"], a["B"], a["J"], a["length"], a["q"], a["dtype"], a["T"], a["Hq"], st,
                                               a["n_sel"], None, a["sel"], 4096, big, None),
        "pages": lambda: lib.gpsr_bank_attend_pages(ref, a["table"], a["B"], a["J"], a["length"], a["q"], a["dtype"], a["T"], a["Hq"], st,
                                                    a["sel"], a["n_sel"], a["scale"], None, a["out"], None, 4096, big, None),
    }, lib


ALL = ("write", "read", "attend", "select", "pages")


@pytest.mark.parametrize("change", [dict(k_codes=0), dict(v_scales=0), dict(centroid=0), dict(offset=4100), dict(k_codes=4104), dict(pages=0),
                                    dict(pages=1 << 31), dict(heads=0), dict(heads=65536), dict(page_rows=8), dict(page_rows=48),
                                    dict(page_rows=512), dict(dim=0), dict(dim=48), dict(dim=160), dict(dim=512), dict(bits=2), dict(bits=16),
                                    dict(kernel_id=1), dict(kernel_id=3), dict(kernel_id=-1)])
def test_banks_that_no_kernel_takes(change):
    calls, lib = _calls(_struct(**change))
    for name in ALL:
        assert calls[name]() == -1, name
        assert b"bank" in lib.gpsr_last_error()


def test_null_and_out_of_range_arguments():
    calls, _ = _calls(None)
    assert all(calls[n]() == -1 for n in ALL)
    for change, which in ((dict(table=0), ALL), (dict(length=0), ("attend", "select", "pages")), (dict(q=0), ("attend", "select", "pages")),
                          (dict(out=0), ("attend", "pages")), (dict(sel=0), ("select", "pages")), (dict(start=0), ("write", "read")),
                          (dict(count=0), ("write", "read")), (dict(k=0), ("write", "read")), (dict(v=0), ("write", "read")),
                          (dict(dtype=3), ALL), (dict(dtype=-1), ALL), (dict(B=65536), ALL), (dict(J=-1), ALL), (dict(J=0), ("write", "read")),
                          (dict(Hq=3), ("attend", "select", "pages")), (dict(Hq=0), ("attend", "select", "pages")),
                          (dict(Hq=131072), ("attend", "select", "pages")), (dict(n_sel=0), ("select", "pages")),
                          (dict(n_sel=65), ("select", "pages")), (dict(scale=0.0), ("attend", "pages")), (dict(scale=-1.0), ("attend", "pages")),
                          (dict(scale=float("nan")), ("attend", "pages")), (dict(scale=float("inf")), ("attend", "pages")),
                          (dict(out=4100), ("attend", "pages")), (dict(k=4100), ("read",))):
        calls, _ = _calls(_struct(), **change)
        for name in which:
            assert calls[name]() == -1, (change, name)


def test_empty_batches_are_no_ops():
    for change in (dict(B=0), dict(T=0)):
        calls, _ = _calls(_struct(), **change)
        assert all(calls[n]() == 0 for n in ALL)


def test_ops_refuse_host_tensors():
    from super_resolution_amd import _lib, ops
    u8, f32, i32 = (lambda *s: torch.zeros(s, dtype=torch.uint8)), (lambda *s: torch.zeros(s)), (lambda *s: torch.zeros(s, dtype=torch.int32))
    bank = ops.Bank(u8(2, 1, 16, 32), u8(2, 1, 16, 2), u8(2, 1, 16, 32), u8(2, 1, 16, 2), f32(2, 1, 16), f32(2, 1, 64))
    for f in (lambda: ops.bank_write(bank, i32(1, 2), i32(1), i32(1), f32(1, 1, 1, 64), f32(1, 1, 1, 64)),
              lambda: ops.bank_read(bank, i32(1, 2), i32(1), i32(1), 1), lambda: ops.bank_attend(bank, i32(1, 2), i32(1), f32(1, 1, 1, 64), 1.0),
              lambda: ops.bank_select(bank, i32(1, 2), i32(1), f32(1, 1, 1, 64), 1),
              lambda: ops.bank_attend_pages(bank, i32(1, 2), i32(1), f32(1, 1, 1, 64), i32(1, 1, 1, 2), 1.0)):
        with pytest.raises(_lib.GpsrError, match="device tensors"):
            f()


def test_windows_and_blend_refuse():
    from super_resolution_amd import _lib
    lib = _lib.load()
    ok = dict(img=4096, H=20, W=20, side=7, rows=4096, dtype=0, dim=64, out=4096)
    for change in (dict(img=0), dict(rows=0), dict(side=4), dict(side=1), dict(side=17), dict(H=6), dict(W=6), dict(dim=48), dict(dim=257),
                   dict(dtype=3), dict(H=65536)):
        a = {**ok, **change}
        assert lib.gpsr_bank_windows(a["img"], a["H"], a["W"], a["side"], 1, a["rows"], a["dtype"], a["dim"], None) == -1, change
        assert lib.gpsr_bank_blend(a["img"], a["H"], a["W"], a["side"], a["rows"], a["dtype"], a["dim"], a["out"], None) == -1, change
    a = {**ok, "out": 0}
    assert lib.gpsr_bank_blend(a["img"], a["H"], a["W"], a["side"], a["rows"], a["dtype"], a["dim"], a["out"], None) == -1


def test_calls_too_large_for_a_launch_are_refused():
    """A launch has fewer than 2^32 threads along a dimension: 256 for 4 queries, 8 columns a thread, or a page."""
    most = (1 << 31) - 1
    for change, which in ((dict(T=most), ("read", "attend", "select", "pages")), (dict(T=most, J=1 << 25), ("write",)),
                          (dict(T=(1 << 26) + 1, J=1 << 20, n_sel=1), ("attend", "select", "pages")), (dict(T=1 << 24, J=0, n_sel=2), ("pages",))):
        calls, lib = _calls(_struct(page_rows=16), **change)
        for name in which:
            assert calls[name]() == -1 and b"too many" in lib.gpsr_last_error(), (change, name)
    for call in (lambda lib: lib.gpsr_bank_windows(4096, 9, (1 << 24) + 1, 3, 1, 4096, 0, 32, None),
                 lambda lib: lib.gpsr_bank_blend(4096, 9, (1 << 24) + 1, 3, 4096, 0, 32, 4096, None)):
        lib = _calls(_struct())[1]
        assert call(lib) == -1 and b"columns" in lib.gpsr_last_error()
