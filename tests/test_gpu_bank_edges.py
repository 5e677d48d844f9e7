"""Example bank at its edges: pages and columns of unlike size, keys past the range, queries that are not numbers, rows that are
not there, the ways that only many queries take.  Definitions and bounds as in test_gpu_bank.py."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_bank import BF16, F16, F32, Case, _ops, _skips, held


def _rewrite(c, kernel="RBF"):
    """Writes c.k and c.v as they are now, and what the bank holds of them in 64 bits."""
    _ops().bank_write(c.bank, c.table, torch.zeros_like(c.length), c.length, c.k.to(c.dev), c.v.to(c.dev))
    c.hk, c.hv = held(c.k.double().numpy(), c.bits), held(c.v.double().numpy(), c.bits)
    c.o = -0.5 * (c.hk ** 2).sum(-1) if kernel == "RBF" else np.zeros(c.hk.shape[:-1])


def _choices(c, T, S):
    """S different pages for each query, and who sees what."""
    pages = -(-c.lengths[0] // c.P)
    sel = c.rng.permuted(np.tile(np.arange(pages), (T, 1)), axis=1)[None, :, None, :S].astype(np.int32)
    seen = lambda b, t, h: np.isin(np.arange(c.lengths[0]) // c.P, sel[b, t, h])
    return torch.as_tensor(np.ascontiguousarray(sel)).to(c.dev), seen


def _pages_workspace(c, T, Hq, S, dtype):
    from super_resolution_amd import _lib
    ref, _, _ = _ops()._bank(c.bank, c.dev.index)
    code = {BF16: 0, F16: 1, F32: 2}[dtype]
    return _lib.load().gpsr_bank_attend_pages_workspace_bytes(ref, 1, c.table.shape[1], T, Hq, S, code)


# 40 queries go by query, 2900 by page (test_which_way_the_pages_go in test_gpu_bank.py)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [40, 2900])
def test_pages_whose_values_are_of_unlike_size_weigh_what_their_keys_say(dtype, T):
    """Equal keys, values of 2^-100 in every second page and of 2^60 in the others."""
    ops = _ops()
    c = Case([900], 1, 64, 32, 4, "RBF", dtype, seed=T)
    c.k.zero_()
    c.v = torch.where((torch.arange(900) // 32 % 2 == 0)[None, :, None, None], 2.0 ** -100, 2.0 ** 60).expand(1, 900, 1, 64).to(dtype).contiguous()
    _rewrite(c)
    q, qd = c.queries(T, 1, dtype)
    sel, seen = _choices(c, T, 16)
    out, lse = ops.bank_attend_pages(c.bank, c.table, c.length, qd, sel, 0.25, want_lse=True)
    c.check(q, out, lse, 0.25, seen)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [40, 2900])
def test_pages_whose_heavy_rows_are_zero(dtype, T):
    """In every second page all rows but one hold zeros, and that one has 2^-40 of their weight and values of 2^-85."""
    ops = _ops()
    c = Case([928], 1, 64, 32, 4, "LINEAR", dtype, seed=T)
    rows = torch.arange(928)
    light = (rows // 32 % 2 == 0) & (rows % 32 == 31)
    c.k.zero_()
    c.k[0, ~light, 0, 0] = 48.0
    c.v = torch.where(rows // 32 % 2 == 1, 1.0, torch.where(light, 2.0 ** -85, 0.0))[None, :, None, None].expand(1, 928, 1, 64).to(dtype).contiguous()
    _rewrite(c, "LINEAR")
    q = torch.zeros(1, T, 1, 64, dtype=dtype)
    q[..., 0] = 1.0
    s = float(np.float32(40 * math.log(2) / 48))
    sel, seen = _choices(c, T, 16)
    out, lse = ops.bank_attend_pages(c.bank, c.table, c.length, q.to(c.dev), sel, s, want_lse=True)
    c.check(q, out, lse, s, seen)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [40, 2900])
def test_columns_of_unlike_size_keep_their_precision(dtype, T):
    """Values of a few in columns 0 .. 31 and 2^-30 of that in the others, by pages and over the whole bank."""
    ops = _ops()
    c = Case([900], 1, 64, 32, 4, "RBF", dtype, seed=T + 1)
    c.v[..., 32:] *= 2.0 ** -30
    _rewrite(c)
    q, qd = c.queries(T, 1, dtype)
    sel, seen = _choices(c, T, 16)
    out, lse = ops.bank_attend_pages(c.bank, c.table, c.length, qd, sel, 0.25, want_lse=True)
    c.check(q, out, lse, 0.25, seen)
    out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, 0.25, want_lse=True)
    c.check(q, out, lse, 0.25, lambda b, t, h: np.ones(900, bool))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [3, 20, 100])
def test_columns_at_both_ends_of_the_range(dtype, T):
    """Sums past float32's range in columns 0 .. 31, values of 2^-108 in the others."""
    ops = _ops()
    c = Case([900], 1, 64, 32, 4, "RBF", dtype, seed=T)
    n = torch.as_tensor(c.rng.integers(1, 3, size=(1, 900, 1, 64))).double()
    c.v = torch.cat([(n[..., :32] * 1.25e38), n[..., 32:] * 2.0 ** -108], -1).to(dtype)
    _rewrite(c)
    q, qd = c.queries(T, 1, dtype)
    out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, 0.25, want_lse=True)
    c.check(q, out, lse, 0.25, lambda b, t, h: np.ones(900, bool))


@pytest.mark.parametrize("T,whole", [(1, True), (3, True), (30, True), (40, False), (2900, False)])
def test_weights_of_bf16_callers_keep_16_bits_where_few_ask_or_pages_are_chosen(T, whole, monkeypatch):
    """The general bound with 2^-16 in place of 2^-8 for the weights; means of signed values, so that they are smaller than A."""
    import test_gpu_bank
    monkeypatch.setitem(test_gpu_bank.U_W, BF16, 2.0 ** -16)
    ops = _ops()
    c = Case([900], 1, 64, 32, 4, "RBF", BF16, seed=T + 2)
    q, qd = c.queries(T, 1, BF16)
    if whole:
        out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, 0.25, want_lse=True)
        c.check(q, out, lse, 0.25, lambda b, t, h: np.ones(900, bool))
    sel, seen = _choices(c, T, 4 if T < 40 else 16)
    out, lse = ops.bank_attend_pages(c.bank, c.table, c.length, qd, sel, 0.25, want_lse=True)
    c.check(q, out, lse, 0.25, seen)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D", [32, 128, 192])
def test_many_queries_of_the_other_numbers_of_columns(dtype, bits, D):
    """More than 32 columns of a bank head, so that a tile is shared by the waves of a workgroup."""
    ops = _ops()
    c = Case([300, 7], 1, D, 32, bits, "RBF", dtype, seed=D)
    q, qd = c.queries(70, 2, dtype)
    s = float(np.float32(1.0 / math.sqrt(D)))
    skip, sd = _skips(2, 70, c.lengths, c.rng, c.dev)
    out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, s, skip=sd, want_lse=True)

    def seen(b, t, h):
        r = np.arange(c.lengths[b])
        return ~((r >= skip[b, t, 0]) & (r < skip[b, t, 1]))
    c.check(q, out, lse, s, seen)


# ------------------------------------------------------------ the screen of bank_select
def _screened(c, qd, n_sel):
    """bank_select through the library with a workspace of our own: the choice, and how many candidates the screen left each query
    (-1: more than it keeps, -2: the choice was clear)."""
    import ctypes
    from super_resolution_amd import _lib
    ops, lib = _ops(), _lib.load()
    ref, H, D = ops._bank(c.bank, c.dev.index)
    B, T, Hq, _ = qd.shape
    J, code = c.table.shape[1], {BF16: 0, F16: 1, F32: 2}[qd.dtype]
    n = lib.gpsr_bank_select_workspace_bytes(ref, B, J, T, Hq, n_sel, code)
    assert n > 0, "not screened"
    ws = torch.zeros(n, dtype=torch.uint8, device=c.dev)
    sel = torch.empty(B, T, H, n_sel, dtype=torch.int32, device=c.dev)
    st = (ctypes.c_int64 * 3)(*qd.stride()[:3])
    _lib.check(lib.gpsr_bank_select(ref, c.table.data_ptr(), B, J, c.length.data_ptr(), qd.data_ptr(), code, T, Hq, st, n_sel, None,
                                    sel.data_ptr(), ws.data_ptr(), n, ops._stream()), "gpsr_bank_select")
    # the workspace ends with a count for each query and, aligned to 256 bytes, the candidates: 64 for n_sel <= 16
    up = lambda x: -(-x // 256) * 256
    at = n - up(B * T * H * 64 * 4) - up(B * T * H * 4)
    return sel, ws[at:at + B * T * H * 4].view(torch.int32)


@pytest.mark.parametrize("kernel", ["RBF", "LINEAR"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pages_that_are_not_numbers_do_not_blind_the_screen(dtype, kernel):
    """A NaN in the keys of a few pages: they are not chosen, and the others are told apart as without them."""
    ops = _ops()
    c = Case([16 * 700], 1, 64, 16, 4, kernel, dtype, seed=12)
    q, qd = c.queries(1300, 1, dtype)
    bad = c.rng.choice(700, 6, replace=False)
    for j in bad:
        c.k[0, j * 16 + 5, 0, 3] = math.nan
    ops.bank_write(c.bank, c.table, torch.zeros_like(c.length), c.length, c.k.to(c.dev), c.v.to(c.dev))
    sel, count = _screened(c, qd, 16)
    assert not np.isin(sel.cpu().numpy(), bad).any() and (sel >= 0).all()
    assert float((count == -1).float().mean()) < 0.01
    far = c.bank.centroid.clone()
    gone = torch.as_tensor(c.table_np[0, bad].astype(np.int64)).to(c.dev)
    # the same choice as from a table without these pages
    table = c.table.clone()
    table[0, torch.as_tensor(bad.astype(np.int64)).to(c.dev)] = -1
    assert torch.equal(sel, ops.bank_select(c.bank, table, c.length, qd, 16)) and torch.isnan(far[gone]).any()


# ------------------------------------------------------------ keys past the range, queries that are not numbers
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bits", [4, 8])
def test_keys_past_the_range_have_no_weight(dtype, bits):
    """RBF keys whose |k|^2 / 2 is past float32's range, and queries for which q.k is as well."""
    ops = _ops()
    for T in (3, 20, 100, 2900):
        c = Case([900], 1, 64, 32, bits, "RBF", F32, seed=T)
        huge = np.zeros(900, bool)
        huge[[0, 17, 33, 34, 500, 899]] = True
        sign = torch.as_tensor(c.rng.choice([-1.0, 1.0], size=(1, 6, 1, 64))).float()
        sign[:, ::2] = 1.0
        c.k[:, huge] = sign * 2.9e38
        ops.bank_write(c.bank, c.table, torch.zeros_like(c.length), c.length, c.k.to(c.dev), c.v.to(c.dev))
        assert int(torch.isinf(c.bank.offset).sum()) == 6
        c.k[:, huge] = 0
        c.hk, c.hv = held(c.k.double().numpy(), bits), held(c.v.double().numpy(), bits)
        c.o = -0.5 * (c.hk ** 2).sum(-1)
        q, _ = c.queries(T, 1, dtype)
        q[0, 0], q[0, 1], q[0, 2] = 0, 1, 4
        qd = q.to(c.dev)
        out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, 0.25, want_lse=True)
        c.check(q[:, :100], out[:, :100], lse[..., :100], 0.25, lambda b, t, h: ~huge)
        sel, seen = _choices(c, T, 16)
        out, lse = ops.bank_attend_pages(c.bank, c.table, c.length, qd, sel, 0.25, want_lse=True)
        c.check(q[:, :100], out[:, :100], lse[..., :100], 0.25, lambda b, t, h: seen(b, t, h) & ~huge)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T", [2, 20, 100, 6000])
def test_queries_that_are_not_numbers_and_see_no_row(dtype, T):
    """Zeros and -inf for whoever sees no row, whatever the query holds; NaN for such a query that does see one; nothing for others."""
    ops = _ops()
    c = Case([75], 1, 64, 16, 4, "RBF", dtype, seed=3)
    q, _ = c.queries(T, 1, dtype)
    q[0, 0], q[0, 1, 0, ::2] = math.nan, math.inf
    qd = q.to(c.dev)
    skip = torch.zeros(1, T, 2, dtype=torch.int32, device=c.dev)
    skip[0, :2, 1] = 75                                    # all rows, and none behind them
    pages = torch.arange(5, dtype=torch.int32, device=c.dev).expand(1, T, 1, 5).repeat(1, 1, 1, 3)
    gone = torch.full_like(c.table, -1)
    gone[0, 0] = c.table[0, 0]
    first = torch.tensor([[[0, 16]]], dtype=torch.int32, device=c.dev).expand(1, T, 2).contiguous()
    for table, sk, none in ((c.table, skip, 2), (torch.full_like(c.table, -1), None, T), (gone, first, T)):
        for out, lse in (ops.bank_attend(c.bank, table, c.length, qd, 0.25, skip=sk, want_lse=True),
                         ops.bank_attend_pages(c.bank, table, c.length, qd, pages, 0.25, skip=sk, want_lse=True)):
            assert not out[:, :none].any() and (lse[..., :none] == -math.inf).all()
            assert torch.isfinite(out).all() and torch.isfinite(lse[..., none:]).all()
    for out, lse in (ops.bank_attend(c.bank, c.table, c.length, qd, 0.25, want_lse=True),
                     ops.bank_attend_pages(c.bank, c.table, c.length, qd, pages, 0.25, want_lse=True)):
        assert torch.isnan(out[:, :2]).all() and torch.isnan(lse[..., :2]).all() and torch.isfinite(out[:, 2:]).all()


def test_float32_queries_at_the_end_of_their_range():
    """A query that a bf16 term does not reach (above 2^128 - 2^119): keys of 2^-100 bring its logits back."""
    ops = _ops()
    c = Case([300], 1, 64, 16, 8, "LINEAR", F32, seed=6)
    c.k *= 2.0 ** -100
    _rewrite(c, "LINEAR")
    q = torch.full((1, 40, 1, 64), torch.finfo(F32).max)
    q[0, ::2] *= -1
    out, lse = ops.bank_attend(c.bank, c.table, c.length, q.to(c.dev), 2.0 ** -27, want_lse=True)
    c.check(q, out, lse, 2.0 ** -27, lambda b, t, h: np.ones(300, bool))


# ------------------------------------------------------------ many calls at once and again
def test_two_streams_at_once_with_many_queries():
    """Enough queries for the screen and for the way by page, whose lists and partials lie in a workspace."""
    ops = _ops()
    T = 4500
    cs = [Case([12000], 1, 64, 64, 4, "RBF", BF16, seed=40 + i) for i in range(2)]
    qs = [c.queries(T, 1, BF16)[1] for c in cs]
    for c, q in zip(cs, qs):
        _screened(c, q, 8)
        assert _pages_workspace(c, T, 1, 8, BF16) > 0

    def run(c, q):
        sel = ops.bank_select(c.bank, c.table, c.length, q, 8)
        return (sel, *ops.bank_attend_pages(c.bank, c.table, c.length, q, sel, 0.2, want_lse=True))
    want = [run(c, q) for c, q in zip(cs, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(cs[i], qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_agpr_with_a_bank_by_page(tmp_path, golden_dir, monkeypatch):
    """1564 windows with 16 pages of 64 rows each go by page; fewer pages would go by query."""
    import test_gpu_agpr_bank
    from super_resolution_amd import _lib, ops
    ref, _, _ = ops._bank(ops.bank_alloc(47, 1, 64), torch.cuda.current_device())
    size = _lib.load().gpsr_bank_attend_pages_workspace_bytes
    assert size(ref, 1, 47, 1564, 1, 16, 0) > 0 and size(ref, 1, 47, 1564, 1, 4, 0) == 0
    test_gpu_agpr_bank.test_agpr_with_a_bank_runs_as_its_definition(tmp_path, golden_dir, monkeypatch, 16)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_many_columns_are_the_same_every_time_in_the_other_ways_too(dtype):
    """Banks shared out and joined, pages by query, and the choice by the screen and without it: every bit the same."""
    ops = _ops()
    c = Case([5003], 1, 32, 16, 4, "RBF", dtype, seed=9)
    q, qd = c.queries(20000, 1, dtype)

    def calls():
        yield ops.bank_attend(c.bank, c.table, c.length, qd, 0.2, want_lse=True)
        sel = ops.bank_select(c.bank, c.table, c.length, qd, 8)
        yield (sel,)
        yield (torch.cat([ops.bank_select(c.bank, c.table, c.length, qd[:, t:t + 500], 8) for t in range(0, 20000, 500)], 1),)
        for t in range(0, 2000, 200):
            yield ops.bank_attend_pages(c.bank, c.table, c.length, qd[:, t:t + 200], sel[:, t:t + 200].contiguous(), 0.2, want_lse=True)
        for t in range(0, 3000, 20):
            yield ops.bank_attend(c.bank, c.table, c.length, qd[:, t:t + 20], 0.2, want_lse=True)
    first = list(calls())
    assert torch.equal(first[1][0], first[2][0])
    for _ in range(3):
        for a, b in zip(first, calls()):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------ refusals
def test_rows_and_queries_that_ask_for_gradients_are_refused():
    from super_resolution_amd import _lib
    from super_resolution_amd.bank import ExampleBank
    ops = _ops()
    c = Case([100], 1, 64, 16, 4, "RBF", F32, seed=1)
    q = c.queries(3, 1, F32)[1].requires_grad_()
    k, v = c.k.to(c.dev), c.v.to(c.dev)
    sel = torch.zeros(1, 3, 1, 4, dtype=torch.int32, device=c.dev)
    img = torch.zeros(9, 9, dtype=torch.float64, device=c.dev)
    rows = torch.zeros(1, 9, 1, 64, device=c.dev)
    b = ExampleBank(100, 49).append(k[0, :, 0, :49], v[0, :, 0, :49])
    calls = [lambda: ops.bank_attend(c.bank, c.table, c.length, q, 1.0), lambda: ops.bank_select(c.bank, c.table, c.length, q, 2),
             lambda: ops.bank_attend_pages(c.bank, c.table, c.length, q, sel, 1.0), lambda: b.predict(q[0, :, 0, :49], 1.0),
             lambda: ops.bank_write(c.bank, c.table, torch.zeros_like(c.length), c.length, k.clone().requires_grad_(), v),
             lambda: ops.bank_write(c.bank, c.table, torch.zeros_like(c.length), c.length, k, v.clone().requires_grad_()),
             lambda: ops.bank_windows(img.clone().requires_grad_(), 7, 64), lambda: ops.bank_blend(img.clone().requires_grad_(), rows, 7),
             lambda: ops.bank_blend(img, rows.clone().requires_grad_(), 7)]
    for i, f in enumerate(calls):
        with pytest.raises(_lib.GpsrError, match="gradients"):
            f()
            pytest.fail(f"call {i} was not refused")
        with torch.no_grad():
            f()


def test_numbers_of_rows_that_a_read_cannot_have_are_refused():
    from super_resolution_amd import _lib
    ops = _ops()
    c = Case([100], 1, 32, 16, 4, "RBF", F32, seed=1)
    for rows in (-1, 2 ** 31, 2 ** 32 + 5):
        with pytest.raises(_lib.GpsrError, match="rows"):
            ops.bank_read(c.bank, c.table, torch.zeros_like(c.length), c.length, rows, BF16)


def test_choose_scale_passes_over_what_is_not_a_number_and_refuses_an_empty_bank():
    """One example whose value is NaN, seen by every query in 32 columns: the others decide, as without it."""
    from super_resolution_amd import _lib
    from super_resolution_amd.bank import ExampleBank
    rng = np.random.default_rng(4)
    dev = torch.device("cuda", torch.cuda.current_device())
    k = torch.as_tensor(rng.normal(size=(700, 49)).astype(np.float32)).to(dev) * 0.2
    v = torch.tanh(k @ torch.as_tensor(rng.normal(size=(49, 49)).astype(np.float32) * 0.25).to(dev))
    assert ExampleBank(700, 49, bits=8).append(k, v).choose_scale([1e-6, 5.0], sample=300) == 5.0
    v[333, 40] = math.nan
    assert ExampleBank(700, 49, bits=8).append(k, v).choose_scale([1e-6, 5.0], sample=300) == 5.0
    for b in (ExampleBank(10, 49), ExampleBank(700, 49).append(k, torch.full_like(v, math.nan))):
        with pytest.raises(_lib.GpsrError, match="numbers"):
            b.choose_scale([1.0, 2.0])


def test_example_bank_reads_from_its_first_row_on():
    from super_resolution_amd import _lib
    from super_resolution_amd.bank import ExampleBank
    dev = torch.device("cuda", torch.cuda.current_device())
    k = torch.ones(10, 49, device=dev)
    b = ExampleBank(20, 49).append(k, k)
    with pytest.raises(_lib.GpsrError, match="from 0"):
        b.read(-5, 10)
    for start, rows in ((4, 6), (9, 1), (10, 0), (25, 0)):
        got = b.read(start, 8)
        assert all((x[:rows] == 1).all() and not x[rows:].any() and len(x) == 8 for x in got)
