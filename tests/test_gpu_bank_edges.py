"""Example bank at its edges: pages and columns of unlike size, keys past the range, queries that are not numbers, rows that are
not there, the ways that only many queries take.  Definitions and bounds as in test_gpu_bank.py."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_bank import BF16, F16, F32, Case, _ops, held


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
