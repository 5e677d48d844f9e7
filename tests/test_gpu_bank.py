"""Example bank (include/gpsr.h gpsr_bank_*): every entry point against its definition in 64 bits.

Bounds, fixed before the first run.  u(t) = finfo(t).eps / 2 is the half step of a type, e = 2^-23 the rounding of one
32-bit operation whichever way it rounds.  A logit x = s (q.k + o) is a 32-bit sum of dim products and o, so it is off by
at most E = e ((dim + 4) s max(sum |q_i k_i| + |o|) + 2); weights are off by 2 E relatively once normalised, their sum of
n terms by n e; weights enter the second product rounded to u(w): bf16 queries 2^-9 .. one bf16 term, half a step 2^-8;
f16 queries two terms, 2^-16; f32 three, 2^-24.  With A = sum w |v| / sum w:
    |out - exact| <= u(t) |exact| + (u(w) + 2 E + 2 n e) A        |lse - exact| <= E + (n + 4) e + 2 e |exact|
Held values, offsets, centroids and chosen pages have to be equal."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 2.0 ** -23
U_W = {BF16: 2.0 ** -8, F16: 2.0 ** -16, F32: 2.0 ** -24}


def _ops():
    from super_resolution_amd import ops
    return ops


# ------------------------------------------------------------ the definition, in numpy and 64 bits
def _grid(bits):
    if bits == 4:
        return np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
    return np.array([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def held(x, bits):
    """[..., D] float64 -> the values that the bank holds."""
    grid, lo, hi = _grid(bits), -110, 125 if bits == 4 else 119
    mid = (grid[1:] + grid[:-1]) / 2
    g = x.reshape(*x.shape[:-1], -1, 32)
    out = np.empty_like(g)
    with np.errstate(invalid="ignore"):
        bad = ~np.isfinite(g).all(-1)
        top = np.where(bad, 0.0, np.abs(g).max(-1))
        m, e = np.frexp(top / grid[-1])
        e = np.where(m == 0.5, e - 1, e)                      # smallest e with top <= grid[-1] 2^e
        e = np.clip(np.where(top == 0, lo, e), lo, hi)
        unit = np.ldexp(1.0, e)[..., None]
        a = np.where(bad[..., None], 0.0, np.abs(g)) / unit
        left, right = np.searchsorted(mid, a, "left"), np.searchsorted(mid, a, "right")
        out = np.copysign(grid[np.where(left % 2 == 0, left, right)] * unit, g)
    out[bad] = np.nan
    return out.reshape(x.shape)


def softmax_mean(q, k, o, v, ok, s):
    """q [D], k [n,D], o [n], v [n,D], ok [n] -> exact out, lse, A, max of sum |q_i k_i| + |o|, n."""
    k, o, v = k[ok], o[ok], v[ok]
    if not len(k):
        return np.zeros(len(q)), -math.inf, np.zeros(len(q)), 0.0, 0
    x = s * (k @ q + o)
    m = x.max()
    w = np.exp(x - m)
    return w @ v / w.sum(), m + math.log(w.sum()), w @ np.abs(v) / w.sum(), float((np.abs(k) @ np.abs(q) + np.abs(o)).max()), len(k)


# ------------------------------------------------------------ a bank with its contents in 64 bits
class Case:
    """Banks of the given lengths over shuffled pages, written by bank_write; keys / values / offsets as held, per entry."""

    def __init__(self, lengths, H=1, D=64, P=16, bits=4, kernel="RBF", dtype=F32, seed=0, spare=3, gain=0.5, poison=True):
        ops = _ops()
        rng = np.random.default_rng(seed)
        self.P, self.H, self.D, self.bits, self.lengths = P, H, D, bits, lengths
        B, T = len(lengths), max(max(lengths), 1)
        per = [-(-n // P) for n in lengths]
        J = max(max(per), 1) + 1
        pages = sum(per) + spare
        place = rng.permutation(pages)
        table = np.full((B, J), -1, np.int32)
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = place[at:at + n]
            at += n
        self.table_np = table
        dev = torch.device("cuda", torch.cuda.current_device())
        self.dev = dev
        self.bank = ops.bank_alloc(pages, H, D, P, bits, getattr(ops, kernel))
        if poison:      # what no row covers holds not-a-numbers
            for t in self.bank[:4]:
                t.fill_(255)
            self.bank.offset.fill_(math.nan)
            self.bank.centroid.fill_(math.nan)
        self.table = torch.as_tensor(table).to(dev)
        self.length = torch.tensor(lengths, dtype=torch.int32, device=dev)
        self.k = torch.as_tensor(rng.normal(size=(B, T, H, D)) * gain).to(dtype)
        self.v = torch.as_tensor(rng.normal(size=(B, T, H, D))).to(dtype)
        ops.bank_write(self.bank, self.table, torch.zeros_like(self.length), self.length, self.k.to(dev), self.v.to(dev))
        self.hk, self.hv = held(self.k.double().numpy(), bits), held(self.v.double().numpy(), bits)
        self.o = -0.5 * (self.hk ** 2).sum(-1) if kernel == "RBF" else np.zeros(self.hk.shape[:-1])
        self.rng = rng

    def queries(self, T, G, dtype, gain=0.5):
        q = torch.as_tensor(self.rng.normal(size=(len(self.lengths), T, self.H * G, self.D)) * gain).to(dtype)
        return q, q.to(self.dev)

    def check(self, q, out, lse, s, visible):
        """visible(b, t, h) -> bool [length[b]]."""
        B, T, Hq, D = q.shape
        qd, got, gl = q.double().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
        u, uw = torch.finfo(out.dtype).eps / 2, U_W[out.dtype]
        for b in range(B):
            n = self.lengths[b]
            for t in range(T):
                for hq in range(Hq):
                    h = hq // (Hq // self.H)
                    want, wl, A, big, m = softmax_mean(qd[b, t, hq], self.hk[b, :n, h], self.o[b, :n, h], self.hv[b, :n, h], visible(b, t, h), s)
                    E = EPS * ((D + 4) * s * big + 2)
                    bound = u * np.abs(want) + (uw + 2 * E + 2 * m * EPS) * A
                    err = np.abs(got[b, t, hq] - want)
                    assert (err <= bound).all(), (b, t, hq, float((err / np.maximum(bound, 1e-300)).max()))
                    if m == 0:
                        assert gl[b, hq, t] == -math.inf
                    else:
                        assert abs(gl[b, hq, t] - wl) <= E + (m + 4) * EPS + 2 * EPS * abs(wl), (b, t, hq, gl[b, hq, t], wl)


def _skips(B, T, lengths, rng, dev):
    lo = rng.integers(0, max(lengths) + 1, (B, T))
    hi = lo + rng.integers(0, max(lengths) + 1, (B, T))
    lo[:, 0], hi[:, 0] = 0, max(lengths) + 5        # the first query sees nothing
    if T > 1:
        lo[:, 1], hi[:, 1] = 5, 2                   # an empty range
    if T > 2:
        lo[:, 2], hi[:, 2] = -7, 2 ** 31 - 1        # everything, by a range beyond the bank
    a = np.stack([lo, hi], -1).astype(np.int32)
    return a, torch.as_tensor(a).to(dev)


# ------------------------------------------------------------ write and read
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,P,H", [(32, 16, 1), (64, 64, 2), (96, 32, 1), (128, 16, 3), (192, 64, 1), (256, 256, 1)])
def test_write_holds_the_nearest_values_and_read_returns_them(bits, dtype, D, P, H):
    ops = _ops()
    c = Case([P + 5, 1, 3 * P, 0], H, D, P, bits, dtype=dtype, seed=D + bits, gain=1.0)
    start = torch.zeros_like(c.length)
    k, v = ops.bank_read(c.bank, c.table, start, c.length, 3 * P + 2, dtype)
    assert k.shape == v.shape == (4, 3 * P + 2, H, D) and k.dtype == dtype
    for b, n in enumerate(c.lengths):
        for got, want in ((k, c.hk), (v, c.hv)):
            assert torch.equal(got[b, :n].cpu(), torch.as_tensor(want[b, :n]).to(dtype))
            assert not got[b, n:].any()
    off, cent = c.bank.offset.cpu(), c.bank.centroid.cpu()
    for b, n in enumerate(c.lengths):
        for j in range(-(-n // P)):
            page, rows = c.table_np[b, j], range(j * P, min(n, (j + 1) * P))
            assert torch.equal(off[page, :, :len(rows)], torch.as_tensor(c.o[b, rows]).float().T)
            mean = c.hk[b, rows].sum(0) / len(rows)
            assert torch.equal(cent[page], torch.as_tensor(mean).float())


@pytest.mark.parametrize("bits", [4, 8])
def test_write_range_of_values(bits):
    """Ties, signed zeros, subnormal and huge values, the borders of a scale, one bad value in a group."""
    ops = _ops()
    grid = _grid(bits)
    mids = (grid[1:] + grid[:-1]) / 2
    rows = []
    for top in (6.0, 448.0, 6.0000005, 447.99997, 0.75, 1.0, 3.0e38, 1.2e-38, 2.0 ** -120, 2.0 ** -140):
        r = np.zeros(64)
        vals = np.resize(np.concatenate([mids[:15], -mids[-15:], grid[-4:]]) / grid[-1] * top, 31)
        r[0], r[1:32], r[32], r[33:] = top, vals, -top, -vals[::-1]
        rows.append(r)
    rows += [np.zeros(64), -np.zeros(64)]
    for bad in (np.nan, np.inf, -np.inf):
        r = np.linspace(-1, 1, 64)
        r[40] = bad
        rows.append(r)
    x = torch.as_tensor(np.array(rows)).to(F32)
    n = len(x)
    bank = ops.bank_alloc(2, 1, 64, 16, bits, ops.LINEAR)
    dev = bank.offset.device
    table = torch.tensor([[1]], dtype=torch.int32, device=dev)
    one = lambda i: torch.tensor([i], dtype=torch.int32, device=dev)
    xd = x.to(dev).view(1, n, 1, 64)
    ops.bank_write(bank, table, one(0), one(n), xd, -xd)
    k, v = ops.bank_read(bank, table, one(0), one(n), n, F32)
    want = torch.as_tensor(held(x.double().numpy(), bits)).float()
    assert torch.equal(torch.nan_to_num(k.cpu().view(n, 64), nan=1e30), torch.nan_to_num(want, nan=1e30))
    assert torch.equal(torch.nan_to_num(v.cpu().view(n, 64), nan=1e30), torch.nan_to_num(-want, nan=1e30))
    assert torch.isnan(k.cpu().view(n, 2, 32)[-3:, 1]).all() and torch.isfinite(k.cpu().view(n, 2, 32)[-3:, 0]).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_append_in_steps_equals_one_write_and_touches_nothing_else(bits):
    ops = _ops()
    c = Case([77, 40], 2, 64, 32, bits, seed=3, poison=False)
    twin = ops.Bank(*[t.clone().zero_() for t in c.bank[:6]], bits, ops.RBF)
    k, v = c.k.to(c.dev), c.v.to(c.dev)
    at = np.zeros(2, np.int32)
    for step in (1, 1, 5, 31, 0, 39):
        n = np.minimum(step, np.array(c.lengths) - at).astype(np.int32)
        rows = max(int(n.max()), 1)
        kk, vv = torch.zeros(2, rows + 3, 4, 64, device=c.dev), torch.zeros(2, rows + 3, 4, 64, device=c.dev)
        for b in range(2):          # rows of a wider buffer, every second head: strides of their own
            kk[b, :n[b], ::2], vv[b, :n[b], ::2] = k[b, at[b]:at[b] + n[b]], v[b, at[b]:at[b] + n[b]]
        ops.bank_write(twin, c.table, torch.as_tensor(at).to(c.dev), torch.as_tensor(n).to(c.dev), kk[:, :rows, ::2], vv[:, :rows, ::2])
        at += n
    for a, b in zip(twin[:6], c.bank[:6]):
        assert torch.equal(a, b)
    # nothing of an entry with count 0, a negative start, a page that does not exist, or a position behind the table
    before = [t.clone() for t in twin[:6]]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=c.dev)
    big = torch.full((2, 8, 2, 64), 9.0, device=c.dev)
    ops.bank_write(twin, c.table, i32(0, -3), i32(0, 8), big, big)
    ops.bank_write(twin, torch.full_like(c.table, -1), i32(0, 0), i32(8, 8), big, big)
    ops.bank_write(twin, torch.full_like(c.table, 10 ** 6), i32(0, 0), i32(8, 8), big, big)
    ops.bank_write(twin, c.table, i32(c.table.shape[1] * 32, 2 ** 31 - 4), i32(8, 8), big, big)
    assert all(torch.equal(a, b) for a, b in zip(before, twin[:6]))
    rk, rv = ops.bank_read(twin, c.table, i32(-1, 2 ** 31 - 4), i32(8, 8), 8)
    assert not rk.any() and not rv.any()


def test_unaligned_rows_are_read_element_by_element():
    ops = _ops()
    for dtype in (BF16, F16, F32):
        c = Case([37], 1, 64, 16, 4, dtype=dtype, seed=11)
        flat = torch.zeros(37 * 67 + 1, dtype=dtype, device=c.dev)
        kk = flat[1:].as_strided((1, 37, 1, 64), (37 * 67, 67, 67, 1))
        kk.copy_(c.k)
        twin = ops.Bank(*[t.clone() for t in c.bank[:6]], 4, ops.RBF)
        ops.bank_write(twin, c.table, torch.zeros_like(c.length), c.length, kk, c.v.to(c.dev))
        assert all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())) for a, b in zip(c.bank[:6], twin[:6]))
        q, qd = c.queries(5, 1, dtype)
        buf = torch.zeros(5 * 65 + 1, dtype=dtype, device=c.dev)[1:].as_strided((1, 5, 1, 64), (325, 65, 65, 1))
        buf.copy_(q)
        assert torch.equal(ops.bank_attend(c.bank, c.table, c.length, buf, 0.3), ops.bank_attend(c.bank, c.table, c.length, qd, 0.3))
        assert torch.equal(ops.bank_select(c.bank, c.table, c.length, buf, 2), ops.bank_select(c.bank, c.table, c.length, qd, 2))


# ------------------------------------------------------------ attention over the bank
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D,P,H,G,T,lengths", [
    (64, 16, 1, 1, 1, [1, 0, 33]), (64, 64, 1, 1, 67, [200, 64, 63]), (32, 32, 2, 2, 5, [65, 3]), (96, 16, 1, 3, 33, [130]),
    (128, 64, 2, 4, 3, [515, 1]), (192, 32, 1, 1, 9, [100]), (256, 128, 1, 2, 20, [300, 7])])
def test_attend(dtype, bits, D, P, H, G, T, lengths):
    ops = _ops()
    for kernel, s in (("RBF", 1.5 / math.sqrt(D)), ("LINEAR", 4.0 / math.sqrt(D))):
        c = Case(lengths, H, D, P, bits, kernel, dtype, seed=D + T)
        q, qd = c.queries(T, G, dtype)
        out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, s, want_lse=True)
        s = float(np.float32(s))
        c.check(q, out, lse, s, lambda b, t, h: np.ones(lengths[b], bool))
        skip, sd = _skips(len(lengths), T, lengths, c.rng, c.dev)
        out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, s, skip=sd, want_lse=True)

        def seen(b, t, h):
            r = np.arange(lengths[b])
            return ~((r >= skip[b, t, 0]) & (r < skip[b, t, 1]))
        c.check(q, out, lse, s, seen)
        assert torch.equal(out, ops.bank_attend(c.bank, c.table, c.length, qd, s, skip=sd))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,G,n", [(1, 1, 9001), (2, 8, 5003), (300, 1, 1500), (1, 40, 4097)])
def test_attend_long(dtype, T, G, n):
    """Banks long enough to be shared between workgroups, and enough queries for several of them."""
    ops = _ops()
    c = Case([n, n // 3, 0], 1, 64, 64, 4, "RBF", dtype, seed=n)
    q, qd = c.queries(T, G, dtype)
    out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, 0.25, want_lse=True)
    c.check(q, out, lse, 0.25, lambda b, t, h: np.ones(c.lengths[b], bool))


def test_attend_peaks_and_far_queries():
    """Weights between one-hot and flat; logits of some thousands; a query far from every example."""
    ops = _ops()
    for dtype in (BF16, F16, F32):
        c = Case([500], 1, 64, 32, 8, "RBF", dtype, seed=5, gain=1.0)
        q, _ = c.queries(6, 1, dtype, gain=1.0)
        q[0, 0] = torch.as_tensor(c.hk[0, 123]).to(dtype)
        q[0, 1] *= 60
        q[0, 2] = 0
        qd = q.to(c.dev)
        for s in (1e-4, 0.5, 40.0):
            out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, s, want_lse=True)
            c.check(q, out, lse, float(np.float32(s)), lambda b, t, h: np.ones(500, bool))


def test_not_a_number_rows_matter_only_to_those_who_see_them():
    ops = _ops()
    c = Case([90], 1, 64, 16, 4, "RBF", F32, seed=8)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=c.dev)
    bad = torch.full((1, 1, 1, 64), math.nan, device=c.dev)
    ops.bank_write(c.bank, c.table, i32(41), i32(1), bad, bad)
    # the write ended entry 0's page 2 at row 41: what lay behind is written again
    ops.bank_write(c.bank, c.table, i32(42), i32(48), c.k[:, 42:].to(c.dev), c.v[:, 42:].to(c.dev))
    q, qd = c.queries(2, 1, F32)
    skip = torch.tensor([[[41, 42], [0, 0]]], dtype=torch.int32, device=c.dev)
    for f in (lambda: ops.bank_attend(c.bank, c.table, c.length, qd, 0.5, skip=skip, want_lse=True),
              lambda: ops.bank_attend_pages(c.bank, c.table, c.length, qd, torch.arange(6, dtype=torch.int32, device=c.dev).expand(1, 2, 1, 6).contiguous(),
                                            0.5, skip=skip, want_lse=True)):
        out, lse = f()
        assert torch.isnan(out[0, 1]).all() and torch.isnan(lse[0, 0, 1])
        r = np.arange(90)
        c.check(q[:, :1], out[:, :1], lse[:, :, :1], 0.5, lambda b, t, h: r != 41)


def test_pages_that_do_not_exist_are_passed_over():
    ops = _ops()
    for dtype in (BF16, F32):
        c = Case([150, 40], 1, 64, 16, 4, "RBF", dtype, seed=9)
        c.table[0, 3], c.table[0, 5], c.table[1, 0] = -1, 10 ** 6, -2 ** 31
        q, qd = c.queries(40, 1, dtype)
        gone = {0: (3, 5), 1: (0,)}
        seen = lambda b, t, h: ~np.isin(np.arange(c.lengths[b]) // 16, gone[b])
        far = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device=c.dev)
        out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, 0.5, want_lse=True)
        c.check(q, out, lse, 0.5, seen)
        sel = torch.arange(-2, 12, dtype=torch.int32, device=c.dev).expand(2, 40, 1, 14).contiguous()
        out, lse = ops.bank_attend_pages(c.bank, c.table, c.length, qd, sel, 0.5, want_lse=True)
        c.check(q, out, lse, 0.5, seen)
        picked = ops.bank_select(c.bank, c.table, c.length, qd, 16).cpu()
        assert not np.isin(picked[0].numpy(), (3, 5)).any() and not (picked[1] == 0).any()
        # lengths beyond the table end with it, negative ones are empty
        out, lse = ops.bank_attend(c.bank, c.table[:, :2].contiguous(), far, qd, 0.5, want_lse=True)
        c.check(q[:1], out[:1], lse[:1], 0.5, lambda b, t, h: np.arange(150) < 32)
        assert not out[1].any() and torch.isinf(lse[1]).all()


# ------------------------------------------------------------ page choice
def _select_exact(c, q, n_sel, skip=None, rbf=True):
    B, T, Hq, D = q.shape
    G = Hq // c.H
    cent = c.bank.centroid.double().cpu().numpy()
    qd = q.double().numpy()
    out = np.full((B, T, c.H, n_sel), -1, np.int32)
    for b in range(B):
        n = c.lengths[b]
        for t in range(T):
            for h in range(c.H):
                qs = qd[b, t, h * G:(h + 1) * G].sum(0)
                best = []
                for j in range(-(-n // c.P)):
                    lo, hi = j * c.P, min(n, (j + 1) * c.P)
                    if skip is not None and skip[b, t, 0] <= lo and skip[b, t, 1] >= hi:
                        continue
                    ce = cent[c.table_np[b, j], h]
                    best.append((-(qs @ ce - (G * (ce @ ce) / 2 if rbf else 0.0)), j))
                chosen = sorted(j for _, j in sorted(best)[:n_sel])
                out[b, t, h, :len(chosen)] = chosen
    return out


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,P,H,G,T,n_sel,lengths", [
    (64, 16, 1, 1, 1, 4, [700, 5, 0]), (64, 16, 1, 1, 70, 16, [1600]), (32, 16, 2, 3, 9, 1, [300, 170]),
    (128, 32, 1, 2, 40, 64, [999]), (96, 16, 1, 1, 17, 7, [333]), (192, 16, 2, 1, 3, 8, [400]), (256, 64, 1, 1, 33, 3, [1030])])
def test_select(dtype, D, P, H, G, T, n_sel, lengths):
    ops = _ops()
    for kernel in ("RBF", "LINEAR"):
        c = Case(lengths, H, D, P, 4, kernel, dtype, seed=D + T + 1)
        q, qd = c.queries(T, G, dtype)
        got = ops.bank_select(c.bank, c.table, c.length, qd, n_sel)
        assert got.dtype == torch.int32
        assert np.array_equal(got.cpu().numpy(), _select_exact(c, q, n_sel, rbf=kernel == "RBF"))
        skip, sd = _skips(len(lengths), T, lengths, c.rng, c.dev)
        got = ops.bank_select(c.bank, c.table, c.length, qd, n_sel, skip=sd)
        assert np.array_equal(got.cpu().numpy(), _select_exact(c, q, n_sel, skip, kernel == "RBF"))


def test_select_many_pages():
    ops = _ops()
    for dtype in (BF16, F32):
        c = Case([16 * 5000 - 3], 1, 32, 16, 4, "RBF", dtype, seed=21)
        q, qd = c.queries(20, 1, dtype)
        got = ops.bank_select(c.bank, c.table, c.length, qd, 32)
        assert np.array_equal(got.cpu().numpy(), _select_exact(c, q, 32))


def test_select_equal_scores_take_the_lower_page():
    """Pages of equal rows have equal centroids: whole runs of ties, and one query of zeros (LINEAR: all scores 0)."""
    ops = _ops()
    c = Case([16 * 300], 1, 64, 16, 4, "LINEAR", F32, seed=2)
    rows = c.k[:, :16].repeat(1, 300, 1, 1)
    rows[:, 16 * 7:16 * 9] *= 2
    ops.bank_write(c.bank, c.table, torch.zeros_like(c.length), c.length, rows.to(c.dev), c.v.to(c.dev))
    for dtype in (BF16, F16, F32):
        q, qd = c.queries(40, 1, dtype)
        q[0, 0] = 0
        qd = q.to(c.dev)
        got = ops.bank_select(c.bank, c.table, c.length, qd, 5).cpu().numpy()
        assert np.array_equal(got, _select_exact(c, q, 5, rbf=False))
        assert np.array_equal(got[0, 0, 0], np.arange(5))


def test_select_near_ties_are_decided_in_64_bits():
    """Scores that differ by less than 32 bits tell apart: one column of the centroids moved by one step at a time."""
    ops = _ops()
    P, n = 16, 200
    c = Case([P * n], 1, 64, P, 8, "LINEAR", F32, seed=4)
    cent = torch.ones(c.bank.centroid.shape[0], 1, 64)
    order = c.rng.permutation(n)
    for j in range(n):
        cent[c.table_np[0, j], 0, 0] = 1.0 + int(order[j]) * 2.0 ** -23
    c.bank.centroid.copy_(cent)
    q = torch.ones(1, 8, 1, 64)
    q[0, :, 0, 1:] = 64.0 * torch.arange(1, 9)[:, None]
    got = ops.bank_select(c.bank, c.table, c.length, q.to(c.dev), 9).cpu().numpy()
    assert np.array_equal(got, _select_exact(c, q, 9, rbf=False))
    assert np.array_equal(got[0, 0, 0], np.sort(np.argsort(-order)[:9]))
    got = ops.bank_select(c.bank, c.table, c.length, q.bfloat16().to(c.dev), 9).cpu().numpy()
    assert np.array_equal(got[0, 3, 0], np.sort(np.argsort(-order)[:9]))


def _select_exact_many(c, q, n_sel, skip=None, rbf=True):
    """The same for many queries: a stable sort by falling score."""
    B, T, Hq, D = q.shape
    G = Hq // c.H
    cent = c.bank.centroid.double().cpu().numpy()
    qd = q.double().numpy().reshape(B, T, c.H, G, D).sum(3)
    out = np.full((B, T, c.H, n_sel), -1, np.int32)
    for b in range(B):
        n = c.lengths[b]
        first = np.arange(-(-n // c.P)) * c.P
        ok = np.ones((T, len(first)), bool)
        if skip is not None:
            ok = ~((skip[b, :, :1] <= first) & (skip[b, :, 1:] >= np.minimum(first + c.P, n)))
        for h in range(c.H):
            ce = cent[c.table_np[b, :len(first)], h]
            # one sum for each score, all in the same order: a matrix product gives equal pages scores that differ in the last bit
            dot = np.stack([(x * ce).sum(-1) for x in qd[b, :, h]])
            score = np.where(ok, dot - (G * (ce * ce).sum(1) / 2 if rbf else 0.0), -np.inf)
            at = np.argsort(-score, axis=1, kind="stable")[:, :n_sel]
            at = np.sort(np.where(np.take_along_axis(score, at, 1) == -np.inf, 2 ** 30, at), 1)
            out[b, :, h, :at.shape[1]] = np.where(at == 2 ** 30, -1, at)
    return out


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,P,H,G,T,n_sel,lengths", [
    (64, 16, 1, 1, 700, 16, [16 * 400 - 3]), (32, 16, 2, 1, 301, 4, [1100, 16 * 70]), (128, 32, 1, 3, 513, 64, [32 * 300]),
    (96, 16, 1, 2, 600, 33, [16 * 3000]), (192, 64, 1, 1, 520, 1, [64 * 80]), (256, 16, 1, 1, 550, 9, [16 * 99 + 1]),
    (64, 16, 1, 1, 1700, 16, [16 * 400 - 3]), (32, 16, 2, 1, 430, 4, [1100, 16 * 70]), (128, 32, 1, 3, 1301, 64, [32 * 300]),
    (192, 64, 1, 1, 1600, 1, [64 * 80]), (256, 16, 1, 1, 1550, 9, [16 * 99 + 1])])
def test_select_for_many_queries(dtype, D, P, H, G, T, n_sel, lengths):
    """Enough queries and pages for the screen in fewer bits: the choice has to stay the one in 64."""
    ops = _ops()
    for kernel in ("RBF", "LINEAR"):
        c = Case(lengths, H, D, P, 4, kernel, dtype, seed=D + T + 1)
        q, qd = c.queries(T, G, dtype)
        got = ops.bank_select(c.bank, c.table, c.length, qd, n_sel)
        assert np.array_equal(got.cpu().numpy(), _select_exact_many(c, q, n_sel, rbf=kernel == "RBF"))
        skip, sd = _skips(len(lengths), T, lengths, c.rng, c.dev)
        got = ops.bank_select(c.bank, c.table, c.length, qd, n_sel, skip=sd)
        assert np.array_equal(got.cpu().numpy(), _select_exact_many(c, q, n_sel, skip, kernel == "RBF"))


@pytest.mark.parametrize("T", [600, 1300])
def test_select_for_many_queries_where_few_bits_do_not_tell(T):
    """Runs of equal pages (more candidates than the screen holds), scores one 32-bit step apart, pages of huge and of tiny norm,
    pages that are not numbers (never chosen), queries of zeros and of huge values."""
    ops = _ops()
    P, n = 16, 700
    for kernel in ("RBF", "LINEAR"):
        for dtype in (BF16, F32):
            c = Case([P * n], 1, 64, P, 4, kernel, dtype, seed=77)
            q, _ = c.queries(T, 1, dtype)
            rng = c.rng
            cent = rng.normal(size=(n, 64)).astype(np.float32) * 0.2
            cent[100:400] = cent[99]                                            # equal
            cent[400:500] = cent[99]
            cent[400:500, 0] += np.arange(100, dtype=np.float32) * 2.0 ** -24   # next to equal
            cent[500:510] *= np.float32(1e25)
            cent[510:520] *= np.float32(1e-30)
            order = torch.as_tensor(c.table_np[0, :n].astype(np.int64)).to(c.dev)
            q[0, :4] = 0
            q[0, 4:200] = torch.as_tensor(cent[99]).to(dtype) * 2
            q[0, 200] *= 1e25
            q[0, 201] *= 1e-30
            qd = q.to(c.dev)
            c.bank.centroid[order, 0] = torch.as_tensor(cent).to(c.dev)
            for n_sel in (5, 64):
                got = ops.bank_select(c.bank, c.table, c.length, qd, n_sel).cpu().numpy()
                assert np.array_equal(got, _select_exact_many(c, q, n_sel, rbf=kernel == "RBF"))
            bad = rng.choice(n, 60, replace=False)
            c.bank.centroid[order[torch.as_tensor(bad).to(c.dev)], 0, 7] = math.nan
            got = ops.bank_select(c.bank, c.table, c.length, qd, 20).cpu().numpy()
            assert not np.isin(got, bad).any() and (got >= 0).all()
            c.bank.centroid[order[torch.as_tensor(bad).to(c.dev)], 0] = -1e30 if kernel == "RBF" else 0.0
            if kernel == "RBF":     # the same choice as with those pages as far away as can be
                assert np.array_equal(got, _select_exact_many(c, q, 20))


# ------------------------------------------------------------ attention over chosen pages
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D,P,H,G,T,S,lengths", [
    (64, 16, 1, 1, 1, 1, [40, 0]), (64, 64, 1, 1, 70, 4, [900, 64]), (32, 32, 2, 2, 5, 16, [300, 3]), (128, 16, 1, 4, 33, 9, [333]),
    (96, 128, 1, 1, 40, 2, [1000]), (192, 16, 1, 2, 3, 64, [500]), (256, 256, 1, 1, 3, 2, [700])])
def test_attend_pages(dtype, bits, D, P, H, G, T, S, lengths):
    ops = _ops()
    c = Case(lengths, H, D, P, bits, "RBF", dtype, seed=D + S)
    q, qd = c.queries(T, G, dtype)
    s = float(np.float32(1.0 / math.sqrt(D)))
    J = c.table.shape[1]
    sel = c.rng.integers(-2, J + 2, (len(lengths), T, H, S)).astype(np.int32)      # repeats, and numbers outside the table
    sd = torch.as_tensor(sel).to(c.dev)
    skip, kd = _skips(len(lengths), T, lengths, c.rng, c.dev)
    for sk, skd in ((None, None), (skip, kd)):
        out, lse = ops.bank_attend_pages(c.bank, c.table, c.length, qd, sd, s, skip=skd, want_lse=True)

        def seen(b, t, h):
            r = np.arange(lengths[b])
            ok = np.isin(r // P, sel[b, t, h])
            return ok if sk is None else ok & ~((r >= sk[b, t, 0]) & (r < sk[b, t, 1]))
        c.check(q, out, lse, s, seen)


@pytest.mark.parametrize("dtype,bits", [(BF16, 4), (F16, 8), (F32, 4)])
@pytest.mark.parametrize("D,P,H,G,T,S,lengths", [
    (64, 64, 1, 1, 600, 8, [900]), (32, 16, 2, 2, 150, 8, [200, 77]), (128, 128, 1, 1, 700, 6, [1500]), (96, 32, 1, 3, 100, 16, [333]),
    (256, 256, 1, 1, 1100, 4, [700]), (192, 16, 3, 1, 100, 16, [160]), (64, 64, 1, 1, 3100, 8, [900]), (32, 16, 2, 2, 4500, 8, [200, 77]),
    (128, 128, 1, 1, 1400, 6, [1500]), (96, 32, 1, 3, 2300, 16, [333]), (192, 16, 3, 1, 400, 16, [160])])
def test_attend_pages_of_many_queries(dtype, bits, D, P, H, G, T, S, lengths):
    """Enough queries for each page to be taken page by page; repeats, numbers outside the table and skipped rows among them."""
    ops = _ops()
    c = Case(lengths, H, D, P, bits, "RBF", dtype, seed=D + S)
    q, qd = c.queries(T, G, dtype)
    s = float(np.float32(1.0 / math.sqrt(D)))
    J = c.table.shape[1]
    sel = c.rng.integers(-2, J + 1, (len(lengths), T, H, S)).astype(np.int32)
    sd = torch.as_tensor(sel).to(c.dev)
    skip, kd = _skips(len(lengths), T, lengths, c.rng, c.dev)
    out, lse = ops.bank_attend_pages(c.bank, c.table, c.length, qd, sd, s, skip=kd, want_lse=True)

    def seen(b, t, h):
        r = np.arange(lengths[b])
        return np.isin(r // P, sel[b, t, h]) & ~((r >= skip[b, t, 0]) & (r < skip[b, t, 1]))
    c.check(q, out, lse, s, seen)
    again = [ops.bank_attend_pages(c.bank, c.table, c.length, qd, sd, s, skip=kd) for _ in range(3)]
    assert all(torch.equal(out, a) for a in again)


def test_all_pages_chosen_equals_the_whole_bank_and_banks_join_by_lse():
    """The set as a user runs it: append, read back, choose, attend; two halves of a bank joined by their lse."""
    ops = _ops()
    c = Case([16 * 40 - 3], 2, 64, 16, 4, "RBF", F32, seed=31)
    q, qd = c.queries(33, 2, F32)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=c.dev)
    out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, 0.2, want_lse=True)
    sel = ops.bank_select(c.bank, c.table, c.length, qd, 40)
    assert np.array_equal(sel.cpu().numpy(), np.broadcast_to(np.arange(40, dtype=np.int32), sel.shape))
    o2, l2 = ops.bank_attend_pages(c.bank, c.table, c.length, qd, sel, 0.2, want_lse=True)
    for o, l in ((out, lse), (o2, l2)):
        c.check(q, o, l, float(np.float32(0.2)), lambda b, t, h: np.ones(637, bool))
    # two halves, each a bank of its own over the same pages
    parts = [ops.bank_attend(c.bank, t.contiguous(), n, qd, 0.2, want_lse=True)
             for t, n in ((c.table[:, :20], i32(320)), (c.table[:, 20:], i32(317)))]
    w = torch.softmax(torch.stack([l for _, l in parts]).double(), 0).permute(0, 1, 3, 2)[..., None]
    joined = sum(wi * o.double() for wi, (o, _) in zip(w, parts))
    c.check(q, joined.float(), torch.logsumexp(torch.stack([l for _, l in parts]).double(), 0), float(np.float32(0.2)), lambda b, t, h: np.ones(637, bool))
    # eight new rows, then the same questions
    c2 = Case([16 * 40 - 3 + 8], 2, 64, 16, 4, "RBF", F32, seed=32)
    c2.k[:, :637], c2.v[:, :637] = c.k, c.v
    ops.bank_write(c2.bank, c2.table, i32(0), i32(637), c.k.to(c.dev), c.v.to(c.dev))
    ops.bank_write(c2.bank, c2.table, i32(637), i32(8), c2.k[:, 637:].to(c.dev), c2.v[:, 637:].to(c.dev))
    c2.hk, c2.hv = held(c2.k.double().numpy(), 4), held(c2.v.double().numpy(), 4)
    c2.o = -0.5 * (c2.hk ** 2).sum(-1)
    k, v = ops.bank_read(c2.bank, c2.table, i32(630), i32(15), 15)
    assert torch.equal(k.cpu().double(), torch.as_tensor(c2.hk[:, 630:])) and torch.equal(v.cpu().double(), torch.as_tensor(c2.hv[:, 630:]))
    sel = ops.bank_select(c2.bank, c2.table, c2.length, qd, 6)
    exact = _select_exact(c2, q, 6)
    assert np.array_equal(sel.cpu().numpy(), exact)
    out, lse = ops.bank_attend_pages(c2.bank, c2.table, c2.length, qd, sel, 0.2, want_lse=True)
    c2.check(q, out, lse, float(np.float32(0.2)), lambda b, t, h: np.isin(np.arange(645) // 16, exact[b, t, h]))


# ------------------------------------------------------------ streams, graphs, batches
def test_broadcast_queries_empty_batches_and_no_rows():
    ops = _ops()
    c = Case([100, 33], 1, 64, 16, 4, "RBF", BF16, seed=6)
    q, qd = c.queries(1, 1, BF16)
    wide = qd[:1, :1].expand(2, 50, 4, 64)
    out = ops.bank_attend(c.bank, c.table, c.length, wide, 0.3)
    assert out.is_contiguous() and (out == out[:, :1, :1]).all()
    sel = ops.bank_select(c.bank, c.table, c.length, wide, 2)
    assert (sel == sel[:, :1]).all()
    for T in (0,):
        e = torch.empty(2, 0, 1, 64, dtype=BF16, device=c.dev)
        assert ops.bank_attend(c.bank, c.table, c.length, e, 0.3).shape == e.shape
        assert ops.bank_select(c.bank, c.table, c.length, e, 2).shape == (2, 0, 1, 2)
        ops.bank_write(c.bank, c.table, c.length, c.length, e, e)
    none = torch.empty(0, 64, dtype=torch.int32, device=c.dev), torch.empty(0, dtype=torch.int32, device=c.dev)
    assert ops.bank_attend(c.bank, *none, torch.empty(0, 3, 1, 64, dtype=BF16, device=c.dev), 0.3).shape == (0, 3, 1, 64)
    # a table without columns: banks without rows
    out, lse = ops.bank_attend(c.bank, c.table[:, :0].contiguous(), c.length, qd, 0.3, want_lse=True)
    assert not out.any() and torch.isinf(lse).all()
    assert (ops.bank_select(c.bank, c.table[:, :0].contiguous(), c.length, qd, 3) == -1).all()


@pytest.mark.parametrize("T,n", [(1, 6000), (400, 900), (4500, 12000)])
def test_captured_and_replayed_beside_eager_calls(T, n):
    """One graph of the whole set, replayed with new queries and rows, another graph of the same calls between, eager calls beside."""
    ops = _ops()
    c = Case([n, n // 2], 1, 64, 64, 4, "RBF", BF16, seed=13, spare=9)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=c.dev)
    q, qd = c.queries(T, 1, BF16)
    start, count = i32(n - 5, n // 2 - 3), i32(5, 3)
    rows = [torch.as_tensor(c.rng.normal(size=(2, 5, 1, 64))).to(BF16).to(c.dev) for _ in range(2)]

    def step(q):
        ops.bank_write(c.bank, c.table, start, count, *rows)
        k, v = ops.bank_read(c.bank, c.table, start, count, 5, BF16)
        sel = ops.bank_select(c.bank, c.table, c.length, q, 8)
        out = ops.bank_attend_pages(c.bank, c.table, c.length, q, sel, 0.2, want_lse=True)
        return (k, v, sel, *out, *ops.bank_attend(c.bank, c.table, c.length, q, 0.2, want_lse=True))
    q2 = qd.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(qd)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for buf in (qd, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(buf)
        graphs.append((g, buf, res))
    for i in range(4):
        for g, buf, res in graphs:
            buf.copy_(torch.as_tensor(c.rng.normal(size=tuple(buf.shape)) * 0.5).to(BF16))
            rows[0].copy_(torch.as_tensor(c.rng.normal(size=(2, 5, 1, 64))).to(BF16))
            g.replay()
            got = [r.clone() for r in res]
            torch.cuda.synchronize()
            want = step(buf)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    ops = _ops()
    cs = [Case([5000], 1, 64, 64, 4, "RBF", BF16, seed=40 + i) for i in range(2)]
    qs = [c.queries(300, 1, BF16)[1] for c in cs]

    def run(c, q):
        sel = ops.bank_select(c.bank, c.table, c.length, q, 8)
        return sel, ops.bank_attend_pages(c.bank, c.table, c.length, q, sel, 0.2), ops.bank_attend(c.bank, c.table, c.length, q, 0.2)
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


def test_refusals_on_the_device():
    from super_resolution_amd import _lib
    ops = _ops()
    c = Case([100], 2, 64, 16, 4, "RBF", BF16, seed=1)
    q, qd = c.queries(3, 2, BF16)
    sel = torch.zeros(1, 3, 2, 4, dtype=torch.int32, device=c.dev)
    ok = dict(bank=c.bank, table=c.table, length=c.length, q=qd)
    bad = [
        lambda: ops.bank_attend(**{**ok, "q": qd.double()}, scale=1.0),
        lambda: ops.bank_attend(**{**ok, "q": qd[:, :, :3]}, scale=1.0),
        lambda: ops.bank_attend(**{**ok, "q": qd[..., :32]}, scale=1.0),
        lambda: ops.bank_attend(**{**ok, "q": qd.transpose(2, 3).contiguous().transpose(2, 3)}, scale=1.0),
        lambda: ops.bank_attend(**{**ok, "q": q}, scale=1.0),
        lambda: ops.bank_attend(**{**ok, "length": c.length.long()}, scale=1.0),
        lambda: ops.bank_attend(**{**ok, "table": c.table.long()}, scale=1.0),
        lambda: ops.bank_attend(**{**ok, "table": c.table[0]}, scale=1.0),
        lambda: ops.bank_attend(**ok, scale=0.0), lambda: ops.bank_attend(**ok, scale=math.nan),
        lambda: ops.bank_attend(**ok, scale=math.inf), lambda: ops.bank_attend(**ok, scale=-1.0),
        lambda: ops.bank_attend(**ok, scale=1.0, skip=torch.zeros(1, 3, 1, dtype=torch.int32, device=c.dev)),
        lambda: ops.bank_attend(**{**ok, "bank": c.bank._replace(bits=8)}, scale=1.0),
        lambda: ops.bank_attend(**{**ok, "bank": c.bank._replace(kernel_id=ops.MATERN52)}, scale=1.0),
        lambda: ops.bank_attend(**{**ok, "bank": c.bank._replace(offset=c.bank.offset[..., :8])}, scale=1.0),
        lambda: ops.bank_select(**ok, n_sel=0), lambda: ops.bank_select(**ok, n_sel=65),
        lambda: ops.bank_attend_pages(**ok, pages=sel[:, :2], scale=1.0),
        lambda: ops.bank_attend_pages(**ok, pages=sel.long(), scale=1.0),
        lambda: ops.bank_attend_pages(**ok, pages=sel[..., :0], scale=1.0),
        lambda: ops.bank_write(c.bank, c.table, c.length, c.length, c.k.to(c.dev), c.v.float().to(c.dev)),
        lambda: ops.bank_write(c.bank, c.table, c.length, c.length, c.k.to(c.dev)[:, :, :1], c.v.to(c.dev)[:, :, :1]),
        lambda: ops.bank_read(c.bank, c.table, c.length, c.length, 4, torch.float64),
        lambda: ops.bank_alloc(4, 1, 48), lambda: ops.bank_alloc(4, 1, 64, page_rows=24), lambda: ops.bank_alloc(0, 1, 64),
        lambda: ops.bank_alloc(4, 1, 64, bits=2), lambda: ops.bank_alloc(4, 1, 64, kernel_id=ops.MATERN12),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.GpsrError):
            f()
            pytest.fail(f"call {i} was not refused")


# ------------------------------------------------------------ sums near the end of float32's range
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,T", [(32, 3), (32, 20), (32, 100), (64, 100), (256, 40)])
def test_a_row_far_above_all_before_it(dtype, D, T):
    """A weight of 2^126.5 against the rows before it, times a value of 6, is past float32's range, the weight and the mean are not."""
    ops = _ops()
    c = Case([900], 1, D, 32, 4, "LINEAR", dtype, seed=D + T)
    c.k.zero_()
    c.k[0, 555, 0, 0] = 96.0
    c.v[0, 555, 0, :] = 6.0
    ops.bank_write(c.bank, c.table, torch.zeros_like(c.length), c.length, c.k.to(c.dev), c.v.to(c.dev))
    c.hk, c.hv, c.o = held(c.k.double().numpy(), 4), held(c.v.double().numpy(), 4), np.zeros((1, 900, 1))
    q = torch.zeros(1, T, 1, D, dtype=dtype)
    q[..., 0] = 1.0
    s = float(np.float32(126.5 * math.log(2) / 96))
    out, lse = ops.bank_attend(c.bank, c.table, c.length, q.to(c.dev), s, want_lse=True)
    c.check(q, out, lse, s, lambda b, t, h: np.ones(900, bool))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [2.5e38, 2.0 ** -108])
@pytest.mark.parametrize("T", [3, 20, 100, 700, 2900])
def test_values_of_the_ends_of_the_range(dtype, size, T):
    """Means of 900 values of up to 6 * 2^125, whose sum is past float32's range; and of the smallest ones."""
    ops = _ops()
    c = Case([900], 1, 64, 32, 4, "RBF", dtype, seed=T)
    c.v = (torch.as_tensor(c.rng.integers(-1, 2, size=(1, 900, 1, 64))).double() * size + size).to(dtype)     # 0, size, 2 size
    c.v.clamp_(max=2.5e38)
    ops.bank_write(c.bank, c.table, torch.zeros_like(c.length), c.length, c.k.to(c.dev), c.v.to(c.dev))
    c.hv = held(c.v.double().numpy(), 4)
    q, qd = c.queries(T, 1, dtype)
    out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, 0.25, want_lse=True)
    c.check(q, out, lse, 0.25, lambda b, t, h: np.ones(900, bool))
    sel = torch.as_tensor(c.rng.integers(0, 29, (1, T, 1, 16)).astype(np.int32))
    out, lse = ops.bank_attend_pages(c.bank, c.table, c.length, qd, sel.to(c.dev), 0.25, want_lse=True)
    c.check(q, out, lse, 0.25, lambda b, t, h: np.isin(np.arange(900) // 32, sel[b, t, h].numpy()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [2, 20, 100, 700, 1600])
def test_a_value_group_that_is_not_a_number(dtype, T):
    """NaN in columns 32 .. 63 of one row's value: those columns of the queries that see the row, and nothing else; T = 1600 goes page by page."""
    ops = _ops()
    c = Case([900], 1, 96, 32, 4, "RBF", dtype, seed=T)
    c.v[0, 333, 0, 40] = math.nan
    ops.bank_write(c.bank, c.table, torch.zeros_like(c.length), c.length, c.k.to(c.dev), c.v.to(c.dev))
    q, qd = c.queries(T, 1, dtype)
    skip = torch.zeros(1, T, 2, dtype=torch.int32)
    skip[:, ::2] = torch.tensor([333, 334])
    sel = torch.as_tensor(c.rng.permuted(np.tile(np.arange(29), (T, 1)), axis=1)[None, :, None, :16].astype(np.int32)).contiguous()
    every = lambda b, t, h: np.ones(900, bool)
    chosen = lambda b, t, h: np.isin(np.arange(900) // 32, sel[b, t, h].numpy())
    for see, f in ((every, lambda: ops.bank_attend(c.bank, c.table, c.length, qd, 0.25, skip=skip.to(c.dev), want_lse=True)),
                   (chosen, lambda: ops.bank_attend_pages(c.bank, c.table, c.length, qd, sel.to(c.dev), 0.25, skip=skip.to(c.dev), want_lse=True))):
        out, lse = f()
        seen = torch.tensor([bool(see(0, t, 0)[333]) and t % 2 == 1 for t in range(T)])
        gone = torch.isnan(out[0, :, 0]).cpu()
        assert torch.equal(gone[:, 32:64], seen[:, None].expand(T, 32)) and not gone[:, :32].any() and not gone[:, 64:].any()
        # the rest as if the row's value were zero there
        c.hv = held(torch.nan_to_num(c.v).double().numpy(), 4)
        c.hv[0, 333, 0, 32:64] = 0
        fixed = out.clone()
        for t in range(T):
            if seen[t]:
                e = softmax_mean(q[0, t, 0].double().numpy(), c.hk[0, :, 0], c.o[0, :, 0], c.hv[0, :, 0], see(0, t, 0), 0.25)[0]
                fixed[0, t, 0, 32:64] = torch.as_tensor(e[32:64]).to(dtype)
        r = np.arange(900)
        c.check(q, fixed, lse, 0.25, lambda b, t, h: see(b, t, h) & ~((r >= int(skip[b, t, 0])) & (r < int(skip[b, t, 1]))))


def test_which_way_the_pages_go():
    """The calls above that are to go page by page do: only that way has a workspace where there are this many queries."""
    from super_resolution_amd import _lib
    ops, lib = _ops(), _lib.load()
    for D, P, H, G, T, S, pages in ((64, 64, 1, 1, 3100, 8, 15), (32, 16, 2, 2, 4500, 8, 14), (128, 128, 1, 1, 1400, 6, 13), (96, 32, 1, 3, 2300, 16, 12),
                                    (192, 16, 3, 1, 400, 16, 11), (256, 256, 1, 1, 1100, 4, 4), (64, 32, 1, 1, 2900, 16, 30), (96, 32, 1, 1, 1600, 16, 30)):
        bank = ops.bank_alloc(pages, H, D, P, 4, ops.RBF)
        ref, _, _ = ops._bank(bank, bank.offset.get_device())
        B = 2 if T == 4500 else 1
        assert lib.gpsr_bank_attend_pages_workspace_bytes(ref, B, pages, T, H * G, S, 0) > 0, (D, T)


@pytest.mark.parametrize("dtype,D,bits", [(BF16, 64, 4), (F16, 96, 8), (F32, 32, 4), (BF16, 256, 4), (F32, 192, 8)])
@pytest.mark.parametrize("T,G", [(1, 1), (3, 10), (70, 1)])
def test_attend_of_few_queries_to_a_long_bank(dtype, D, bits, T, G):
    """More partial results of a column than one wave joins."""
    ops = _ops()
    c = Case([70001], 1, D, 64, bits, "RBF", dtype, seed=D + T)
    q, qd = c.queries(T, G, dtype)
    skip = torch.zeros(1, T, 2, dtype=torch.int32)
    skip[0, 0] = torch.tensor([0, 69000])         # most partials saw nothing
    out, lse = ops.bank_attend(c.bank, c.table, c.length, qd, 0.25, skip=skip.to(c.dev), want_lse=True)
    r = np.arange(70001)
    c.check(q, out, lse, 0.25, lambda b, t, h: ~((r >= int(skip[b, t, 0])) & (r < int(skip[b, t, 1]))))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [32, 64, 96])
def test_many_joined_columns_are_the_same_every_time(dtype, D):
    """Tens of thousands of columns joined from their partials, several times: every bit the same."""
    ops = _ops()
    c = Case([200, 77], 2, D, 16, 4, "RBF", dtype, seed=D)
    q, qd = c.queries(9000, 2, dtype)
    sel = torch.as_tensor(c.rng.integers(-2, 14, (2, 9000, 2, 4)).astype(np.int32)).to(c.dev)
    first = ops.bank_attend_pages(c.bank, c.table, c.length, qd, sel, 0.2, want_lse=True)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.bank_attend_pages(c.bank, c.table, c.length, qd, sel, 0.2, want_lse=True)))
    part = [ops.bank_attend_pages(c.bank, c.table, c.length, qd[:, t:t + 50].contiguous(), sel[:, t:t + 50].contiguous(), 0.2) for t in range(0, 9000, 50)]
    u, uw = torch.finfo(dtype).eps / 2, U_W[dtype]
    # the same rows taken query by query: two roundings of each kind, of means of values of at most 5
    assert (torch.cat(part, 1).double() - first[0].double()).abs().max() <= 5 * 2 * (u + uw + 2.0 ** -12)
