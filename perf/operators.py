"""Measured cases of the example-bank operators: writing a bank in 4 or 8 bits and reading it back, attention over it, the
choice of pages for each query, and attention over the chosen pages only.

A bank holds example windows of images (keys) and what belongs to them (values): side x side windows, zero-padded to a
multiple of 32 columns.  Codes are E2M1 pairs (low nibble first) or E4M3 bytes with one power-of-two scale byte (exponent +
127; 255: not a number) per 32 columns; rows lie in pages, and a table gives each bank's pages in order.
"""
import math

import torch

own = False

RBF, LINEAR = 0, 4                      # the framework's kernel ids
GROUP = 32                              # columns that share a scale
TOP = {4: 6.0, 8: 448.0}                # largest element value
SPAN = {4: (-110, 125), 8: (-110, 119)}  # exponents that a scale byte may hold
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------ cases
def listed():
    return [
        # one new example put behind the framework's 5000 candidates
        dict(name="write_one", op="write", B=1, T=1, H=1, side=7, P=64, bits=4, dtype="bf16", kernel=RBF, have=4999),
        # five images' examples, three planes each, appended to banks that end inside a page
        dict(name="write_ragged", op="write", B=5, T=701, H=3, side=11, P=32, bits=8, dtype="f16", kernel=RBF, have=1237),
        # a bank of a whole data set's windows, built in one call
        dict(name="write_build", op="write", B=1, T=400000, H=1, side=7, P=64, bits=4, dtype="f32", kernel=RBF, have=0),
        # one window asked of the framework's 5000 candidates: latency
        dict(name="attend_one", op="attend", B=1, T=1, G=1, H=1, rows=5000, side=7, P=64, bits=4, dtype="bf16", kernel=RBF, skip=False),
        # a few windows of four heads per bank head asked of four long banks: the bank is read once
        dict(name="attend_few_long", op="attend", B=4, T=3, G=4, H=2, rows=180001, side=11, P=64, bits=4, dtype="f16", kernel=LINEAR, skip=False),
        # leave-one-image-out in 32 bits over ragged 8-bit banks
        dict(name="attend_leave_out", op="attend", B=3, T=1531, G=1, H=2, rows=7003, side=9, P=32, bits=8, dtype="f32", kernel=RBF, skip=True),
        # every window of a 255 x 255 plane asked of 5000 candidates
        dict(name="attend_image", op="attend", B=1, T=65025, G=1, H=1, rows=5000, side=7, P=64, bits=4, dtype="bf16", kernel=RBF, skip=False),
        # a 200 x 200 plane asked of a whole data set's windows
        dict(name="attend_image_long", op="attend", B=1, T=40000, G=1, H=1, rows=100000, side=7, P=64, bits=4, dtype="bf16", kernel=RBF, skip=False),
        # pages for one window of each of eight banks, four heads together
        dict(name="select_one", op="select", B=8, T=1, G=4, H=1, rows=100000, side=7, P=64, bits=4, dtype="bf16", kernel=RBF, n_sel=16, skip=False),
        # pages for every window of a 200 x 200 plane
        dict(name="select_image", op="select", B=1, T=40000, G=1, H=1, rows=100000, side=7, P=64, bits=4, dtype="bf16", kernel=RBF, n_sel=16, skip=False),
        # attention over the chosen pages: one window of each of eight banks
        dict(name="pages_one", op="pages", B=8, T=1, G=4, H=1, rows=100000, side=7, P=64, bits=4, dtype="bf16", kernel=RBF, n_sel=16, skip=False),
        # and every window of a 200 x 200 plane
        dict(name="pages_image", op="pages", B=1, T=40000, G=1, H=1, rows=100000, side=7, P=64, bits=4, dtype="bf16", kernel=RBF, n_sel=16, skip=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    c = dict(op=rng.choice(["write", "attend", "select", "pages"]), B=rng.choice([1, 1, 2, 3, 5, 8]), H=rng.choice([1, 1, 2, 3]),
             side=rng.choice([5, 7, 7, 9, 11, 13, 15]), P=rng.choice([16, 32, 64, 64, 128]), bits=rng.choice([4, 4, 8]),
             dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), kernel=rng.choice([RBF, RBF, LINEAR]))
    D = _dim(c)
    if c["op"] == "write":
        c["T"] = _log(rng, 1, 400000 * 64 // (c["B"] * c["H"] * D))
        c["have"] = rng.choice([0, _log(rng, 1, 5000)])
        return c
    c["G"] = rng.choice([1, 1, 2, 4])
    c["skip"] = rng.random() < 0.3
    # a choice of pages is asked of banks that have more than it takes
    c["rows"] = _log(rng, 60 * c["P"] if c["op"] == "select" else 1, 100000 if c["B"] > 3 else 180000)
    wide = c["B"] * c["H"] * c["G"] * D
    if c["op"] == "attend":
        most = min(70000, 6.0e10 // (wide * c["rows"]))   # at most a quarter of the largest listed case
    else:
        c["n_sel"] = min(rng.choice([4, 8, 16, 32] if c["op"] == "select" else [1, 4, 8, 16, 32]), -(-c["rows"] // c["P"]))
        most = min(40000, 4.0e9 // (c["B"] * c["H"] * c["rows"] // c["P"] * D + 1), 2.6e9 // (wide * c["n_sel"] * c["P"]))
    c["T"] = _log(rng, 1, max(1, int(most)))
    return c


def _dim(c):
    return -(-c["side"] ** 2 // GROUP) * GROUP


def _dtype(c):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[c["dtype"]]


def _size(c):
    return 4 if c["dtype"] == "f32" else 2


def _row_bytes(c):
    D = _dim(c)
    return D * c["bits"] // 8 + D // GROUP


def work(c):
    D, H, B, T = _dim(c), c["H"], c["B"], c["T"]
    rows = B * H * T
    if c["op"] == "write":   # written, then read back
        return {"bytes": rows * (4 * D * _size(c) + 4 * _row_bytes(c) + 4) + 4 * D * rows / c["P"], "flops": 6 * D * rows}
    lengths = _lengths(c)
    q = B * T * H * c["G"] * D * _size(c)
    off = 4 if c["kernel"] == RBF else 0
    n_pages = sum(-(-n // c["P"]) for n in lengths)
    if c["op"] == "attend":
        return {"bytes": 2 * q + sum(lengths) * H * (2 * _row_bytes(c) + off), "flops": 4 * T * c["G"] * H * D * sum(lengths)}
    picked = B * T * H * c["n_sel"]
    if c["op"] == "select":
        return {"bytes": q + n_pages * H * D * 4 + picked * 4, "flops": 2 * T * H * D * n_pages}
    touched = min(picked, n_pages * H) * c["P"]
    return {"bytes": 2 * q + picked * 4 + touched * (2 * _row_bytes(c) + off), "flops": 4 * picked * c["G"] * c["P"] * D}


# ------------------------------------------------------------ inputs
def _lengths(c):
    return [max(1, c["rows"] - (c["rows"] // 7) * b % c["rows"]) for b in range(c["B"])]


def _field(gen, side):
    """A plane with smooth areas, edges and some grain, in [0, 1] or so, and a blurred copy: what an image and its interpolation look like."""
    def blur(x, r):
        return torch.nn.functional.avg_pool2d(torch.nn.functional.pad(x, (r, r, r, r), mode="reflect"), 2 * r + 1, 1)
    n = lambda: torch.randn(1, 1, side, side, generator=gen, device="cuda")  # noqa: E731
    smooth, edges = blur(blur(n(), 12), 12), torch.tanh(60 * blur(blur(n(), 7), 7))
    x = 0.5 + 3 * smooth + 0.2 * edges + 0.15 * blur(n(), 1)
    return x[0, 0], blur(x, 1)[0, 0]


def _windows(plane, y, x, side, D):
    """side x side windows at (y, x), zero-padded to D columns."""
    d = torch.arange(side, device="cuda")
    w = plane[(y[..., None, None] + d[:, None]), (x[..., None, None] + d)].flatten(-2)
    return torch.nn.functional.pad(w, (0, D - side * side))


def _centred(w, side):
    w = w.clone()
    w[..., :side * side] -= w[..., :side * side].mean(-1, keepdim=True)
    return w


def _examples(gen, plane, soft, shape, c):
    """Windows of the soft plane without their mean, and the detail that the plane has there, ordered by direction and strength of the slope."""
    S, side, D = plane.shape[0], c["side"], _dim(c)
    n = math.prod(shape)
    y, x = (torch.randint(0, S - side, (n,), generator=gen, device="cuda") for _ in range(2))
    m = side // 2
    gy, gx = soft[y + m + 1, x + m] - soft[y + m - 1, x + m], soft[y + m, x + m + 1] - soft[y + m, x + m - 1]
    order = torch.argsort(torch.round(torch.atan2(gy, gx) * (8 / math.pi)) * 10 + torch.hypot(gy, gx))
    y, x = y[order], x[order]
    k = _centred(_windows(soft, y, x, side, D), side)
    v = _windows(plane - soft, y, x, side, D)
    return k.view(*shape, D), v.view(*shape, D)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    D, B, H, T, P = _dim(c), c["B"], c["H"], c["T"], c["P"]
    dtype = _dtype(c)
    plane, soft = _field(gen, 700)
    writing = c["op"] == "write"
    lengths = [c["have"] - (c["have"] // 5) * b % max(1, c["have"]) + T for b in range(B)] if writing else _lengths(c)
    n_pages = [-(-n // P) for n in lengths]
    total, most = sum(n_pages) + 3, max(n_pages)
    places = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((B, most), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(n_pages):
        table[b, :n] = places[at:at + n]
        at += n
    width = D * c["bits"] // 8
    bank = {"k_codes": torch.zeros(total, H, P, width, dtype=torch.uint8, device="cuda"),
            "k_scales": torch.full((total, H, P, D // GROUP), 17, dtype=torch.uint8, device="cuda"),
            "v_codes": torch.zeros(total, H, P, width, dtype=torch.uint8, device="cuda"),
            "v_scales": torch.full((total, H, P, D // GROUP), 17, dtype=torch.uint8, device="cuda"),
            "offset": torch.zeros(total, H, P, device="cuda"), "centroid": torch.zeros(total, H, D, device="cuda")}
    state = {"case": dict(c), "bank": bank, "table": table}

    def fill(first, count, rows):
        k, v = _examples(gen, plane, soft, (B, rows, H), c)
        k, v = k.to(dtype), v.to(dtype)
        return k, v, torch.tensor(first, dtype=torch.int32, device="cuda"), torch.tensor(count, dtype=torch.int32, device="cuda"), _valid(count, rows)

    if writing:
        have = [n - T for n in lengths]
        if max(have):
            k, v, start, count, rows = fill([0] * B, have, max(have))
            _write(bank, table, start, rows, k, v, c)
        # the last banks get fewer rows than the first
        k, v, start, count, rows = fill(have, [T - (T // 9) * b for b in range(B)], T)
        state |= {"k": k, "v": v, "start": start, "count": count, "rows": rows}
        return state
    k, v, start, count, rows = fill([0] * B, lengths, max(lengths))
    _write(bank, table, start, rows, k, v, c)
    del k, v
    state["length"] = count
    # the queries: windows of another plane of the same kind, in the order of its pixels
    plane, soft = _field(gen, 700)
    wide = max(1, math.isqrt(T))
    t = torch.arange(T, device="cuda")[:, None]
    h = torch.arange(H * c["G"], device="cuda")[None]
    room = 700 - c["side"]
    q = torch.stack([_centred(_windows(soft, (t // wide + 37 * h + 61 * b) % room, (t % wide + 53 * h + 29 * b) % room, c["side"], D), c["side"]) for b in range(B)])
    state["q"] = q.to(dtype)
    near = 1.5 / float((q ** 2).sum(-1).mean() + 1e-6)     # a bandwidth of about the windows' own norm, and half of it
    state["scale"] = (8 if c["kernel"] == RBF else 4) * near
    state["skip"] = None
    if c["skip"]:    # a tenth of the bank, another one for each query; now and then all of it
        n = count[:, None].to(torch.float32)
        lo = (torch.rand(B, T, generator=gen, device="cuda") * n).to(torch.int32)
        hi = (lo + n / 10).to(torch.int32)
        none = torch.rand(B, T, generator=gen, device="cuda") < 0.02
        state["skip"] = torch.stack([torch.where(none, 0, lo), torch.where(none, count[:, None], hi)], -1).to(torch.int32).contiguous()
    if c["op"] == "pages":
        state["pages"] = _select(bank, table, count, state["q"], c, state["skip"])
    return state


def _valid(count, rows):
    """The places (bank, row) of a padded batch that hold a row, as flat numbers."""
    return torch.cat([torch.arange(n, device="cuda") + b * rows for b, n in enumerate(count)])


# ------------------------------------------------------------ the plain forms
def _power(byte):
    """2^(byte - 127) of a scale byte; NaN for 255."""
    return torch.where(byte == 255, math.nan, (byte.to(torch.int32) << 23).view(torch.float32))


def _two(e):
    """2^e for whole e in [-126, 127], exactly."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantise(x, bits):
    """[..., D] -> element values on the grid [..., D / 32, 32] and scale bytes [..., D / 32]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    bad = ~torch.isfinite(g).all(-1)
    m, e = torch.frexp(torch.where(bad, 0.0, top))
    e = e - (3 if bits == 4 else 9) + (m > TOP[bits] / 2 ** (3 if bits == 4 else 9)).to(torch.int32)
    e = torch.where(top == 0, SPAN[bits][0], e).clamp(*SPAN[bits])
    y = (g * _two(-e)[..., None]).clamp(-TOP[bits], TOP[bits])
    a = y.abs()
    if bits == 4:
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    else:
        step = _two((torch.frexp(a)[1] - 4).clamp(-9, 5))
    y = torch.where(bad[..., None], 0.0, torch.copysign(torch.round(a / step) * step, y))
    return y, torch.where(bad, 255, e + 127).to(torch.uint8)


def _pack(y, bits):
    """Grid values [..., D / 32, 32] -> code bytes [..., D * bits / 8]."""
    y = y.flatten(-2)
    a, sign = y.abs(), torch.signbit(y)
    if bits == 4:
        code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (sign.to(torch.uint8) << 3)
        return code[..., 0::2] | (code[..., 1::2] << 4)
    e = (torch.frexp(a)[1] - 1).clamp(min=-6)
    steps = (a * _two(3 - e)).to(torch.int32)                       # 8..15 for normal values, below for subnormal ones
    code = torch.where(steps < 8, steps, ((e + 7) << 3) | (steps & 7))
    return (code | (sign.to(torch.int32) << 7)).to(torch.uint8)


def _values(codes, scales, bits):
    """Codes and scale bytes -> the values they stand for, 32 bits."""
    c = codes.to(torch.int32)
    if bits == 4:
        c = torch.stack([c & 15, c >> 4], -1).flatten(-2)
        y = torch.tensor(E2M1, device=codes.device)[c & 7]
        y = torch.where(c > 7, -y, y)
    else:
        e, m = (c >> 3) & 15, (c & 7).float()
        y = torch.where(e == 0, m / 512, (1 + m / 8) * _two(e - 7))
        y = torch.where(c > 127, -y, y)
    return (y.unflatten(-1, (-1, GROUP)) * _power(scales)[..., None]).flatten(-2)


def _slots(table, start, T, P):
    """Physical row of each new row [B, T] (page * P + row)."""
    pos = start[:, None].long() + torch.arange(T, device=table.device)
    page = torch.gather(table.long(), 1, (pos // P).clamp(max=table.shape[1] - 1))
    return page * P + pos % P


def _put(bank, name, x, page, row, bits):
    """Rounds rows, stores their codes and scales, and returns the values held."""
    y, s = _quantise(x, bits)
    bank[name + "_codes"][page, :, row] = _pack(y, bits)
    bank[name + "_scales"][page, :, row] = s
    return (y * _power(s)[..., None]).flatten(-2)


def _write(bank, table, start, rows, k, v, c):
    B, T, H, D = k.shape
    P, bits = c["P"], c["bits"]
    slots = _slots(table, start, T, P).flatten()[rows]
    page, row = slots // P, slots % P
    _put(bank, "v", v.flatten(0, 1)[rows], page, row, bits)
    held = _put(bank, "k", k.flatten(0, 1)[rows], page, row, bits)
    if c["kernel"] == RBF:
        bank["offset"][page, :, row] = (held.double().square().sum(-1) * -0.5).float()
    # the mean key of every page that got a row, over the rows that it now has: those before the call's last one
    last = torch.zeros(bank["offset"].shape[0], dtype=torch.int64, device=k.device).scatter_reduce(0, page, row + 1, "amax")
    hit = torch.unique(page)
    keys = _values(bank["k_codes"][hit], bank["k_scales"][hit], bits).double()
    there = (torch.arange(P, device=k.device) < last[hit][:, None])[:, None, :, None]
    bank["centroid"][hit] = (torch.where(there, keys, 0.0).sum(2) / last[hit][:, None, None]).float()


def _read(bank, table, start, rows, T, c):
    B, (_, H, P, _) = table.shape[0], bank["k_codes"].shape
    slots = _slots(table, start, T, P).flatten()[rows]
    page, row = slots // P, slots % P
    k, v = torch.zeros(2, B * T, H, _dim(c), dtype=_dtype(c), device=table.device)
    k[rows] = _values(bank["k_codes"][page, :, row], bank["k_scales"][page, :, row], c["bits"]).to(k.dtype)
    v[rows] = _values(bank["v_codes"][page, :, row], bank["v_scales"][page, :, row], c["bits"]).to(v.dtype)
    return k.unflatten(0, (B, T)), v.unflatten(0, (B, T))


def _mask(length, skip, pos):
    """[B, Tq or 1, len(pos)]: which positions a query may see."""
    ok = pos < length[:, None, None]
    if skip is not None:
        ok = ok & ~((pos >= skip[..., :1]) & (pos < skip[..., 1:]))
    return ok


def _softmax_sum(x, ok, v):
    """sum softmax(x)_r v_r over the rows that are ok, and the log of the sum of exponentials."""
    x = torch.where(ok, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    return p @ v / torch.where(total == 0, 1.0, total), (torch.log(total) + m).squeeze(-1)


def _attend(bank, table, length, q, scale, skip, c):
    B, T, Hq, D = q.shape
    H, P, G = c["H"], c["P"], c["G"]
    pages = table.clamp(min=0).long()
    k, v = (_values(bank[n + "_codes"][pages], bank[n + "_scales"][pages], c["bits"]).transpose(1, 2).flatten(2, 3) for n in "kv")
    ok = _mask(length, skip, torch.arange(k.shape[2], device=q.device))                  # [B, T or 1, L]
    if skip is None:
        v = torch.where(ok[:, :, :, None], v, 0.0)
    off = bank["offset"][pages].transpose(1, 2).flatten(2, 3)                             # [B, H, L]
    qh = q.float().view(B, T, H, G, D).permute(0, 2, 3, 1, 4).flatten(2, 3)               # [B, H, G T, D]
    x = (qh @ k.transpose(2, 3).contiguous() + off[:, :, None]) * scale
    out, lse = _softmax_sum(x, ok[:, None].repeat(1, 1, G, 1) if skip is not None else ok[:, None], v)
    return (out.view(B, H, G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(q.dtype),
            lse.view(B, H * G, T))


def _select(bank, table, length, q, c, skip):
    B, T, Hq, D = q.shape
    H, P, G = c["H"], c["P"], c["G"]
    cent = bank["centroid"][table.clamp(min=0).long()].double().transpose(1, 2)           # [B, H, pages, D]
    qs = q.double().view(B, T, H, G, D).sum(3).transpose(1, 2)                            # [B, H, T, D]
    score = qs @ cent.transpose(2, 3).contiguous()
    if c["kernel"] == RBF:
        score = score - 0.5 * G * cent.square().sum(-1)[:, :, None]
    first = torch.arange(cent.shape[2], device=q.device) * P
    ok = first < length[:, None, None]
    if skip is not None:    # a page whose every row is left out cannot be chosen
        end = torch.minimum(first + P, length[:, None, None])
        ok = ok & ~((skip[..., :1] <= first) & (skip[..., 1:] >= end))
    score = torch.where(ok[:, None], score, -math.inf)
    best, at = torch.sort(score, dim=-1, descending=True, stable=True)
    best, at = best[..., :c["n_sel"]], at[..., :c["n_sel"]]
    big = torch.iinfo(torch.int32).max
    at = torch.where(best == -math.inf, big, at).sort(-1)[0]
    return torch.where(at == big, -1, at).to(torch.int32).transpose(1, 2).contiguous()   # [B, T, H, n_sel]


def _attend_pages(bank, table, length, q, pages, scale, skip, c):
    B, T, Hq, D = q.shape
    H, P, G = c["H"], c["P"], c["G"]
    there = pages >= 0
    logical = pages.clamp(min=0).long()
    phys = torch.gather(table.long(), 1, logical.flatten(1)).view_as(logical).clamp(min=0)
    head = torch.arange(H, device=q.device)[:, None]
    k, v = (_values(bank[n + "_codes"], bank[n + "_scales"], c["bits"])[phys, head].flatten(3, 4) for n in "kv")   # [B, T, H, S P, D]
    pos = logical[..., None] * P + torch.arange(P, device=q.device)
    ok = there[..., None] & (pos < length[:, None, None, None, None])
    if skip is not None:
        ok = ok & ~((pos >= skip[:, :, None, None, :1]) & (pos < skip[:, :, None, None, 1:]))
    x = q.float().view(B, T, H, G, D) @ k.transpose(3, 4)
    x = (x + bank["offset"][phys, head].flatten(3)[:, :, :, None]) * scale
    out, lse = _softmax_sum(x, ok.flatten(3)[:, :, :, None], v)
    return out.reshape(B, T, Hq, D).to(q.dtype), lse.reshape(B, T, Hq).transpose(1, 2).contiguous()


def run(state):
    c, bank, table = state["case"], state["bank"], state["table"]
    if own:
        from super_resolution_amd import ops
        b = ops.Bank(**bank, bits=c["bits"], kernel_id=c["kernel"])
        if c["op"] == "write":
            ops.bank_write(b, table, state["start"], state["count"], state["k"], state["v"])
            k, v = ops.bank_read(b, table, state["start"], state["count"], c["T"], _dtype(c))
            return k, v, bank["offset"], bank["centroid"]
        if c["op"] == "attend":
            return ops.bank_attend(b, table, state["length"], state["q"], state["scale"], skip=state["skip"], want_lse=True)
        if c["op"] == "select":
            return ops.bank_select(b, table, state["length"], state["q"], c["n_sel"], skip=state["skip"])
        return ops.bank_attend_pages(b, table, state["length"], state["q"], state["pages"], state["scale"], skip=state["skip"], want_lse=True)
    if c["op"] == "write":
        _write(bank, table, state["start"], state["rows"], state["k"], state["v"], c)
        k, v = _read(bank, table, state["start"], state["rows"], c["T"], c)
        return k, v, bank["offset"], bank["centroid"]
    if c["op"] == "attend":
        return _attend(bank, table, state["length"], state["q"], state["scale"], state["skip"], c)
    if c["op"] == "select":
        return _select(bank, table, state["length"], state["q"], c, state["skip"])
    return _attend_pages(bank, table, state["length"], state["q"], state["pages"], state["scale"], state["skip"], c)


# ------------------------------------------------------------ 64 bits, from the definitions
def _unit(e):
    """2^e in 64 bits, exactly, for whole e in [-300, 300]; NaN outside."""
    table = torch.tensor([2.0 ** i for i in range(-300, 301)], dtype=torch.float64, device="cuda")
    return torch.where(e.abs() <= 300, table[(e.clamp(-300, 300) + 300).long()], math.nan)


def _grid(bits):
    """Every value that a code stands for, as 64-bit numbers in the order of the codes."""
    if bits == 4:
        half = [m * 0.5 if e == 0 else (1 + m * 0.5) * 2.0 ** (e - 1) for e in range(4) for m in range(2)]
    else:
        half = [m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)]
        half[-1] = math.nan
    return torch.tensor(half + [-x for x in half], dtype=torch.float64, device="cuda")


def _held(bank, name, bits):
    codes, scales = bank[name + "_codes"], bank[name + "_scales"].double()
    if bits == 4:
        both = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.int64, device=codes.device)
        both[..., 0::2], both[..., 1::2] = codes % 16, codes // 16
    else:
        both = codes.long()
    return _grid(bits)[both] * torch.repeat_interleave(torch.where(scales == 255, math.nan, _unit(scales - 127)), GROUP, -1)


def _nearest(x, bits):
    """64-bit rows -> the nearest values that a bank can hold, ties to the even code."""
    half = _grid(bits)[:8 if bits == 4 else 127]
    between = (half[1:] + half[:-1]) / 2
    g = x.unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / TOP[bits]).clamp(-299, 299))
    e = e - (top <= TOP[bits] * _unit(e - 1)).double()
    unit = _unit(e.clamp(*SPAN[bits]))
    a = (g.abs() / unit).contiguous()
    low, high = torch.searchsorted(between, a, right=False), torch.searchsorted(between, a, right=True)
    return (torch.sign(g) * half[torch.where(low % 2 == 0, low, high)] * unit).flatten(-2)


def exact(case, seed):
    c = case
    if c["op"] == "attend" and work(c)["flops"] > 1.5e14:
        return None
    s = prepare(c, seed)
    bank, table, P, H, bits = s["bank"], s["table"], c["P"], c["H"], c["bits"]
    D = _dim(c)
    if c["op"] == "write":
        keys, values = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in "kv")
        offset, centroid = bank["offset"].double(), bank["centroid"].double()
        held = _held(bank, "k", bits)
        for b in range(c["B"]):
            first, n = int(s["start"][b]), int(s["count"][b])
            keys[b, :n], values[b, :n] = _nearest(s["k"][b, :n].double(), bits), _nearest(s["v"][b, :n].double(), bits)
            pos = torch.arange(first, first + n, device="cuda")
            page = table[b].long()[pos // P]
            held[page, :, pos % P] = keys[b, :n]
            if c["kernel"] == RBF:
                offset[page, :, pos % P] = -keys[b, :n].pow(2).sum(-1) / 2
            mine = table[b, first // P:(first + n - 1) // P + 1].long()
            if len(mine) > 1:
                centroid[mine[:-1]] = held[mine[:-1]].mean(2)
            centroid[mine[-1]] = held[mine[-1], :, :(first + n - 1) % P + 1].mean(1)
        return keys, values, offset, centroid
    B, T, G = c["B"], c["T"], c["G"]
    q = s["q"].double()
    result = torch.full((B, T, H, c["n_sel"]), -1, dtype=torch.int32, device="cuda") if c["op"] == "select" else None
    out, lse = torch.zeros(B, T, H * G, D, dtype=torch.float64, device="cuda"), torch.full((B, H * G, T), -math.inf, dtype=torch.float64, device="cuda")
    keys, values = _held(bank, "k", bits), _held(bank, "v", bits)
    for b in range(B):
        n = int(s["length"][b])
        pages = table[b, :-(-n // P)].long()
        pos = torch.arange(n, device="cuda")
        for h in range(H):
            k, v = (x[pages, h].reshape(-1, D)[:n] for x in (keys, values))
            cent = bank["centroid"][pages, h].double()
            step = max(1, int(2e8 // n))
            for t in range(0, T, step):
                part = slice(t, min(T, t + step))
                gone = torch.zeros(part.stop - t, n, dtype=torch.bool, device="cuda")
                if s["skip"] is not None:
                    lo, hi = s["skip"][b, part, 0, None], s["skip"][b, part, 1, None]
                    gone = (lo <= pos) & (pos < hi)
                if c["op"] == "select":
                    full = torch.nn.functional.pad(gone, (0, len(pages) * P - n), value=True).view(-1, len(pages), P).all(-1)
                    x = sum(q[b, part, h * G + g] @ cent.T for g in range(G))
                    if c["kernel"] == RBF:
                        x = x - G * (cent * cent).sum(1) / 2
                    x[full] = -math.inf
                    for i in range(c["n_sel"]):
                        top = x.max(1, keepdim=True)[0]
                        at = (x == top).to(torch.uint8).argmax(1, keepdim=True)
                        result[b, part, h, i] = torch.where(top == -math.inf, -1, at)[:, 0].int()
                        x.scatter_(1, at, -math.inf)
                    continue
                if c["op"] == "pages":
                    seen = torch.zeros(part.stop - t, len(pages) + 1, dtype=torch.bool, device="cuda")
                    seen.scatter_(1, s["pages"][b, part, h].long() % (len(pages) + 1), True)
                    gone = gone | ~seen[:, :-1].repeat_interleave(P, 1)[:, :n]
                for g in range(G):
                    x = q[b, part, h * G + g] @ k.T
                    if c["kernel"] == RBF:
                        x = x - (k * k).sum(1) / 2
                    x = (x * s["scale"]).masked_fill_(gone, -math.inf)
                    z = torch.logsumexp(x, 1)
                    lse[b, h * G + g, part] = z
                    out[b, part, h * G + g] = torch.exp_(x.sub_(z.clamp(min=-1e300)[:, None])) @ v
    if result is not None:
        big = torch.iinfo(torch.int32).max
        at = torch.where(result < 0, big, result).sort(-1)[0]
        return torch.where(at == big, -1, at)
    return out, lse
