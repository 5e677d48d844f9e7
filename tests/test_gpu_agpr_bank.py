"""The example bank behind AGPR (agpr.PREDICTOR = Predictor.BANK): windows and blending against numpy, ExampleBank's bookkeeping,
and upscale() as a user calls it against the same steps in 64 bits."""
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_kernels import natural_image, to_dev


def _windows(img, side):
    return np.lib.stride_tricks.sliding_window_view(img, (side, side)).reshape(-1, side * side)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,W,side,dim", [(7, 7, 7, 64), (20, 33, 3, 32), (41, 15, 15, 256), (30, 30, 5, 25)])
def test_windows_and_blend(dtype, H, W, side, dim):
    from super_resolution_amd import ops
    img = natural_image(H, W, 3)
    d = to_dev(img)
    u = torch.finfo(dtype).eps / 2
    for centre in (False, True):
        want = _windows(img, side)
        want = want - want.mean(1, keepdims=True) if centre else want
        got = ops.bank_windows(d, side, dim, dtype, centre=centre)
        assert got.shape == (1, len(want), 1, dim) and not got[..., side * side:].any()
        # one rounding to 32 bits, one to the type; the mean of at most 225 numbers in 64 bits.  Below the type's smallest normal
        # number its steps no longer shrink with the value: half of one is finfo.tiny * u there (f16: 2^-14 * 2^-11 = 2^-25, which
        # is what a centred window's small values are off by; for the other types it is nothing).
        err = np.abs(got[0, :, 0, :side * side].double().cpu().numpy() - want)
        assert (err <= (u + 2.0 ** -24) * np.abs(want) + 300 * 2.0 ** -53 + torch.finfo(dtype).tiny * u).all()
    detail = torch.as_tensor(np.random.default_rng(1).normal(size=(1, len(want), 1, dim))).to(dtype)
    out = ops.bank_blend(d, detail.to(d.device), side).cpu().numpy()
    total, n = np.zeros((H, W)), np.zeros((H, W))
    rows = detail.double().numpy()[0, :, 0, :side * side].reshape(H - side + 1, W - side + 1, side, side)
    for y in range(H - side + 1):
        for x in range(W - side + 1):
            total[y:y + side, x:x + side] += rows[y, x]
            n[y:y + side, x:x + side] += 1
    assert np.abs(out - (img + total / n)).max() < 1e-12     # 225 numbers of at most 5, in 64 bits


def test_refusals():
    from super_resolution_amd import _lib, ops
    from super_resolution_amd.bank import ExampleBank
    d = to_dev(natural_image(16, 16, 1))
    rows = torch.zeros(1, 100, 1, 64, device=d.device)
    b = ExampleBank(100, 49)
    k = torch.zeros(60, 49, device=d.device)
    b.append(k, k)
    for f in (lambda: ops.bank_windows(d, 4, 64), lambda: ops.bank_windows(d, 17, 256), lambda: ops.bank_windows(d, 7, 48),
              lambda: ops.bank_windows(d[:6].contiguous(), 7, 64), lambda: ops.bank_windows(d, 7, 64, torch.float64),
              lambda: ops.bank_windows(d.cpu(), 7, 64), lambda: ops.bank_windows(d.float(), 7, 64),
              lambda: ops.bank_blend(d, rows[:, :50], 7), lambda: ops.bank_blend(d, rows.double(), 7),
              lambda: ExampleBank(0, 49), lambda: ExampleBank(10, 257), lambda: b.append(k, k), lambda: b.append(k[:, :48], k[:, :48]),
              lambda: b.predict(k[:, :48], 1.0)):
        with pytest.raises(_lib.GpsrError):
            f()


def test_example_bank_appends_reads_and_predicts():
    from super_resolution_amd import ops
    from super_resolution_amd.bank import ExampleBank
    rng = np.random.default_rng(4)
    dev = torch.device("cuda", torch.cuda.current_device())
    k, v = (torch.as_tensor(rng.normal(size=(700, 49)).astype(np.float32)).to(dev) for _ in range(2))
    b = ExampleBank(1000, 49, page_rows=16, bits=8)
    for i, n in ((0, 1), (1, 299), (300, 400)):
        b.append(k[i:i + n], v[i:i + n])
    hk, hv = (x[:, 0] for x in b.read(0, 700))
    # E4M3: half a step of 2^-4 of the value, or of the smallest step of the row's 32 columns
    top = torch.nn.functional.pad(k, (0, 15)).view(-1, 2, 32).abs().amax(-1).repeat_interleave(32, 1)[:, :49]
    assert ((hk - k).abs() <= torch.maximum(k.abs() * 2.0 ** -4, top * 2.0 ** -17)).all()
    q = k[:50] + 0.1
    out, lse = b.predict(q, 0.4, want_lse=True)
    x = 0.4 * (q.double() @ hk.double().T - hk.double().square().sum(1) / 2)
    want = torch.softmax(x, 1) @ hv.double()
    # 32-bit sums of logits up to some 30 and of 700 rows: 2 e (68 * 30 + 2) + 1400 e, with A <= 4
    assert (out.double() - want).abs().max() < 4 * 2.0 ** -23 * 5600 and (lse[0].double() - torch.logsumexp(x, 1)).abs().max() < 2.0 ** -23 * 5600
    # as many pages as there are: the whole bank; fewer: those of bank_select
    assert torch.equal(out, b.predict(q, 0.4, pages=44))
    sel = ops.bank_select(b.bank, b.table, b.length, torch.nn.functional.pad(q, (0, 15))[None, :, None], 5)
    seen = torch.zeros(50, 44, dtype=torch.bool, device=dev).scatter_(1, sel[0, :, 0].long(), True).repeat_interleave(16, 1)[:, :700]
    some = torch.softmax(x.masked_fill(~seen, -torch.inf), 1) @ hv.double()
    assert (b.predict(q, 0.4, pages=5).double() - some).abs().max() < 4 * 2.0 ** -23 * 5600
    # a scale that says more about the neighbours than one that averages everything
    smooth = torch.tanh(k @ torch.as_tensor(rng.normal(size=(49, 49)).astype(np.float32) * 0.05).to(dev))
    c = ExampleBank(700, 49, bits=8).append(k * 0.2, smooth)
    assert c.choose_scale([1e-6, 5.0], sample=300) == 5.0


@pytest.mark.parametrize("pages", [None, 4])
def test_agpr_with_a_bank_runs_as_its_definition(tmp_path, golden_dir, monkeypatch, pages):
    """Fourteen HR fixtures as training images, one colour image up x2: the detail image against the same sums in 64 bits, upscale()
    for its shape and range, and the saved bank read back."""
    from super_resolution_amd import agpr, ops
    os.symlink(os.path.join(golden_dir, "refset"), tmp_path / "Set14")
    for name, value in (("BASE_DIR", str(tmp_path)), ("SRF", 2), ("DATASET", agpr.TrainingDataset.Set14), ("BANK_ROWS", 3001), ("BANK_PAGES", pages),
                        ("PREDICTOR", agpr.Predictor.BANK), ("COLOR_SPACE", agpr.ColorSpace.YCRCB)):
        monkeypatch.setattr(agpr, name, value)
    np.random.seed(3)
    model = agpr.AGPRSuperResolution(2)
    assert model.bank.rows == 3001 and model.bank_scale > 0
    again = agpr.AGPRSuperResolution(2, use_existing_model=True)
    assert all(torch.equal(a, b) for a, b in zip(model.bank.bank[:6], again.bank.bank[:6])) and model.bank_scale == again.bank_scale

    up = to_dev(natural_image(40, 52, 9))
    q = ops.bank_windows(up, 7, 64, centre=True)
    k, v = (x[:, 0].double() for x in model.bank.read(0, 3001))
    x = model.bank_scale * (q[0, :, 0, :49].double() @ k.T - k.square().sum(1) / 2)
    if pages is not None:
        sel = ops.bank_select(model.bank.bank, model.bank.table, model.bank.length, q, pages)
        seen = torch.zeros(len(x), 47, dtype=torch.bool, device=x.device).scatter_(1, sel[0, :, 0].long(), True).repeat_interleave(64, 1)[:, :3001]
        x = x.masked_fill(~seen, -torch.inf)
    w = torch.softmax(x, 1)
    detail = torch.nn.functional.pad(w @ v, (0, 15))
    exact = ops.bank_blend(up, detail.float()[None, :, None].contiguous(), 7)
    # bf16 weights and details: 2^-8 of the mean absolute detail each, f16 partials 2^-11 of the largest
    bound = 2.5 * 2.0 ** -8 * float((w @ v.abs()).max())
    assert float((model._bank_detail(up) - exact).abs().max()) <= bound

    bgr = (natural_image(24, 30, 5)[..., None] * np.array([255, 240, 200])).astype(np.uint8)
    out = model.upscale(bgr)
    assert out.shape == (48, 60, 3) and out.dtype == np.uint8
    assert np.abs(out.astype(int).mean() - bgr.astype(int).mean()) < 8
