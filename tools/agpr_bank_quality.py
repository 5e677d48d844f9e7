"""Held-out quality of AGPR with an example bank (agpr.Predictor.BANK) next to bicubic interpolation and the GP: luma PSNR (dB, a
border of 4 pixels left out) of five Set14 images x2, windows drawn from the other nine (tests/golden/refset); the GP is the one whose
checkpoint the reference committed for BSD100 x2 (tests/golden/agpr_BSD100_SRF_2.npz).  Then the time of the bank's part for the last
image.  Prints two small tables; needs a GPU.    python tools/agpr_bank_quality.py"""
import os
import shutil
import sys
import tempfile
import time

import numpy as np
import torch
from PIL import Image

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]
from super_resolution_amd import agpr, imgproc, ops  # noqa: E402
from test_gpu_agpr import _write_checkpoint  # noqa: E402

GOLDEN = os.path.join(ROOT, "tests", "golden")
HELD_OUT = (1, 2, 5, 8, 13)
BANKS = (("bank 4 bits, 16 pages", 100000, 4, 16), ("bank 8 bits, 16 pages", 100000, 8, 16), ("bank 4 bits, all pages", 100000, 4, None))


def hr_path(i):
    return os.path.join(GOLDEN, "refset", "image_SRF_2", f"img_{i:03d}_SRF_2_HR.png")


def luma(i):
    bgr = np.ascontiguousarray(np.array(Image.open(hr_path(i)).convert("RGB"))[:, :, ::-1])
    y = imgproc.bgr2ycrcb(bgr)[0] / 255
    return np.ascontiguousarray(y[:y.shape[0] // 2 * 2, :y.shape[1] // 2 * 2])


def psnr(a, b):
    a, b = a[4:-4, 4:-4], b[4:-4, 4:-4]
    return 10 * np.log10(1 / np.mean((a - b) ** 2))


def main():
    base = tempfile.mkdtemp()
    _write_checkpoint(base, GOLDEN, "BSD100/SRF_2")
    train = os.path.join(base, "train")
    os.makedirs(train)
    for i in range(1, 15):
        if i not in HELD_OUT:
            shutil.copy(hr_path(i), train)
    agpr.BASE_DIR, agpr.BSD100_DIR, agpr.SRF, agpr.DATASET = base, train, 2, agpr.TrainingDataset.BSD100
    np.random.seed(0)
    models = {"GP": (agpr.AGPRSuperResolution(2, use_existing_model=True), None)}
    agpr.PREDICTOR = agpr.Predictor.BANK
    for name, rows, bits, pages in BANKS:
        agpr.BANK_ROWS, agpr.BANK_BITS, agpr.BANK_PAGES = rows, bits, pages
        models[name] = (agpr.AGPRSuperResolution(2), pages)
    alone, after = {}, {}
    for i in HELD_OUT:
        hr = luma(i)
        low = torch.as_tensor(agpr.downscale(hr)).cuda()
        up = imgproc.resize_cubic(low, dsize=(hr.shape[1], hr.shape[0]))
        alone.setdefault("bicubic", []).append(psnr(up.cpu().numpy(), hr))
        for name, (m, pages) in models.items():
            agpr.BANK_PAGES = pages
            pred = (m._bank_detail(up) if m.predictor == agpr.Predictor.BANK
                    else ops.agpr_filter(up, agpr.L, m.filter_weights(), m.model.raw[0].contiguous()))
            alone.setdefault(name, []).append(psnr(pred.cpu().numpy(), hr))
            after.setdefault(name, []).append(psnr(m.upscale_channel_device(low).cpu().numpy() / 255, hr))
    print("| method | before back-projection | after |\n|---|---|---|")
    for name, x in alone.items():
        print(f"| {name} | {np.mean(x):.2f} | {np.mean(after[name]):.2f} |" if name in after else f"| {name} | {np.mean(x):.2f} | |")
    print(f"\n| {up.shape[1]} x {up.shape[0]} pixels | ms |\n|---|---|")
    for name, (m, pages) in models.items():
        if m.predictor == agpr.Predictor.BANK:
            agpr.BANK_PAGES = pages
            for n in (3, 10):
                torch.cuda.synchronize()
                t0 = time.time()
                for _ in range(n):
                    m._bank_detail(up)
                torch.cuda.synchronize()
            print(f"| {name} | {(time.time() - t0) / n * 1e3:.2f} |")
    shutil.rmtree(base)


if __name__ == "__main__":
    main()
