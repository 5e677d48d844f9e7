"""One case of perf/operators.py after the other on the framework's own kernels, a dozen passes each: for
    rocprofv3 --kernel-trace --stats --output-format csv -d DIR -o p -- python3 tools/bank_cases.py [NAME ...]
("windows" and "blend": a 3840 x 2160 image in windows of 7 x 7 pixels, and back.)  Prints each case's time a pass."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT]
from perf import operators  # noqa: E402
from super_resolution_amd import ops  # noqa: E402


def timed(name, f):
    for i in range(4):
        f(i)
    a, b = torch.cuda.Event(True), torch.cuda.Event(True)
    a.record()
    for i in range(8):
        f(i)
    b.record()
    torch.cuda.synchronize()
    print(f"{name:20s} {a.elapsed_time(b) / 8 * 1e3:9.1f} us", flush=True)


def main(names):
    operators.own = True
    for c in operators.listed():
        if not names or c["name"] in names:
            states = [operators.prepare(c, i) for i in range(2)]
            timed(c["name"], lambda i: operators.run(states[i % 2]))
    img = torch.rand(2160, 3840, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    if not names or "windows" in names:
        timed("windows", lambda i: ops.bank_windows(img, 7, 64, centre=True))
    if not names or "blend" in names:
        rows = ops.bank_windows(img, 7, 64, centre=True)
        timed("blend", lambda i: ops.bank_blend(img, rows, 7))


if __name__ == "__main__":
    main(sys.argv[1:])
