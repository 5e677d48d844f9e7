"""Where the cycles of a k_update2 compute wave go (off-diagonal trailing tiles, the bulk of the launch).
Needs the instrumented build:
    hipcc -O3 --offload-arch=gfx950 -shared -fPIC -ffp-contract=off -DGPSR_UPD_TRACE=<1|2|3> \
          -Xclang -target-feature -Xclang -packed-fp32-ops \
          -o super_resolution_amd/libgpsr_trace.so super_resolution_amd/csrc/*.hip
    GPSR_LIB=$PWD/super_resolution_amd/libgpsr_trace.so python tools/upd_trace.py [B N]
"""
import ctypes, os, sys
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch
from super_resolution_amd import _lib, ops
B = int(sys.argv[1]) if len(sys.argv) > 1 else 633
N = int(sys.argv[2]) if len(sys.argv) > 2 else 784
lib = _lib.load()
lib.gpsr_debug_upd_trace.restype = ctypes.c_int
lib.gpsr_debug_upd_trace.argtypes = [ctypes.c_void_p]
dev = torch.device("cuda:0")
g = torch.Generator(device=dev); g.manual_seed(0)
Q = torch.randn((B, N, 64), dtype=torch.float64, device=dev, generator=g)
A0 = Q @ Q.transpose(1, 2) / 64 + 0.5 * torch.eye(N, dtype=torch.float64, device=dev)
A = A0.clone(); ops.invert_(A); torch.cuda.synchronize()
buf = (ctypes.c_ulonglong * 8)()
lib.gpsr_debug_upd_trace(buf)          # clear
ops.profile_begin(4096)
A = A0.clone(); ops.invert_(A); torch.cuda.synchronize()
p = ops.profile_end()
lib.gpsr_debug_upd_trace(buf)
n = max(1, buf[0])
names = ["wave-tiles", "entry->exit", "wait own DMA", "wait barrier", "issue DMA", "LDS reads + MFMAs", "entry->first wait", "last MFMA->stores retired"]
print("k_update2:", p.get("update2"))
for i, nm in enumerate(names):
    print(f"  {nm:28s} {buf[i] / n if i else buf[i]:12.0f}" + ("" if i == 0 else f"  cycles per wave-tile ({100.0 * buf[i] / max(1, buf[1]):.1f} %)"))
print("  a full K=224 tile needs 14 chunks x 28 MFMAs x 64 cycles = 25088 MFMA-pipe cycles per wave")
