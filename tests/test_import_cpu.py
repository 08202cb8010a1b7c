"""The package imports, quantises and packs on a host whose torch was built without CUDA."""
import os
import subprocess
import sys

PROGRAM = """
import torch
gone = [n for n in dir(torch._C) if n.startswith("_cuda")]  # a CPU-only build has none of them
assert "_cuda_getDevice" in gone and "_cuda_getCurrentRawStream" in gone
import torch.cuda
for name in gone:
    delattr(torch._C, name)
import soinfer, soinfer.ops, soinfer.quant, soinfer.offload, soinfer.runtime
from soinfer.quant import formats, pack
qt = formats.quantize(torch.randn(8, 256), formats.QuantConfig(4, "group", 128))
assert pack.pack_int4(qt.qweight)[0].shape[0] == 8
k, v = soinfer.ops.paged_kv_alloc(1, 1, 16, 64, 16, "cpu")
try:
    soinfer.ops.paged_decode_attention(k[0], k, v, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
except RuntimeError as e:
    assert "CUDA" in str(e), e
else:
    raise SystemExit("not refused")
"""


def test_import_without_a_cuda_build_of_torch():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=os.path.join(root, "sparse-offload-infer_b200"))
    r = subprocess.run([sys.executable, "-c", PROGRAM], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
