"""The microscaled product under the bounds-checking debug build (libsnnb200_check.so): tail
shapes of every form leave the device status word clear and give the release build's outputs."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "triton-pass-analysis_b200")

CASES = """
import sys
sys.path.insert(0, sys.argv[2])
import torch
from snn_compiler.kernels import conv as KC, mx
out, g = {}, torch.Generator().manual_seed(3)
for rows, N, K in ((1, 1, 1), (5, 131, 33), (30, 77, 520), (60, 260, 1000), (100, 129, 100),
                   (300, 1001, 300), (1300, 4097, 900)):
    for fmt in ("mxfp4", "mxfp8"):
        a = mx.mx_quantize(torch.randn(rows, K, generator=g).cuda(), fmt)
        w = mx.mx_quantize(torch.randn(N, K, generator=g).cuda())
        for dtype in (torch.bfloat16, torch.float32):
            out[f"{rows}x{N}x{K}{fmt}{dtype}"] = mx.mx_linear(a, w, dtype=dtype).cpu()
torch.cuda.synchronize()
out["status"] = torch.tensor(KC.device_status())
torch.save(out, sys.argv[1])
"""


def _run(tmp_path, name, library):
    path = str(tmp_path / f"{name}.pt")
    env = dict(os.environ)
    env.pop("SNNB_LIBRARY", None)
    if library:
        env["SNNB_LIBRARY"] = library
    subprocess.run([sys.executable, "-c", CASES, path, PKG], env=env, check=True, timeout=600)
    return torch.load(path)


def test_tail_shapes_of_the_product_pass_the_bounds_checks(tmp_path):
    check_lib = os.path.join(PKG, "libsnnb200_check.so")
    assert os.path.exists(check_lib), "build it with `make -C triton-pass-analysis_b200 check`"
    rel, chk = _run(tmp_path, "release", None), _run(tmp_path, "check", check_lib)
    assert int(rel["status"]) == 0 and int(chk["status"]) == 0
    assert rel.keys() == chk.keys()
    for k in rel:
        assert torch.equal(rel[k], chk[k]), k
