"""CPU test of how the suite goes without the reference's sources."""
from __future__ import annotations

import os
import subprocess
import sys

import oracle

HERE = os.path.dirname(os.path.abspath(__file__))


def _reports(root):
    env = dict(os.environ, MX_REFERENCE_ROOT=str(root), CUDA_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-rsfE", "-p", "no:cacheprovider",
                        os.path.join(HERE, "test_gemm_gpu.py"), "-k", "vs_reference_cuda_matmul and 512"],
                       capture_output=True, text=True, env=env, cwd=os.path.dirname(HERE), timeout=300)
    return r.returncode, r.stdout


def test_without_the_references_library(tmp_path):
    """Skipped where its sources are absent too, so that the tests behind are
    reached; not skipped where it could be built."""
    if os.path.exists(oracle.reference_gpu_lib_path()):
        return  # the comparisons run
    rc, out = _reports(tmp_path)
    assert rc == 0 and "skipped" in out and "sources" in out, out
    src = tmp_path / "moonxi-net-gpu" / "cuda"
    src.mkdir(parents=True)
    (src / "cuda_kernels.cu").write_text("")
    rc, out = _reports(tmp_path)
    assert rc != 0 and "skipped" not in out, out  # no device here, and no library
