"""Which sources a record of HBM counters speaks for (bench.py kernel_sources_sha16)."""
import os
import shutil

import pytest


@pytest.mark.parametrize("changed,same", [("k_sample.hip", True), ("k_cacheattn.hip", True), ("ps_serve.h", True), ("k_moe.hip", True), ("new_operator.hip", True), ("k_gemv4.hip", False), ("ps_gemv_dev.h", False),
                                          ("ps_expf.h", False), ("ctx.hip", False), ("k_quant.hip", False)])
def test_a_record_speaks_for_the_kernels_that_it_was_taken_on(changed, same, tmp_path, monkeypatch):
    """another operator's sources do not void it, a source or header of the quantized path's kernels does"""
    import bench
    from powerserve_amd import build
    csrc = tmp_path / "csrc"
    shutil.copytree(build.CSRC, csrc)
    want = bench.kernel_sources_sha16()
    monkeypatch.setattr(build, "CSRC", str(csrc))
    assert bench.kernel_sources_sha16() == want
    with open(os.path.join(csrc, changed), "a") as f:
        f.write("// a line more\n")
    assert (bench.kernel_sources_sha16() == want) == same
