"""The non-temporal LDS DMA helper carries its wait states as the others do (test_lds_dma_waits.py)."""

import importlib.util
import subprocess

from test_lds_dma_waits import CSRC, PROBE, _waits


def test_non_temporal_dma_waits(tmp_path):
    spec = importlib.util.spec_from_file_location("esep_build", CSRC.parent / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    src = tmp_path / "probe.hip"
    src.write_text(PROBE.replace("lds_dma_x4_s(", "lds_dma_x4_s_nt("))
    res = subprocess.run([build.HIPCC, *build.CFLAGS, "--cuda-device-only", "-S", str(src), "-o", "-"],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    loads = [(ins, states) for ins, states in _waits(res.stdout) if ins.endswith(" nt")]
    assert len(loads) >= 2, res.stdout
    for ins, states in loads:
        assert states >= 5, (ins, states)
