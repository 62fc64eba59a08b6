"""What the build asks of the compiler's output."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def build_module():
    spec = importlib.util.spec_from_file_location("_knhip_build_checks", os.path.join(ROOT, "kyanite_amd", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _report(*kernels):
    return "".join(f"a.hip:1:0: remark: Function Name: {name} [-Rpass-analysis=kernel-resource-usage]\n"
                   f"a.hip:1:0: remark:     VGPRs: 256 [-Rpass-analysis=kernel-resource-usage]\n"
                   f"a.hip:1:0: remark:     AGPRs: {n} [-Rpass-analysis=kernel-resource-usage]\n" for name, n in kernels)


def test_kernels_without_agprs_pass(build_module):
    build_module.check_no_agprs("a.hip", _report(("one", 0), ("two", 0)))


def test_a_kernel_with_agprs_fails_the_build(build_module):
    with pytest.raises(RuntimeError, match="two: 16"):
        build_module.check_no_agprs("a.hip", _report(("one", 0), ("two", 16)))


@pytest.mark.parametrize("report", ["", "warning: unknown argument", "remark: Function Name: one"])
def test_a_missing_report_fails_the_build(report, build_module):
    with pytest.raises(RuntimeError, match="no report"):
        build_module.check_no_agprs("a.hip", report)


def test_a_compile_with_agprs_leaves_no_object(build_module, monkeypatch, tmp_path):
    """(a small kernel in the place of the attention's, and a compiler's report with AGPRs)"""
    monkeypatch.setattr(build_module, "CSRC", str(tmp_path))
    monkeypatch.setattr(build_module, "BUILD_DIR", str(tmp_path))
    (tmp_path / "small.hip").write_text("#include <hip/hip_runtime.h>\n__global__ void small_kernel(float *x) { x[threadIdx.x] = 1.0f; }\n")
    monkeypatch.setattr(build_module, "RESULTS_IN_VGPRS", ["small.hip"])
    assert os.path.exists(build_module._compile("small.hip", False, ""))
    monkeypatch.setattr(build_module, "check_no_agprs", lambda src, report: (_ for _ in ()).throw(RuntimeError("AGPRs")))
    with pytest.raises(RuntimeError, match="AGPRs"):
        build_module._compile("small.hip", True, "")
    assert not os.path.exists(tmp_path / "small.hip.o")
