"""Instruction forms that no kernel of the product may hold, in the gfx950 assembly of all its units (no GPU needed:
hipcc cross-compiles).

* Writes through the scalar data cache (scalar stores and atomics, that cache's write-back and discard).  The cache is
  not coherent with the vector stores' path: what a wave leaves in it reaches memory only by a write-back that has to be
  issued, and waited for, by hand, and a wave that writes a line back can put old bytes over another wave's.
* Packed FP32 arithmetic, some forms of which have given wrong results on MI355X now and then.  The compiler makes it
  from ordinary float code, so the flags of the build take the instructions away; a probe that is built with other flags
  says so itself, at its kernels."""
import re
import shlex
import subprocess
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parent.parent / "libjxl-tiny_amd"
UNITS = sorted(p.stem for p in (PKG / "csrc").glob("*.hip"))

PROBES = sorted(p.name for p in (PKG.parent / "tools").glob("*.hip"))

PACKED_FP32 = re.compile(r"v_pk_(add|mul|fma)_f32")
SCALAR_CACHE_WRITE = re.compile(r"s_(buffer_|scratch_)?(store|atomic)_|s_dcache_(wb|discard)")


def _instructions(assembly):
    """The instructions of `assembly`, without comments, labels, directives and metadata."""
    code = assembly.split(".amdgpu_metadata", 1)[0]
    lines = (ln.split(";")[0].strip() for ln in code.splitlines())
    return [ln for ln in lines if ln and not ln.startswith(".") and not ln.endswith(":")]


@pytest.fixture(scope="module", params=UNITS)
def unit_instructions(request):
    target = "csrc/%s.s" % request.param
    r = subprocess.run(["make", "-C", str(PKG), target], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    insts = _instructions((PKG / target).read_text())
    assert any(i.startswith("s_endpgm") for i in insts)  # (there are kernels in it)
    return insts


def test_no_write_through_the_scalar_data_cache(unit_instructions):
    assert [i for i in unit_instructions if SCALAR_CACHE_WRITE.match(i)] == []


def test_no_packed_fp32_arithmetic(unit_instructions):
    assert [i for i in unit_instructions if PACKED_FP32.match(i)] == []


def test_the_builds_flags_take_packed_fp32_away(tmp_path):
    """With the flags of the product's build, a kernel on pairs of floats compiles to scalar arithmetic."""
    out = subprocess.run(["make", "-n", "-B", "-C", str(PKG), "csrc/%s.s" % UNITS[0]], capture_output=True, text=True, check=True).stdout
    line = next(ln for ln in out.splitlines() if "hipcc" in ln)
    source, target = tmp_path / "pairs.hip", tmp_path / "pairs.s"
    source.write_text("#include <hip/hip_runtime.h>\n"
                      "typedef float F2 __attribute__((ext_vector_type(2)));\n"
                      "__global__ void k(F2* p, F2 a) { p[threadIdx.x] = p[threadIdx.x] * a + a; }\n")
    cmd = [{"csrc/%s.s" % UNITS[0]: str(target), "csrc/%s.hip" % UNITS[0]: str(source)}.get(w, w) for w in shlex.split(line)]
    subprocess.run(cmd, check=True, capture_output=True)
    insts = _instructions(target.read_text())
    assert any(i.startswith("v_mul_f32") for i in insts) and not any(PACKED_FP32.match(i) for i in insts), insts


@pytest.mark.parametrize("probe", PROBES)
def test_no_probe_holds_either_form(probe, tmp_path):
    target = tmp_path / "probe.s"
    subprocess.run(["hipcc", "--offload-arch=gfx950", "-O3", "-ffp-contract=off", "-S", "--cuda-device-only", "-o", str(target),
                    str(PKG.parent / "tools" / probe)], check=True, capture_output=True)
    insts = _instructions(target.read_text())
    assert [i for i in insts if PACKED_FP32.match(i) or SCALAR_CACHE_WRITE.match(i)] == []
