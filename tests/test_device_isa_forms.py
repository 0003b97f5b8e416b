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


# ---- LDS loads that are written in assembly ahead of their wait (JXLT_LDS_LOAD4_NOW_AT, jxlt_device_common.h) ----

REGISTER = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")
LDS_OP = re.compile(r"ds_(?!nop)")
SCALAR_LOAD = re.compile(r"s_(buffer_)?load_|s_memtime|s_memrealtime|s_dcache_inv")


def _registers(text):
    regs = set()
    for kind, one, lo, hi in REGISTER.findall(text):
        regs.update((kind, r) for r in (range(int(lo), int(hi) + 1) if lo else [int(one)]))
    return regs


def _kernels(assembly):
    """{symbol: [(label or None, instruction, written in assembly)]}: an instruction per entry, labels on their own."""
    out = {}
    for m in re.finditer(r"^(_Z\w+):[^\n]*\n(.*?)^\s*\.amdhsa_kernel ", assembly.split(".amdgpu_metadata", 1)[0], re.S | re.M):
        body, by_hand = [], False
        for raw in m.group(2).splitlines():
            if "#ASMSTART" in raw or "#ASMEND" in raw:
                by_hand = "#ASMSTART" in raw
                continue
            ln = raw.split(";")[0].strip()
            if ln.endswith(":"):
                body.append((ln[:-1], None, False))
            elif ln and not ln.startswith("."):
                body.append((None, ln, by_hand))
        out[m.group(1)] = body
    return out


def _touched_in_flight(body):
    """The instructions that touch a register which a hand-written LDS load may not have filled yet, on any path.

    A path's state is what counts towards lgkmcnt, oldest first: a frozenset of registers for a hand-written load, an
    empty one for the compiler's own LDS operations (it waits for those itself), None for scalar loads, which return
    out of order -- only a wait for zero says anything while one is on its way."""
    label = {lb: k for k, (lb, _, _) in enumerate(body) if lb}
    starts = [k for k, (_, i, by_hand) in enumerate(body) if i and by_hand and i.startswith("ds_read")]
    bad, seen, todo = set(), set(), [(k, ()) for k in starts]
    while todo:
        k, state = todo.pop()
        while k < len(body) and (k, state) not in seen:
            seen.add((k, state))
            _, inst, by_hand = body[k]
            if inst is None:
                k += 1
                continue
            wait = re.match(r"s_waitcnt\b.*lgkmcnt\((\d+)\)", inst)
            if wait:
                n = int(wait.group(1))
                if n == 0 or None not in state:
                    state = state[len(state) - n:] if n else ()
            else:
                operands = inst.split(None, 1)[1] if " " in inst or "\t" in inst else ""
                busy = set().union(*(s for s in state if s))
                if _registers(operands) & busy:
                    bad.add((k, inst))
                if LDS_OP.match(inst):
                    state += (frozenset(_registers(operands.split(",", 1)[0])) if by_hand and inst.startswith("ds_read") else frozenset(),)
                elif SCALAR_LOAD.match(inst):
                    state += (None,)
            if not any(state):
                break  # (no hand-written load is on its way any more)
            target = re.match(r"s_c?branch\w*\s+(\S+)", inst)
            if target:
                todo.append((label[target.group(1)], state))
                if inst.startswith("s_branch"):
                    break
            k += 1
    return sorted(bad)


def test_the_walk_finds_a_register_that_is_touched_too_early():
    load = (None, "ds_read_b128 v[4:7], v1 offset:0", True)
    wait = (None, "s_waitcnt lgkmcnt(0)", True)
    use = (None, "v_add_f32_e32 v9, v5, v2", False)
    assert _touched_in_flight([load, wait, use]) == []
    assert _touched_in_flight([load, use, wait]) == [(1, use[1])]
    assert _touched_in_flight([load, (None, "scratch_store_dword off, v7, off", False), wait])
    assert _touched_in_flight([load, (None, "v_mov_b32_e32 v4, 0", False), wait])
    # a newer operation of the compiler's own, and a wait that leaves it on its way
    newer = (None, "ds_read_b32 v8, v1", False)
    assert _touched_in_flight([load, newer, (None, "s_waitcnt lgkmcnt(1)", False), use]) == []
    assert _touched_in_flight([load, newer, (None, "s_waitcnt lgkmcnt(2)", False), use])
    # a scalar load may return first
    assert _touched_in_flight([load, (None, "s_load_dword s0, s[2:3], 0x0", False), (None, "s_waitcnt lgkmcnt(1)", False), use])
    # the path round the wait
    assert _touched_in_flight([load, (None, "s_cbranch_scc1 .LBB0_1", False), wait, (".LBB0_1", None, False), use])


@pytest.fixture(scope="module")
def encode_unit_kernels():
    r = subprocess.run(["make", "-C", str(PKG), "csrc/jxlt_capi_encode.s"], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    return _kernels((PKG / "csrc" / "jxlt_capi_encode.s").read_text())


def test_no_register_of_a_load_in_flight_is_touched(encode_unit_kernels):
    """The compiler takes the registers of a hand-written load as filled at once: what keeps it from using, moving or
    spilling them before the wait is only how the loop is written, so the assembly that ships is walked."""
    with_loads = {s: b for s, b in encode_unit_kernels.items() if any(h and i.startswith("ds_read") for _, i, h in b if i)}
    assert any("tile12_kernelE" in s for s in with_loads)
    assert {s: _touched_in_flight(b) for s, b in with_loads.items()} == {s: [] for s in with_loads}
