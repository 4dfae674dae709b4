"""The product's build rules: what a change of them rebuilds, and the kernels' schedule as compiled by them.

tests/test_kernel_schedule.py compiles with flags of its own, packed fp32
arithmetic among them; here the commands come from the Makefile."""
import os
import re
import shlex
import subprocess

import pytest

import test_kernel_schedule as schedule
from conftest import REPO

CSRC = os.path.join(REPO, "geeps_amd", "csrc")
MAKEFILE = os.path.join(CSRC, "Makefile")
UNITS = {"gp_reduce", "gp_unplanned", "gp_sort", "gp_route", "gp_clip", "gp_runtime"}


def commands(*options):
    """The compile commands that make would run, by the name of their source."""
    out = subprocess.run(["make", "-n", "-C", CSRC, *options], capture_output=True, text=True, check=True).stdout
    found = {}
    for line in out.splitlines():
        words = line.split()
        sources = [w for w in words if re.search(r"/gp_\w+\.(hip|cpp)$", w)]
        if words and ("hipcc" in words[0] or "g++" in words[0]) and sources and "/geeps/" not in sources[0]:
            found[os.path.splitext(os.path.basename(sources[0]))[0]] = line
    return found


def test_a_change_of_the_rules_rebuilds_every_object():
    """A flag changed in the Makefile left objects of the old flags in an incremental build."""
    assert set(commands("-W", MAKEFILE)) == UNITS | {"gp_host", "gp_tensors"}


def test_no_unit_is_built_with_packed_arithmetic():
    for unit, line in commands("-B").items():
        assert unit not in UNITS or "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, unit


def test_no_app_is_built_with_packed_arithmetic(monkeypatch):
    """The test and benchmark apps hold kernels too, and so do the sanitizer builds of them."""
    import __graft_entry__ as entry
    lines = []
    monkeypatch.setattr(entry.subprocess, "run", lambda words, **_: lines.append(" ".join(words)))
    entry.build_apps()
    for script in ("build_ubsan.sh", "build_tsan.sh"):
        with open(os.path.join(REPO, "scripts", script)) as f:
            lines += f.read().replace("\\\n", " ").splitlines()
    hip = [line for line in lines if line.startswith("/opt/rocm/bin/hipcc")]
    assert len(hip) == 4
    for line in hip:
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, line


@pytest.fixture(scope="module")
def shipped(tmp_path_factory):
    """The assembly of both units over gp_kernels.hpp, by the Makefile's own commands."""
    if not os.path.exists(schedule.HIPCC):
        pytest.skip("hipcc not installed")
    d, lines = tmp_path_factory.mktemp("asm"), commands("-B")
    procs = []
    for unit in ("gp_unplanned", "gp_reduce"):
        words = shlex.split(lines[unit])
        words[words.index("-o") + 1] = str(d / f"{unit}.s")
        words[words.index("-c")] = "-S"
        procs.append(subprocess.Popen([*words, "--cuda-device-only"], stdout=subprocess.PIPE, stderr=subprocess.PIPE,
                                      cwd=str(d)))
    for p in procs:
        _, err = p.communicate()
        assert p.returncode == 0, err.decode()[-2000:]
    return "".join((d / f"{unit}.s").read_text() for unit in ("gp_unplanned", "gp_reduce"))


def test_no_packed_arithmetic_in_what_is_shipped(shipped):
    assert not re.findall(r"v_pk_(?:add|mul|fma)_f32", shipped)


@pytest.mark.parametrize("nb,rt,tg,zin,u", schedule.SWEEP_SHAPES)
def test_shipped_sweep_kernel_keeps_burst_schedule(shipped, nb, rt, tg, zin, u):
    schedule.test_sweep_kernel_keeps_burst_schedule(shipped, nb, rt, tg, zin, u)


@pytest.mark.parametrize("rt,tg,zin", [(14, 8, 0), (6, 4, 1), (6, 4, 0)])
def test_shipped_gated_sweep_kernel_keeps_burst_schedule(shipped, rt, tg, zin):
    schedule.test_gated_sweep_kernel_keeps_burst_schedule(shipped, rt, tg, zin)


def test_shipped_wave_kernels_fit_their_occupancy(shipped):
    schedule.test_wave_kernels_fit_their_occupancy(shipped)


def test_the_phased_sum_keeps_its_tiles_in_registers(shipped):
    """Unpacked adds once kept the register tiles' addends apart until the write phase, in 580 bytes of scratch a lane."""
    names = set(re.findall(r"^(_ZN12_GLOBAL__N_124bucket_sum_phased_kernel\S*):", shipped, re.M))
    assert names
    for name in names:
        sizes = re.findall(rf"\.set {re.escape(name)}\.private_seg_size, (\d+)", shipped)
        assert sizes and set(sizes) == {"0"}, (name, sizes)
        assert "scratch_" not in schedule._kernel(shipped, re.escape(name) + r"(?=:)"), name
