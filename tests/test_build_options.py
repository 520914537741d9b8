"""The Makefile's compiler options, from what make would run."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "diff-surfel-tracing_amd", "csrc")


def _commands(*more):
    text = subprocess.run(["make", "-n", "-B", "-C", CSRC, *more], check=True, capture_output=True, text=True).stdout
    return {m.group(1): line for line in text.splitlines() for m in [re.search(r" -c (\w+)\.hip", line)] if m}


def test_options_of_the_command_line_come_beside_those_of_a_file():
    plain, more = _commands(), _commands("EXTRA=-DDST_STATS")
    assert set(plain) == {"dst_api", "lbvh", "trace", "labels", "attend"}
    for name, line in more.items():
        assert "-DDST_STATS" in line and "-packed-fp32-ops" in line
        assert ("-amdgpu-mfma-vgpr-form=1" in line) == (name in ("labels", "attend")), line
        assert sorted(line.replace("-DDST_STATS", "").split()) == sorted(plain[name].split())
