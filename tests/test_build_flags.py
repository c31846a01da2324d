"""How the library is compiled."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pointcloud_rl_amd", "csrc")


def test_no_object_may_hold_packed_fp32_arithmetic():
    """Every kernel source is compiled with the packed fp32 instructions switched off (Makefile), and none is written by hand."""
    plan = subprocess.run(["make", "-C", CSRC, "-n", "-B"], check=True, capture_output=True, text=True).stdout.replace("\\\n", " ")
    compiles = [line for line in plan.splitlines() if " -c " in line and ".hip" in line]
    sources = [f for f in os.listdir(CSRC) if f.endswith(".hip")]
    assert len(compiles) == len(sources) > 10
    for line in compiles:
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, line
    for name in os.listdir(CSRC):
        if name.endswith((".hip", ".h")):
            text = open(os.path.join(CSRC, name)).read()
            assert not any(f"v_pk_{op}_f32" in text for op in ("add", "mul", "fma")), name
