"""The library's build description: what it compiles again, and with which flags."""
import os
import subprocess

import pytest

from helpers import ROOT

CSRC = os.path.join(ROOT, "yolo_amd", "csrc")
UNITS = sorted(f[:-4] for f in os.listdir(CSRC) if f.endswith(".hip"))
NO_TWO_VALUE_FP32 = "-Xclang -target-feature -Xclang -packed-fp32-ops"


def make(*args):
    return subprocess.run(["make", "--no-print-directory", "-C", CSRC, *args], capture_output=True, text=True, check=True).stdout


@pytest.mark.parametrize("what", ["Makefile", "rows_common.h"])
def test_objects_follow_the_flags_and_the_headers(what):
    """A changed Makefile compiles every unit again, as a changed header does (nothing is run: -n prints)."""
    lines = [l for l in make("-n", "-W", os.path.join(CSRC, what) if what == "Makefile" else what).splitlines() if " -c " in l]
    assert sorted(l.split(" -c ")[1].split()[0] for l in lines) == [u + ".hip" for u in UNITS]
    assert all(NO_TWO_VALUE_FP32 in l for l in lines)


def test_variants_and_tools_are_compiled_like_the_library():
    for unit in UNITS:
        flags = make("-s", "flags-" + unit)
        assert NO_TWO_VALUE_FP32 in flags and "--offload-arch=gfx950 -O3" in flags
        assert ("-ffp-contract=off" in flags) == (unit in ("decode", "nms", "nms_flavours", "preproc"))
    with open(os.path.join(ROOT, "tools", "build_variant.sh")) as fh:
        text = fh.read()
    assert "flags-$unit" in text and "-O3" not in text
    for f in sorted(os.listdir(os.path.join(ROOT, "tools"))):
        if f.endswith(".hip"):
            with open(os.path.join(ROOT, "tools", f)) as fh:
                recipe = [l for l in fh if "hipcc" in l]
            assert recipe and all(NO_TWO_VALUE_FP32 in l for l in recipe), f
