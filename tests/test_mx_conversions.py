"""The conversions of a whole block (32 elements to or from 6 bits) write their
result while they still read, so no register may be both: looked up in the device
code that the compiler makes of mx_quantize.hip, with the build's flags and without
optimisation, where registers are given out least carefully."""

from __future__ import annotations

import os
import re
import subprocess

import pytest

from mote_amd import build

WIDE = re.compile(r"^\s*v_cvt_scalef32_(?:pk32_\w+|2xpk16_\w+)\s+(.*)$", re.M)


def registers(operand):
    found = re.fullmatch(r"v\[(\d+):(\d+)\]|v(\d+)", operand.strip())
    if not found:
        return set()  # a constant or a scalar
    first, last, one = found.groups()
    return {int(one)} if one else set(range(int(first), int(last) + 1))


@pytest.mark.parametrize("level", ["-O0", "-O1", "-O3"])
def test_results_share_no_register_with_operands(tmp_path, level):
    out = tmp_path / "mx_quantize.s"
    flags = [f for f in build.COMMON_FLAGS if not f.startswith("-O")]
    subprocess.run([build.HIPCC, *flags, level, f"-I{build.CSRC}", "--cuda-device-only", "-S",
                    os.path.join(build.CSRC, "mx_quantize.hip"), "-o", str(out)], check=True, capture_output=True)
    conversions = [line.split(";")[0].split(", ") for line in WIDE.findall(out.read_text())]
    assert len(conversions) >= 4  # f16 and f32, there and back
    for result, *operands in conversions:
        assert len(registers(result)) in (6, 32)
        for operand in operands:
            assert not registers(result) & registers(operand), (result, operands)
