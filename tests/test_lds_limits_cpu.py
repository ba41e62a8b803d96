"""A kernel's limit of dynamic LDS belongs to a device: no call site remembers for the whole process that it
has raised it, which would leave a second device of the process without."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "kotensor_amd" / "csrc"


def _without_comments(text):
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", text, flags=re.S))


def test_limits_are_raised_for_each_device():
    sites = {p.name: _without_comments(p.read_text()).count("hipFuncSetAttribute(") for p in sorted(CSRC.iterdir()) if p.suffix in (".hip", ".h")}
    # the shared helper, and the quantization's launches, which raise it every time
    assert {name: n for name, n in sites.items() if n} == {"kt_common.h": 1, "kt_quantize.hip": 1}
    helper = _without_comments((CSRC / "kt_common.h").read_text())
    body = helper[helper.index("int32_t allow_lds("):]
    body = body[:body.index("\n}\n")]
    assert "hipGetDevice" in body and "hipFuncSetAttribute" in body and "atomic<uint64_t>" in body
    quantize = _without_comments((CSRC / "kt_quantize.hip").read_text())
    body = quantize[quantize.index("static int32_t resident_grid("):]
    body = body[:body.index("\n}\n")]
    assert "hipFuncSetAttribute" in body and "static bool" not in body and "static std::atomic" not in body
