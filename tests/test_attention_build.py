"""The attention kernels in the built library: a fixed order of instructions goes with registers for all values."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from kermac_amd import _backend, _build


def llvm(tool):
    found = shutil.which(tool) or f"/opt/rocm/llvm/bin/{tool}"
    if not Path(found).exists():
        pytest.skip(f"no {tool}")
    return found


def spills(tmp_path):
    return {name: count for name, (count, _) in metadata(tmp_path, b"attention_").items()}


def metadata(tmp_path, part):
    """{kernel: (spilled vector registers, accumulation registers)} from the library's code objects that hold `part`."""
    fat = tmp_path / "fat"
    subprocess.run([llvm("llvm-objcopy"), f"--dump-section=.hip_fatbin={fat}", str(_backend.LIB_PATH), str(tmp_path / "copy.so")], check=True)
    blob, found = fat.read_bytes(), {}
    for at in (m.start() for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", blob)):
        number = lambda offset: int.from_bytes(blob[offset:offset + 8], "little")
        entry = at + 32
        for _ in range(number(at + 24)):
            start, size, length = number(entry), number(entry + 8), number(entry + 16)
            target = blob[entry + 24:entry + 24 + length].decode()
            entry += 24 + length
            code = blob[at + start:at + start + size]
            if "gfx950" in target and part in code:
                path = tmp_path / f"{at}.co"
                path.write_bytes(code)
                notes = subprocess.run([llvm("llvm-readelf"), "--notes", str(path)], check=True, capture_output=True, text=True).stdout
                for kernel in re.split(r"\n\s+- \.agpr_count", notes)[1:]:
                    found[re.search(r"\.name:\s+(\S+)", kernel).group(1)] = (int(re.search(r"\.vgpr_spill_count:\s+(\d+)", kernel).group(1)),
                                                                               int(re.match(r":\s+(\d+)", kernel).group(1)))
    return found


def test_ordered_kernels_have_their_values_in_registers(tmp_path):
    found = spills(tmp_path)
    ordered = {name: count for name, count in found.items() if re.search(r"attention_(forward|grad_queries|grad_keys)\w*Lb1E+v", name)}
    # 64, 96 and 128 features in three types, three kernels
    assert len(ordered) == 27, sorted(found)
    assert not any(ordered.values()), {name: count for name, count in ordered.items() if count}
    # and none of the rest has the order: unaligned rows, rows of 256 features
    assert all(re.search(r"Li(64|96|128)ELb1E", name) for name in ordered)


def test_the_build_refuses_an_ordered_kernel_that_spills():
    def remark(name, spilled):
        return (f"a.hpp:1:1: remark: Function Name: {name} [-Rpass-analysis=kernel-resource-usage]\na.hpp:1:1: remark:     VGPRs: 256 [-R]\n"
                f"a.hpp:1:1: remark:     SGPRs Spill: 9 [-R]\na.hpp:1:1: remark:     VGPRs Spill: {spilled} [-R]\n")
    ordered, free = "_ZN3kmc17attention_forwardIfLi64ELb1ELb1EEEvNS_13AttentionArgsE", "_ZN3kmc17attention_forwardIfLi256ELb1ELb0EEEvNS_13AttentionArgsE"
    assert _build.ordered_kernels_that_spill(remark(ordered, 0) + remark(free, 80)) == []
    assert _build.ordered_kernels_that_spill(remark(free, 0) + remark(ordered, 1)) == [ordered]


def test_spilled_values_stay_out_of_accumulation_registers():
    """The compiler loses registers of values that it spills partly to accumulation registers: the units whose kernels spill with such registers are built without.

    All other kernels of the library that spill have none of them."""
    attention = [src for src, _, _ in _build._jobs() if _build.is_attention(src)]
    assert len(attention) == 6
    at = _build.ATTENTION_FLAGS.index("-amdgpu-spill-vgpr-to-agpr=0")
    assert _build.ATTENTION_FLAGS[at - 1] == "-mllvm"


def test_other_kernels_that_spill_have_no_accumulation_registers(tmp_path):
    """(the count of these registers that a kernel's metadata gives, beside its spills)"""
    for name, (count, accumulation) in metadata(tmp_path, b"").items():
        assert "attention_" in name or count == 0 or accumulation == 0, name
