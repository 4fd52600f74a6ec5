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


def vector_written_scalars(op, args):
    """Scalar registers that a vector instruction writes."""
    if op.startswith(("v_readfirstlane", "v_readlane", "v_cmp")):
        return scalars(args[0])
    if op.startswith(("v_mad_u64", "v_mad_i64", "v_div_scale", "v_add_co", "v_addc_co", "v_sub_co", "v_subb_co")):
        return scalars(args[1])
    return set()


def scalars(operand):
    one, many = re.fullmatch(r"s(\d+)", operand), re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    return {int(one.group(1))} if one else set(range(int(many.group(1)), int(many.group(2)) + 1)) if many else set()


def short_waits(lines, needed):
    """Loads into LDS that read a scalar register less than `needed` wait states behind a vector instruction that wrote it; the hardware does not wait, and the
    compiler, which does elsewhere, does not look into the assembly statements that these loads are written in."""
    found, at_target = set(), {}
    for _ in range(2):                                                  # twice: backward branches bring their state to labels that were passed
        pending = {}                                                    # register: wait states since
        for address, op, args, target in lines:
            for register, age in at_target.get(address, {}).items():
                pending[register] = min(age, pending.get(register, needed))
            if op.startswith("buffer_load") and "lds" in args[-1].split():
                if any(register in pending for register in scalars(args[1])):
                    found.add(address)
            states = int(args[0], 0) + 1 if op == "s_nop" else 1
            pending = {register: age + states for register, age in pending.items() if age + states < needed}
            for register in vector_written_scalars(op, args):
                pending[register] = 0
            if op.startswith("s_") and not op.startswith(("s_cmp", "s_cbranch", "s_nop", "s_waitcnt")) and args:
                for register in scalars(args[0]):
                    pending.pop(register, None)
            if target is not None:
                known = at_target.setdefault(target, {})
                for register, age in pending.items():
                    known[register] = min(age, known.get(register, needed))
    return found


def test_loads_into_lds_wait_for_their_descriptors(tmp_path):
    metadata(tmp_path, b"attention_")
    loads = 0
    for path in tmp_path.glob("*.co"):
        text = subprocess.run([llvm("llvm-objdump"), "-d", "--no-show-raw-insn", str(path)], check=True, capture_output=True, text=True).stdout
        for function in re.split(r"\n[0-9a-f]+ <(?=\w)", text)[1:]:
            name, lines, start = function.split(">", 1)[0], [], None
            for line in function.splitlines()[1:]:
                parsed = re.match(r"\s+(\w+)\s*(.*?)\s*// ([0-9A-F]+):(.*)$", line)
                if not parsed:
                    continue
                op, rest, address, behind = parsed.groups()
                address = int(address, 16)
                start = address if start is None else start
                jump = re.search(r"<[^>+]+(?:\+0x([0-9a-f]+))?>", behind) if op.startswith(("s_branch", "s_cbranch")) else None
                args = [x.strip() for x in re.split(r",(?![^\[]*\])", rest)] if rest else [""]
                lines.append((address, op, args, start + int(jump.group(1) or "0", 16) if jump else None))
                loads += op.startswith("buffer_load") and "lds" in rest.split()
            assert not short_waits(lines, 5), name
    assert loads > 100


def test_short_waits_are_found():
    def program(*texts):
        return [(4 * i, t.split(None, 1)[0], [x.strip() for x in re.split(r",(?![^\[]*\])", t.split(None, 1)[1])], None) for i, t in enumerate(texts)]
    load = "buffer_load_dwordx4 v5, s[12:15], 0 offen lds"
    assert short_waits(program("v_readfirstlane_b32 s13, v0", "s_mov_b32 m0, s3", "s_nop 0", load), 5) == {12}
    assert short_waits(program("v_readlane_b32 s15, v0, 3", "s_nop 4", load), 5) == set()
    assert short_waits(program("v_readfirstlane_b32 s16, v0", load), 5) == set()
    assert short_waits(program("v_readfirstlane_b32 s13, v0", "s_mov_b32 s13, s2", load), 5) == set()
    jump = program("s_nop 0", load, "v_readfirstlane_b32 s12, v0", "s_branch 0")
    assert short_waits(jump[:3] + [(12, "s_branch", ["0"], 0)], 5) == {4}
