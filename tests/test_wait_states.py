"""Wait states in the built kernels, from their disassembly.

gfx950: a VGPR that a vector instruction writes may be read through DPP, and by v_permlane16_swap / v_permlane32_swap, two wait
states later at the earliest.  The compiler keeps that between its own instructions, but not behind inline assembly, which it
does not look into."""
import os
import re
import struct
import subprocess

import pytest

import shivae_amd
from shivae_amd import _native as N

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
NEED = 2


def _code_objects(path):
    """The gfx950 code objects of a library: bundles of (offset, size, target) entries, one bundle for each source."""
    data = open(path, "rb").read()
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + 24)
        pos = at + 32
        for _ in range(count):
            off, size, n = struct.unpack_from("<QQQ", data, pos)
            target = data[pos + 24:pos + 24 + n].decode()
            pos += 24 + n
            if target.endswith("gfx950") and size:
                yield data[at + off:at + off + size]
        at = data.find(MAGIC, at + 24)


def _registers(operand):
    """The VGPRs of an operand: v7, v[4:7]."""
    out = set()
    for lo, hi, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", operand):
        out |= {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return out


def missing_waits(listing):
    """-> (instructions that were checked, [(symbol, instruction, wait states)])."""
    age, symbol, checked, bad = {}, "", 0, []  # VGPR -> wait states since a vector instruction wrote it
    for line in listing:
        m = re.match(r"[0-9a-f]+ <(.*)>:", line)
        if m:
            symbol, age = m.group(1), {}
            continue
        text = line.split("//")[0].strip()
        parts = text.split(None, 1)
        if not parts or not re.match(r"[a-z]+_", parts[0]):
            continue
        op, operands = parts[0], parts[1].split(",") if len(parts) > 1 else []
        if op == "s_nop":
            age = {r: a + int(operands[0], 0) + 1 for r, a in age.items()}
            continue
        swap = op.startswith("v_permlane") and "_swap" in op
        reads = _registers(operands[0]) | _registers(operands[1]) if swap else _registers(operands[1]) if "_dpp" in op else set()
        if reads:
            checked += 1
            least = min([age.get(r, NEED) for r in reads])
            if least < NEED:
                bad.append((symbol, text, least))
        age = {r: a + 1 for r, a in age.items() if a + 1 < NEED}
        if op in ("s_branch", "s_endpgm", "s_setpc_b64"):
            age = {}
        if op.startswith("v_") and operands:
            for r in _registers(operands[0]) | (_registers(operands[1]) if swap else set()):
                age[r] = 0
        elif operands:  # loads: another counter
            for r in _registers(operands[0]):
                age.pop(r, None)
    return checked, bad


def test_the_check_itself():
    good = ["0000 <k>:", " v_add_f32_e32 v1, v2, v3 // 00", " s_nop 1", " v_permlane32_swap_b32_e32 v1, v4", " v_mov_b32_e32 v5, v6",
            " v_mov_b32_e32 v7, v6", " s_nop 0", " v_mul_f32_dpp v8, v5, v9 row_newbcast:1 row_mask:0xf bank_mask:0xf"]
    assert missing_waits(good) == (2, [])
    for drop, waits in ((2, 0), (6, 1)):
        checked, bad = missing_waits(good[:drop] + good[drop + 1:])
        assert checked == 2 and [b[2] for b in bad] == [waits]


def test_results_are_ready_when_lanes_are_exchanged(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    N.lib()
    checked, bad = 0, []
    for i, code in enumerate(_code_objects(os.path.join(os.path.dirname(shivae_amd.ssm.__file__), "libshivae_hip.so"))):
        path = tmp_path / ("%d.co" % i)
        path.write_bytes(code)
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], check=True, capture_output=True, text=True).stdout
        n, b = missing_waits(listing.splitlines())
        checked, bad = checked + n, bad + b
    assert checked > 5000
    assert not bad, "%d of %d, first %s" % (len(bad), checked, bad[:3])
