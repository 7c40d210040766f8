"""The microscaled tiles read LDS through inline asm with waits of their own (csrc/mx_gemm.hip). Until such a
read's wait the compiler must neither read its registers (it takes them as filled) nor write them (it may take
them as free): either would be wrong data now and then. This compiles the source to gfx950 assembly with the
library's flags and scans every kernel. CPU only; skipped without hipcc."""

from __future__ import annotations

import re
import shutil
import subprocess

import pytest

from rus_amd import build
from test_asm_lds_waits import early_reads

_VREG = re.compile(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b")


def _regs(text: str) -> set[str]:
    out: set[str] = set()
    for m in _VREG.finditer(text):
        if m.group(4):
            out.add(m.group(4) + m.group(5))
        else:
            out.update(f"{m.group(1)}{i}" for i in range(int(m.group(2)), int(m.group(3)) + 1))
    return out


def touched(asm: str) -> tuple[int, dict[str, list[str]]]:
    """(asm LDS reads seen, {kernel: what touches a register that such a read fills and no lgkmcnt(0) has
    covered}). A branch with reads in flight is listed too: a linear scan does not see where it leads."""
    lines = [l.strip() for l in asm.split("\n")]
    reads, found = 0, {}
    for fn in re.findall(r"^\s+\.type\s+(\w+),@function", asm, re.M):
        pending: set[str] = set()
        in_asm, bad = False, []
        for s in lines[lines.index(next(l for l in lines if l.startswith(fn + ":"))) + 1:]:
            if s.startswith("s_endpgm"):
                break
            if s.startswith(";;#ASM"):
                in_asm = s == ";;#ASMSTART"
                continue
            if not s or s.startswith((";", ".")) or s.split()[0].endswith(":"):
                continue
            op = s.split()[0]
            if op == "s_waitcnt" and "lgkmcnt(0)" in s:
                pending.clear()
            elif in_asm and op.startswith("ds_read"):
                into = _regs(s[len(op):].split(",")[0])
                if into & pending or _regs(s[len(op):].split(",", 1)[1]) & pending:
                    bad.append(s)
                pending |= into
                reads += 1
            elif op.startswith(("s_cbranch", "s_branch", "s_setpc")):
                if pending:
                    bad.append(s)
            elif pending & _regs(s[len(op):].split(";")[0]):
                bad.append(s)
        if bad:
            found[fn] = bad
    return reads, found


def _kernel(*body: str) -> str:
    asm = lambda s: [";;#ASMSTART", s, ";;#ASMEND"]
    out = ["\t.type\t_Zk,@function", "_Zk:", *asm("ds_read_b128 v[8:11], v2 offset:64")]
    for s in body:
        out += asm(s[1:]) if s.startswith("!") else [s]
    return "\n".join([*out, "s_endpgm"])


@pytest.mark.parametrize("body,bad", [
    (["!s_waitcnt lgkmcnt(0)", "v_mov_b32_e32 v20, v11", "v_mov_b32_e32 v9, 0"], 0),
    (["v_mov_b32_e32 v20, v11"], 1),  # read too early
    (["v_mov_b32_e32 v9, 0"], 1),  # overwritten by the load when it lands
    (["v_accvgpr_write_b32 a0, v10"], 1),  # spilled too early
    (["scratch_store_dwordx4 off, v[8:11], s0"], 1),
    (["!ds_read_u16 v8, v3 offset:2"], 1),  # two loads into one register
    (["s_cbranch_scc0 .LBB0_1"], 1),
    (["!s_waitcnt lgkmcnt(1)", "v_add_u32_e32 v20, v20, v8"], 1),  # not the wait that covers all
    (["v_mfma_f32_32x32x16_f16 a[0:15], v[12:15], v[4:7], a[0:15]", "s_add_u32 s0, s0, 1"], 0),
])
def test_scan_finds(body, bad):
    reads, found = touched(_kernel(*body))
    assert reads >= 1 and len(found.get("_Zk", [])) == bad


@pytest.mark.skipif(shutil.which("hipcc") is None and not build.Path("/opt/rocm/bin/hipcc").exists(),
                    reason="hipcc not available")
def test_no_register_is_touched_before_its_wait(tmp_path):
    out = tmp_path / "mx_gemm.s"
    cmd = [build.hipcc(), *build.HIPCC_FLAGS, "--offload-device-only", "-S", str(build.CSRC_DIR / "mx_gemm.hip"),
           "-o", str(out)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    text = out.read_text()
    reads, found = touched(text)
    assert reads > 1000 and found == {}
    assert early_reads(text) == {}
    # nothing is kept in scratch memory: a spill between a read and its wait would store stale data
    assert set(re.findall(r"\.private_segment_fixed_size:\s*(\d+)", text)) == {"0"}
