"""The kernels as they are compiled: registers that come back while lanes are missing.

A wave takes both sides of a branch with the lanes of each in EXEC; a side without lanes is jumped over (s_cbranch_execz).  Where
the end of an inner branch and the end of the one around it fall together, the compiler restores EXEC once, at the outer end, and lets the
jump go straight there.  A register that was spilled and comes back between the two then comes back in no lane, and the lanes that the outer
end restores go on with what the register held in between.  That has happened in a kernel with 512 registers and spills: its
lanes took results for row numbers and stored at addresses made of them.  Registers that come back are put in late, so
no source shows it; here the library is looked through for it.  (scratch_load: no kernel has arrays in scratch memory,
so these are registers that come back.)"""
import os
import re
import struct
import subprocess
from concurrent.futures import ProcessPoolExecutor

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "deep-learning-math-kernel-research_amd", "libeuler_hip.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"

VECTOR = ("v_", "global_", "scratch_", "ds_", "buffer_", "flat_")
SCALAR_RESULT = ("v_readlane", "v_readfirstlane", "v_writelane", "v_cmp")   # (a compare without lanes is 0, as it should be)


def narrows(t):
    """t takes lanes out of EXEC, or may"""
    return "saveexec" in t or t.startswith(("s_and_b64 exec,", "s_andn2_b64 exec,", "s_xor_b64 exec,", "s_mov_b64 exec,"))


def without_lanes(code):
    """Vector instructions of [instruction or "label:"] that a wave reaches by a jump for having no lanes before EXEC is restored; and
    scratch_loads behind a branch whose end is not the one that restores EXEC next."""
    ins, labels = [], {}
    for t in code:
        if t.endswith(":"):
            labels[t[:-1]] = len(ins)
        else:
            ins.append(t)
    starts, found = set(labels.values()), []
    for i, t in enumerate(ins):
        if t.startswith("s_cbranch_execz"):
            j = i   # only where this block took the lanes away: elsewhere it is a jump that is never taken
            while j > 0 and j not in starts and not ins[j - 1].startswith(("s_cbranch", "s_branch", "s_or_b64 exec")) and not narrows(ins[j - 1]):
                j -= 1
            if j == 0 or j in starts or not narrows(ins[j - 1]):
                continue
            p, seen = labels.get(t.split()[1], len(ins)), set()
            todo = [p]
            while todo:
                p = todo.pop()
                while p < len(ins) and p not in seen:
                    seen.add(p)
                    q = ins[p]
                    if narrows(q) or q.startswith(("s_or_b64 exec,", "s_endpgm")):
                        break
                    if q.startswith(("s_branch", "s_cbranch_execz")):
                        p = labels.get(q.split()[1], len(ins))
                        continue
                    if q.startswith("s_cbranch") and not q.startswith("s_cbranch_execnz"):
                        todo.append(labels.get(q.split()[1], len(ins)))
                    if q.startswith(VECTOR) and not q.startswith(SCALAR_RESULT):
                        found.append(q)
                    p += 1
        elif t.startswith("scratch_load"):
            dst = registers(t.split(",")[0])
            p = i + 1
            while p < len(ins) and not ins[p].startswith(("s_branch", "s_endpgm", "s_or_b64 exec,")) and not narrows(ins[p]) and not (
                    dst & registers(ins[p])):
                p += 1
            if p == len(ins) or not ins[p].startswith("s_or_b64 exec,"):
                continue
            j = i - 1
            while j >= 0 and not narrows(ins[j]) and not ins[j].startswith(("s_branch", "s_or_b64 exec,")):
                j -= 1
            if j >= 0 and "saveexec" in ins[j] and ins[j].split()[1].rstrip(",") != ins[p].split()[-1]:
                found.append(t)
    return found


def m0_for_others(code):
    """k_linear_tile writes m0 in inline assembly, for the load into LDS behind it: nothing else may use m0 there, nor reach LDS by
    addresses that are looked up (flat_*), whose waits would be others"""
    found = [t for t in code if t.startswith("flat_")]
    for i, t in enumerate(code):
        own = t.startswith("s_mov_b32 m0,") and [c.split()[0] for c in code[i + 1:i + 3]] == ["s_nop", "global_load_lds_dwordx4"]
        if re.search(r"\bm0\b", t) and not own or t.startswith("global_load_lds") and not code[i - 2].startswith("s_mov_b32 m0,"):
            found.append(t)
    return found


def registers(t):
    out = set()
    for a, lo, hi, n in re.findall(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)", t):
        out |= {a + n} if n else {a + str(i) for i in range(int(lo), int(hi) + 1)}
    return out


def code_objects(path):
    data = open(path, "rb").read()
    for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", data):
        at = m.start()
        q = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            off, size, name = struct.unpack_from("<QQQ", data, q)
            if b"gfx950" in data[q + 24:q + 24 + name] and size:
                yield data[at + off:at + off + size]
            q += 24 + name


def look_through(path):
    """(kernels, {kernel: what was found}) of a code object"""
    text = subprocess.run([OBJDUMP, "-d", "--symbolize-operands", "--no-show-raw-insn", path], capture_output=True, text=True, check=True).stdout
    kernels, bad, name, code = 0, {}, None, []
    for line in text.splitlines() + ["0 <>:"]:
        if line.startswith(("\t", " ")):
            code.append(line.split("//")[0].strip().replace("<", "").replace(">", ""))
        elif line.endswith(">:"):
            label = line[line.rindex("<") + 1:-2]
            if re.fullmatch(r"L\d+", label):
                code.append(label + ":")
                continue
            if name:
                kernels += 1
                found = without_lanes(code) + (m0_for_others(code) if "k_linear_tile" in name else [])
                if found:
                    bad[name] = found
            name, code = label, []
    return kernels, bad


def test_the_rule_finds_what_it_is_for():
    """the end of a store of rows, as the kernel had it, and with the register back where it belongs"""
    wrong = ["s_and_saveexec_b64 s[90:91], vcc", "s_cbranch_execz L9", "v_mov_b32_e32 v18, v4", "s_and_saveexec_b64 s[0:1], s[4:5]", "s_cbranch_execz L8",
             "global_store_dword v[0:1], v68, off", "L7:", "s_or_b64 exec, exec, s[0:1]", "L8:", "scratch_load_dwordx2 v[18:19], off, off offset:16",
             "L9:", "s_or_b64 exec, exec, s[90:91]", "v_lshl_add_u64 v[0:1], v[18:19], 0, s[0:1]", "s_endpgm"]
    assert without_lanes(wrong) == ["scratch_load_dwordx2 v[18:19], off, off offset:16"]
    assert without_lanes([t.replace("execz L8", "execz L7") for t in wrong]) == []
    # no jump, and no restoring between
    short = [t for t in wrong if t not in ("s_cbranch_execz L8", "L7:", "s_or_b64 exec, exec, s[0:1]", "L8:")]
    assert without_lanes(short) == ["scratch_load_dwordx2 v[18:19], off, off offset:16"]


def test_no_register_comes_back_without_lanes(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    paths = []
    for i, data in enumerate(code_objects(LIB)):
        paths.append(str(tmp_path / ("%d.co" % i)))
        open(paths[-1], "wb").write(data)
    kernels, bad = 0, {}
    with ProcessPoolExecutor(4) as pool:
        for n, b in pool.map(look_through, sorted(paths, key=os.path.getsize, reverse=True)):
            kernels += n
            bad.update(b)
    assert kernels > 500
    assert not bad, bad
