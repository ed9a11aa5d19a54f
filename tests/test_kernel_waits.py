"""Wait states that the hardware does not keep by itself, in every kernel's assembly, which the
library's own flags give: one between a write of M0 and a load into LDS, five between a vector
instruction's write of a scalar register and a memory instruction that reads it. The compiler
adds them between its own instructions, but not inside or in front of inline assembly. CPU only:
hipcc cross-compiles gfx950."""
import os
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_kernel_resources import CSRC, FLAGS, HIPCC

SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))
MEMORY = ("buffer_", "global_", "flat_", "scratch_")
TO_SCALAR = ("v_readlane", "v_readfirstlane", "v_cmp_", "v_cmpx_", "v_div_scale")
ENDS = ("s_branch", "s_endpgm", "s_setpc_b64", "s_trap")

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) and shutil.which("hipcc") is None,
                                reason="hipcc not available")


def _scalars(text):
    """Scalar registers named in an operand list."""
    out = set()
    for a, b, c in re.findall(r"(?<![a-z0-9_])s(?:\[(\d+):(\d+)\]|(\d+))", text):
        out |= set(range(int(a), int(b) + 1)) if a else {int(c)}
    if "vcc" in text:
        out.add("vcc")
    return out


def _functions(text):
    """(name, instructions, label -> index) of each function; an instruction is (mnemonic, operands)."""
    name, code, labels = None, [], {}
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        m = re.match(r"([.\w$]+):$", line)
        if m:
            if m[1].startswith("_Z"):
                if code:
                    yield name, code, labels
                name, code, labels = m[1], [], {}
            labels[m[1]] = len(code)
        elif line and not line.startswith(".") and name:
            parts = line.split(None, 1)
            code.append((parts[0], parts[1] if len(parts) > 1 else ""))
    if code:
        yield name, code, labels


def missing_waits(text):
    found = []
    for name, code, labels in _functions(text):
        sources = {}  # index -> branches that lead there
        for i, (op, args) in enumerate(code):
            if op.startswith(("s_cbranch", "s_branch")) and args in labels:
                sources.setdefault(labels[args], []).append(i)

        def before(i):
            if i > 0 and not code[i - 1][0].startswith(ENDS):
                yield i - 1
            yield from sources.get(i, ())

        for i, (op, args) in enumerate(code):
            if not op.startswith(MEMORY):
                continue
            to_lds = "load" in op and ("_lds_" in op or re.search(r"\blds\b", args))
            reads = _scalars(args)
            todo, seen = [(j, 0) for j in before(i)], set()
            while todo:
                j, states = todo.pop()
                if states >= 5 or (j, states) in seen:
                    continue
                seen.add((j, states))
                p, a = code[j]
                into = a.split(",")[0].strip()
                if to_lds and states < 1 and into == "m0":
                    found.append((name, i, f"{p} {a}", f"{op} {args}"))
                if p.startswith(TO_SCALAR) and reads & _scalars(into):
                    found.append((name, i, f"{p} {a}", f"{op} {args}"))
                states += int(a, 0) + 1 if p == "s_nop" else 1
                todo += [(k, states) for k in before(j)]
    return found


def test_the_check_sees_what_is_missing():
    head = "_Zk:\n"
    load = "\tbuffer_load_dword v1, s[0:3], 0 offen lds\n"
    assert missing_waits(head + "\ts_mov_b32 m0, s9\n" + load)
    assert not missing_waits(head + "\ts_mov_b32 m0, s9\n\ts_nop 0\n" + load)
    assert missing_waits(head + "\tv_readlane_b32 s2, v3, 1\n\ts_nop 3\n" + load)
    assert not missing_waits(head + "\tv_readlane_b32 s2, v3, 1\n\ts_nop 4\n" + load)
    assert not missing_waits(head + "\tv_readlane_b32 s4, v3, 1\n" + load)
    # around a loop
    loop = "\ts_nop 4\n.L1:\n" + load + "\ts_nop 0\n%s\ts_cbranch_scc1 .L1\n\ts_endpgm\n"
    assert missing_waits(head + loop % "\tv_readfirstlane_b32 s3, v1\n") and not missing_waits(head + loop % "")


def _assembly(src, out_dir):
    out = os.path.join(out_dir, src + ".s")
    flags = [f for f in FLAGS if f not in ("-c", "-Rpass-analysis=kernel-resource-usage")]
    r = subprocess.run([HIPCC, *flags, "-S", os.path.join(CSRC, src), "-o", out], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    with open(out) as f:
        return missing_waits(f.read())


def test_no_kernel_misses_one(tmp_path):
    with ThreadPoolExecutor(max_workers=max(1, (os.cpu_count() or 2) // 2)) as ex:
        for src, found in zip(SOURCES, ex.map(lambda s: _assembly(s, str(tmp_path)), SOURCES)):
            assert not found, (src, len(found), found[:3])
