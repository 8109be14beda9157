"""The built kernels leave an MFMA's result alone until it is there.

On gfx950 a vector instruction that reads an MFMA's result too soon gets what the register held
before: the compiler has to put other work, or s_nop, in between. It counts those issue slots
through branches, but not always (a branch between a product and the scaling of its sum has lost
them, at -O3 of ROCm 7.2), and a kernel built that way is wrong only now and then. So the
listing of every build is read: what the compiler keeps between the two in straight
code is the least that any path may have.
"""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

LIB = Path(__file__).resolve().parent.parent / "llms_amd" / "libllms_amd_fp.so"
OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
LIMIT = 20  # issue slots that a path is followed for


def regs(operand):
    """The vector registers of an operand, as (file, number)."""
    m = re.match(r"[-|]*([va])(?:(\d+)|\[(\d+):(\d+)\])", operand.strip())
    if not m:
        return frozenset()
    lo = int(m[2] or m[3])
    return frozenset((m[1], i) for i in range(lo, int(m[4] or lo) + 1))


def kernels(listing):
    """(name, instructions) of a listing, an instruction as (operation, operands' registers,
    target's index or None, slots it takes)."""
    name, base, raw = None, 0, []
    for line in listing.splitlines() + ["0 <end>:"]:
        head = re.match(r"([0-9a-f]+) <(.+)>:$", line)
        if head:
            if raw:
                at = {a: i for i, (a, *_) in enumerate(raw)}
                yield name, [(op, r, at.get(base + t) if t is not None and op.startswith(("s_branch", "s_cbranch"))
                              else None, n) for _, op, r, t, n in raw]
            name, base, raw = head[2], int(head[1], 16), []
            continue
        m = re.match(r"\t(\S+)\s*(.*?)\s*// ([0-9A-F]+):(?:.*\+0x([0-9a-f]+)>)?", line)
        if m:
            n = int(m[2]) + 1 if m[1] == "s_nop" else 1
            raw.append((int(m[3], 16), m[1], [regs(o) for o in m[2].split(",")], int(m[4], 16) if m[4] else None, n))


def reads(op, r):
    """The registers that an instruction reads."""
    if not r:
        return frozenset()
    whole = op.startswith(("ds_write", "ds_add", "v_cmp")) or "store" in op or "atomic" in op or "mac_" in op or "swap" in op
    return frozenset().union(*(r if whole else r[1:]))


def early(ins):
    """For each MFMA and path to the first reader of its result: (operation, slots between,
    whether the path passes a branch or a branch's target, index). A following MFMA's sum
    operand is left out: the matrix core waits for that itself."""
    targets = {t for _, _, t, _ in ins if t is not None}
    for k, (op, r, _, _) in enumerate(ins):
        if not op.startswith("v_mfma"):
            continue
        dst, todo, seen = r[0], [(k + 1, 0, False)], set()
        while todo:
            p, slots, branch = todo.pop()
            if p >= len(ins) or slots >= LIMIT or (p, slots, branch) in seen:
                continue
            seen.add((p, slots, branch))
            branch = branch or p in targets
            o, rr, target, n = ins[p]
            if o.startswith("s_endpgm"):
                continue
            if o.startswith("v_mfma"):
                if (rr[1] | rr[2]) & dst:
                    yield op, slots, branch, k
                    continue
                if (rr[0] | rr[3]) & dst:
                    continue
            elif reads(o, rr) & dst:
                yield op, slots, branch, k
                continue
            elif rr and rr[0] & dst:
                continue
            if target is not None:
                todo.append((target, slots + 1, True))
                if o == "s_branch":
                    continue
                branch = True
            todo.append((p + 1, slots + n, branch))


def test_the_walk_sees_a_branch():
    listing = """
0000000000000000 <k>:
\tv_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[0:3] // 000000000000: 00000000 00000000
\ts_nop 3                                                    // 000000000008: 00000000
\ts_cbranch_scc1 2                                           // 00000000000C: 00000000 <k+0x18>
\ts_nop 7                                                    // 000000000010: 00000000
\tv_add_f32_e32 v4, v5, v6                                   // 000000000014: 00000000
\tv_mul_f32_e32 v4, v5, v2                                   // 000000000018: 00000000
\ts_endpgm                                                   // 00000000001C: 00000000
"""
    (_, ins), = kernels(listing)
    assert sorted((n, b) for _, n, b, _ in early(ins)) == [(5, True), (14, True)]


@pytest.mark.skipif(not OBJDUMP.exists(), reason="no llvm-objdump")
def test_no_result_is_read_early(tmp_path):
    if not LIB.exists():
        pytest.skip("the library is not built")
    shutil.copy(LIB, tmp_path / "lib.so")  # the parts are written beside it
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    found = []
    for part in sorted(tmp_path.glob("lib.so.*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", part], check=True, capture_output=True, text=True).stdout
        found += [(name, *e) for name, ins in kernels(text) for e in early(ins)]
    assert found
    least = {}
    for _, op, slots, branch, _ in found:
        if not branch:
            least[op] = min(slots, least.get(op, LIMIT))
    assert least and all(n >= 5 for n in least.values()), least  # two passes and three slots at least
    bad = [(name, op, slots, k) for name, op, slots, branch, k in found if slots < least.get(op, LIMIT)]
    assert not bad, bad[:5]
