"""The loss head's wide tiles write their MFMAs out with the sums' registers as
their own source, so the waits that the compiler puts around an MFMA of its own
are the source's to keep (GcCore::kTied in bf16_gemm_core.hpp).  This reads the
listing of the kernels as built and holds every such MFMA to them, along every
path into and out of it:

  - its sum is its own source, in place;
  - no VALU instruction writes one of its operands within 2 wait states before;
  - nothing but another MFMA touches its sum within 18 wait states after.
"""

import os
import re
import shutil
import subprocess

import pytest

from aethelstream_amd import build

BEFORE, AFTER = 2, 18


def _regs(text):
    out = set()
    for kind, one, first, last in re.findall(r"\b([va])(?:(\d+)|\[(\d+):(\d+)\])", text):
        lo, hi = (int(one), int(one)) if one else (int(first), int(last))
        out.update((kind, r) for r in range(lo, hi + 1))
    return out


class Kernel:
    """One kernel's instructions: (opcode, operands, inline?), and its control flow."""

    def __init__(self, lines):
        self.ins, at, inline, targets = [], {}, False, {}
        for line in lines:
            t = line.strip()
            if t.startswith(";;#ASMSTART"):
                inline = True
            elif t.startswith(";;#ASMEND"):
                inline = False
            t = t.split(";")[0].strip()
            if re.match(r"^\.LBB\w+:$", t):
                at[t[:-1]] = len(self.ins)
            elif t and not t.startswith(".") and not t.endswith(":"):
                op, _, rest = t.partition(" ")
                self.ins.append((op, [a.strip() for a in rest.split(",")], inline))
        n = len(self.ins)
        self.succ = [[i + 1] if i + 1 < n else [] for i in range(n)]
        for i, (op, args, _) in enumerate(self.ins):
            if op in ("s_endpgm", "s_branch"):
                self.succ[i] = []
            if op == "s_branch" or op.startswith("s_cbranch"):
                self.succ[i].append(at[args[0]])
        self.pred = [[] for _ in range(n)]
        for i, nexts in enumerate(self.succ):
            for j in nexts:
                self.pred[j].append(i)

    def near(self, i, edges, states):
        """Instructions fewer than `states` wait states away along `edges`."""
        seen, todo = {}, [(j, 0) for j in edges[i]]
        while todo:
            j, d = todo.pop()
            if d >= states or seen.get(j, states) <= d:
                continue
            seen[j] = d
            op, args, _ = self.ins[j]
            d += 1 + (int(args[0], 0) if op == "s_nop" else 0)
            todo.extend((k, d) for k in edges[j])
        return seen

    def faults(self):
        tied, found = 0, []
        for i, (op, args, inline) in enumerate(self.ins):
            if not (inline and op.startswith("v_mfma")):
                continue
            tied += 1
            total = _regs(args[0])
            if _regs(args[3]) != total:
                found.append(f"{i}: {op} {args}: not in place")
            used = _regs(" ".join(args))
            for j in self.near(i, self.pred, BEFORE):
                o, a, _ = self.ins[j]
                # A swap writes both of its operands, anything else the first.
                written = _regs(" ".join(a[:2] if "swap" in o else a[:1]))
                if o.startswith("v_") and not o.startswith("v_mfma") and written & used:
                    found.append(f"{i}: {op} {args}: {o} {a} just before")
            for j in self.near(i, self.succ, AFTER):
                o, a, _ = self.ins[j]
                if not o.startswith("v_mfma") and _regs(" ".join(a)) & total:
                    found.append(f"{i}: {op} {args}: {o} {a} too early")
        return tied, found


def _kernels(listing):
    out, name = {}, None
    for line in listing.splitlines():
        m = re.match(r"^(_ZN4nf4s\w+):", line)
        if m:
            name = m.group(1)
            out[name] = []
        elif line.startswith(".Lfunc_end"):
            name = None
        elif name:
            out[name].append(line)
    return {n: Kernel(ls) for n, ls in out.items()}


@pytest.mark.skipif(not (os.path.exists(build.HIPCC) or shutil.which(build.HIPCC)),
                    reason="needs hipcc")
def test_tied_mfmas_keep_their_waits(tmp_path):
    src = os.path.join(build.CSRC, "linear_ce.hip")
    out = str(tmp_path / "linear_ce.s")
    subprocess.run([build.HIPCC, *build.HIP_FLAGS, "-S", "--offload-device-only", src, "-o", out],
                   check=True, capture_output=True)
    with open(out) as f:
        kernels = _kernels(f.read())
    tied = {}
    for name, k in kernels.items():
        n, found = k.faults()
        if n:
            tied[name] = n
        assert not found, (name, found[:5])
    # Logits and products of 128 x 256 and 256 x 256 tiles.
    assert len(tied) == 11, sorted(tied)


@pytest.mark.parametrize("before,after,ok", [
    ("s_nop 1", "s_nop 15\n s_nop 3\n v_accvgpr_read_b32 v9, a0", True),
    ("s_nop 0", "s_nop 15\n s_nop 3\n v_accvgpr_read_b32 v9, a0", False),
    ("s_nop 1", "s_nop 15\n v_accvgpr_read_b32 v9, a3", False),
    ("s_nop 1", "v_accvgpr_read_b32 v9, a4", True),
    ("s_cbranch_scc0 .LBB0_1\n s_nop 1", "s_nop 0", False),
])
def test_the_reading_itself(before, after, ok):
    text = (f" v_mov_b32_e32 v3, 0\n {before}\n.LBB0_1:\n ;;#ASMSTART\n"
            f" v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]\n ;;#ASMEND\n"
            f" {after}\n s_endpgm")
    tied, found = Kernel(text.splitlines()).faults()
    assert tied == 1 and (not found) == ok, found
