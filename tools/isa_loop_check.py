#!/usr/bin/env python3
"""Check of the generated ISA of the software-pipelined catalog kernel (catalog_bf16.hip).

Its MFMAs are inline asm, so hipcc's hazard recogniser does not protect register copies it might place next to them.
The steady-state loop is correct only while hipcc places NO such copy inside it; this script disassembles the kernel,
finds the steady-state loop (the longest backward `s_branch` loop) and fails if it contains v_accvgpr_* / v_mov_* /
scratch_* instructions.  Run by tests/test_host_logic.py (no GPU needed: hipcc cross-compiles)."""
import collections
import os
import re
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
from pivotcvae_amd import build  # noqa: E402
FORBIDDEN = ("v_accvgpr_", "v_mov_b", "scratch_", "buffer_store", "v_readlane", "v_writelane")


def _regs(tok):
    """'v[10:13]' / 'v7' -> ('v', {10, 11, 12, 13})"""
    tok = tok.strip()
    m = re.match(r"([va])\[(\d+):(\d+)\]", tok)
    if m:
        return m.group(1), set(range(int(m.group(2)), int(m.group(3)) + 1))
    m = re.match(r"([va])(\d+)$", tok)
    if m:
        return m.group(1), {int(m.group(2))}
    return None, set()


def forbidden_in(loop, no_mov=False):
    """register copies / spills hipcc placed in an unfenced loop that could read an MFMA result too early: any v_accvgpr_*,
    any scratch access, and a v_mov whose SOURCE is a register some MFMA of the loop writes.  (A v_mov from an SGPR, a literal
    or a VALU-produced register - the rare candidate path of the screening kernels builds its list entries that way - moves
    no MFMA result.)  no_mov=True (the cross-entropy kernels): no v_mov at all - their row-sum MFMAs read the packed numerators
    without wait states, so hipcc must not assemble that operand with copies either."""
    mfma_dst = {"v": set(), "a": set()}
    for l in loop:
        if l.startswith("v_mfma"):
            k, r = _regs(l.split(None, 1)[1].split(",")[0])
            if k:
                mfma_dst[k] |= r
    bad = []
    n = len(loop)
    for i, l in enumerate(loop):
        if l.startswith("v_accvgpr_read_b32"):
            # a READ of an accumulator that no MFMA of the loop wrote in the last 16 instructions (the back edge included) moves a
            # finished result, wherever hipcc puts it: the bf16x6 kernel hands its chunk of row sums to the running total that
            # way once per trip (catalog_x3.h, X6_CHUNK_LSUM).  Anything closer to its writer stays forbidden.
            k, src = _regs(l.split(",")[-1])
            recent = [loop[(i - d) % n] for d in range(1, 17)]
            close = any(x.startswith("v_mfma") and (_regs(x.split(None, 1)[1].split(",")[0])[1] & src) for x in recent)
            if k != "a" or close:
                bad.append(l)
            continue
        if l.startswith(("v_accvgpr_", "scratch_", "buffer_store", "v_readlane", "v_writelane")):
            bad.append(l)
        elif l.startswith("v_mov_b"):
            k, r = _regs(l.split(",")[-1])
            if no_mov or (k and (r & mfma_dst[k])):
                bad.append(l)
    return bad


def queued_operand_clobbers(loop, depth=4):
    """LDS reads / VALU ops whose DESTINATION is a VGPR that one of the last `depth` MFMAs in front of them reads as A or B operand.

    The SIMD issues an MFMA every 8 cycles, the matrix pipe starts one every 16: in MFMA-dense stretches MFMAs queue up and read
    their operands when they START.  hipcc (which sees those operands dead behind their last MFMA) may hand the register to the
    next asm result; data of a ds_read issued two MFMAs behind such a read has been seen to land before the queued MFMA consumed
    the old value (catalog_x3.h, x3_keep).  The loop is walked twice so that the back edge is covered."""
    seq = loop + loop
    n = len(loop)
    recent = []   # operand register sets of the last MFMAs
    bad = []
    for i, l in enumerate(seq):
        op = l.split()[0]
        args = [a.strip().split(" ")[0] for a in l[len(op):].split(",")] if " " in l else []
        if op.startswith("v_mfma"):
            srcs = set()
            for a in args[1:3]:
                k, r = _regs(a)
                if k == "v":
                    srcs |= r
            recent.append(srcs)
            recent = recent[-depth:]
            continue
        if i < n:
            continue   # report on the second pass only (the first one warms `recent` up across the back edge)
        if op.startswith("ds_read") or (op.startswith("v_") and not op.startswith("v_cmp")):
            k, dst = _regs(args[0]) if args else (None, set())
            if k == "v" and any(dst & r for r in recent):
                bad.append(l)
    return bad


_ASM_CACHE = {}


def _asm_of(src, extra=()):
    """gfx950 ISA of one translation unit with the library's flags (hipcc -S), compiled once per process"""
    key = (src, tuple(extra))
    if key not in _ASM_CACHE:
        _ASM_CACHE[key] = subprocess.run(["/opt/rocm/bin/hipcc", *build.FLAGS, "-S", "--cuda-device-only", "-x", "hip", *extra, src, "-o", "-"],
                                         capture_output=True, text=True, check=True).stdout
    return _ASM_CACHE[key]


def forbidden(line):   # kept for callers that test single lines: the conservative form
    return line.startswith(FORBIDDEN)


def hot_loops(pattern="pipe"):
    """-> {kernel name: [loop bodies]} for every loop with >= 60 MFMAs of which at least one is NOT fenced (followed by
    `s_nop 15`): those are the loops whose correctness depends on hipcc placing no register copy / spill inside."""
    src = os.path.join(ROOT, "pivotcvae_amd", "csrc", "catalog_bf16.hip")
    extra = os.environ.get("PCVAE_ISA_FLAGS", "").split()   # e.g. -DPIPE_OPS_MODE=0 when judging a variant
    asm = _asm_of(src, extra)
    out = {}
    for m in re.finditer(r"^(_Z\S+):\s*; @", asm, re.M):
        name = subprocess.run(["c++filt", m.group(1)], capture_output=True, text=True).stdout.strip()
        if pattern not in name or "kernel" not in name:
            continue
        body = asm[m.end():asm.find(".Lfunc_end", m.end())].split("\n")
        lines = [l.split(";")[0].strip() for l in body]
        lines = [l for l in lines if l]
        labels = {mm.group(1): n for n, l in enumerate(lines) if (mm := re.match(r"(\.LBB\d+_\d+):", l))}
        loops = []
        for n, l in enumerate(lines):
            mm = re.match(r"s_c?branch\w*\s+(\.LBB\d+_\d+)", l)
            if mm and labels.get(mm.group(1), 1 << 30) < n:
                lo = labels[mm.group(1)]
                loop = [x for x in lines[lo:n + 1] if not x.startswith(".")]
                mf = [i for i, x in enumerate(loop) if x.startswith("v_mfma")]
                unfenced = [i for i in mf if not (i + 1 < len(loop) and loop[i + 1].startswith("s_nop 15"))]
                # an unfenced MFMA writing AGPRs / fed by asm is what needs protection; builtin MFMAs in fenced loops are followed
                # by hipcc's own nops, so require a majority of unfenced MFMAs to call the loop a steady-state one
                if len(mf) >= 60 and len(unfenced) * 2 > len(mf):
                    loops.append(loop)
        # nested detection returns enclosing loops too: keep the innermost ones (no other candidate strictly inside)
        keep = [lp for lp in loops if not any(o is not lp and len(o) < len(lp) and all(x in lp for x in o[:5]) and " ".join(o) in " ".join(lp) for o in loops)]
        out[re.sub(r"\(anonymous namespace\)::", "", name)] = keep
    return out


def arrival_counter_waits(sources=("gemm_f32.hip", "elementwise.hip")):
    """-> list of (file, kernel, line) where an arrival counter is bumped (integer global_atomic_add) behind device-scope (sc1)
    stores of partial results WITHOUT an `s_waitcnt vmcnt(0)` in between.  A workgroup-scope release emits no vmcnt wait on
    gfx950, so the hand-off of the weight gradients' batch splits (gemm_f32.hip) and of the KL partials (elementwise.hip)
    carries an explicit one; this check keeps hipcc (and future edits) from losing it.  Also returns the number of hand-offs seen."""
    bad, seen = [], 0
    for f in sources:
        src = os.path.join(ROOT, "pivotcvae_amd", "csrc", f)
        asm = _asm_of(src)
        for m in re.finditer(r"^(_Z\S+):\s*; @", asm, re.M):
            body = asm[m.end():asm.find(".Lfunc_end", m.end())].split("\n")
            lines = [l.split(";")[0].strip() for l in body]
            last_sc1, waited = None, True
            for n, l in enumerate(lines):
                if l.startswith("global_store") and " sc1" in l and "sc0" not in l:
                    last_sc1, waited = n, False
                elif l.startswith("s_waitcnt") and "vmcnt(0)" in l:
                    waited = True
                elif re.match(r"global_atomic_add(_u32)?\s", l) and last_sc1 is not None:
                    seen += 1
                    if not waited:
                        bad.append((f, m.group(1), l))
                    last_sc1 = None
    return bad, seen


def mfma_fresh_operand_reads(pattern=("x3_pipe", "bf16_pipe", "screen_pipe"), wait_states=2):
    """-> [(kernel, index, writer, mfma)]: MFMAs that read (A, B or C operand) a VGPR which a VALU instruction wrote fewer than
    `wait_states` wait states earlier, anywhere in a kernel (straight-line order: fall-through paths, which is how a loop's
    preheader reaches its header).  hipcc's hazard recogniser inserts these wait states for MFMAs it knows; an inline-asm MFMA is
    opaque to it.  Round 3: the preheader copies of a steady-state loop's carried values (v_mov) ended right in front of the
    loop's first asm MFMA - with one instruction between them the MFMA read a stale A fragment (column tile 0 of every wave
    wrong); the loops now begin with a fence, and this check keeps every asm MFMA of the pipelined kernels two wait states
    away from any VALU write of its operands."""
    asm = _asm_of(os.path.join(ROOT, "pivotcvae_amd", "csrc", "catalog_bf16.hip"))
    bad, seen = [], 0
    for m in re.finditer(r"^(_Z\S+):\s*; @", asm, re.M):
        if not any(p in m.group(1) for p in pattern):
            continue
        body = asm[m.end():asm.find(".Lfunc_end", m.end())].split("\n")
        lines = [l.split(";")[0].strip() for l in body]
        lines = [l for l in lines if l and not l.startswith(".") or re.match(r"\.LBB", l)]
        for i, l in enumerate(lines):
            if not l.startswith("v_mfma"):
                continue
            seen += 1
            args = [a.strip().split(" ")[0] for a in l[len(l.split()[0]):].split(",")]
            srcs = set()
            for a in args[1:4]:
                k, r = _regs(a)
                if k == "v":
                    srcs |= r
            ws, j = 0, i - 1
            while j >= 0 and ws < wait_states:
                p = lines[j]
                if p.endswith(":"):          # a label: not an instruction
                    j -= 1
                    continue
                op = p.split()[0]
                if op == "s_nop":
                    ws += int(p.split()[1]) + 1
                else:
                    if op.startswith("v_") and not op.startswith(("v_mfma", "v_cmp")):
                        k, dst = _regs(p[len(op):].split(",")[0].strip())
                        if k == "v" and (dst & srcs):
                            bad.append((m.group(1)[:60], i, p, l))
                    ws += 1
                j -= 1
    return bad, seen


def mfma_result_early_reads(pattern=("x3_pipe", "bf16_pipe", "screen_pipe"), wait_states=5):
    """-> [(kernel, index, mfma, reader)]: a VALU / LDS-write / store instruction that reads a VGPR (or AGPR) which an MFMA wrote
    fewer than `wait_states` wait states earlier (straight-line order; an instruction counts 1, `s_nop n` n + 1, an MFMA 4 - its
    issue alone holds the port that long).  The matrix pipe delivers a 16x16x32 result a few passes after issue; hipcc pads
    such reads for MFMAs it knows, not for inline asm - the pipelined kernels keep them apart by schedule (the numerators are
    taken >= 2 CT MFMAs behind the logits' last MFMA), and this check holds every one of them to it."""
    asm = _asm_of(os.path.join(ROOT, "pivotcvae_amd", "csrc", "catalog_bf16.hip"))
    bad, seen = [], 0
    for m in re.finditer(r"^(_Z\S+):\s*; @", asm, re.M):
        if not any(p in m.group(1) for p in pattern):
            continue
        body = asm[m.end():asm.find(".Lfunc_end", m.end())].split("\n")
        lines = [l.split(";")[0].strip() for l in body]
        lines = [l for l in lines if l and not l.startswith(".")]
        recent = []   # (wait states since, dst regs, text) of the last MFMAs
        for i, l in enumerate(lines):
            op = l.split()[0]
            args = [a.strip().split(" ")[0] for a in l[len(op):].split(",")] if " " in l else []
            if op.startswith(("v_", "ds_write", "global_store", "buffer_store", "scratch_store")) and not op.startswith("v_mfma"):
                srcs = set()
                for a in (args[1:] if op.startswith("v_") else args):
                    k, r = _regs(a)
                    if k:
                        srcs |= {(k, x) for x in r}
                for ws, dst, text in recent:
                    if ws < wait_states and (srcs & dst):
                        bad.append((m.group(1)[:60], i, text, l))
            step = (int(l.split()[1]) + 1) if op == "s_nop" else (4 if op.startswith("v_mfma") else 1)
            recent = [(ws + step, d, t) for ws, d, t in recent if ws + step < wait_states]
            if op.startswith("v_mfma"):
                seen += 1
                k, r = _regs(args[0])
                recent.append((0, {(k, x) for x in r}, l))
    return bad, seen


def main():
    ok = True
    for name, loops in hot_loops().items():
        ok = ok and bool(loops)
        for loop in loops:
            c = collections.Counter(l.split()[0] for l in loop)
            bad = forbidden_in(loop, no_mov="catalog_ce_" in name)
            clob = queued_operand_clobbers(loop)
            print(f"{name[:70]}: unfenced loop of {len(loop)} instructions, {c['v_mfma_f32_16x16x32_bf16']} MFMA, {len(bad)} forbidden, "
                  f"{len(clob)} writes into operands of the last 4 MFMAs")
            for b in (bad + (clob if "x3" in name else []))[:10]:
                print("   ", b)
            # enforced for the bf16x3 kernel, whose schedule has MFMA-dense stretches where the hazard was observed; the round-1
            # kernels (parity-tested on hardware at every size) are reported only
            ok = ok and not bad and not (clob and "x3" in name)
    fresh, nm = mfma_fresh_operand_reads()
    print(f"asm MFMAs of the pipelined kernels: {nm}, {len(fresh)} reading a VGPR a VALU op wrote < 2 wait states earlier")
    for b in fresh[:10]:
        print("   ", b)
    ok = ok and nm > 0 and not fresh
    early, nm2 = mfma_result_early_reads()
    print(f"MFMA results read by VALU / stores fewer than 5 wait states behind the MFMA: {len(early)} (of {nm2} MFMAs)")
    for b in early[:10]:
        print("   ", b)
    ok = ok and not early
    bad, seen = arrival_counter_waits()
    print(f"arrival counters behind sc1 stores: {seen} hand-offs, {len(bad)} without s_waitcnt vmcnt(0)")
    for b in bad[:10]:
        print("   ", b)
    ok = ok and seen > 0 and not bad
    return 0 if ok else 1


if __name__ == "__main__":
    sys.exit(main())
