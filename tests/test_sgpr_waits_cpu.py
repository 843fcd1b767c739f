"""Vector memory instructions that take their base from scalar registers: five
wait states lie between a vector instruction that writes such a register
(v_readlane, v_readfirstlane, a comparison, a carry) and the access, on every
path.  The compiler counts them for its own loads; inside inline assembly, where
the loads straight into LDS stand, it does not."""

import re

import pytest

import asm_hazards as H

NEED = 5
_SREG = re.compile(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\b(vcc)\b")
_CARRY = ("v_add_co", "v_addc_co", "v_sub_co", "v_subb_co", "v_div_scale", "v_mad_u64", "v_mad_i64")


def sregs(text):
    out = set()
    for m in _SREG.finditer(text):
        if m.group(1):
            out.update(range(int(m.group(1)), int(m.group(2)) + 1))
        else:
            out.add(m.group(4) or int(m.group(3)))
    return frozenset(out)


def written(op, args):
    """Scalar registers that a vector instruction writes."""
    ops = H.operands(args)
    if op.startswith(("v_readlane", "v_readfirstlane")):
        return sregs(ops[0])
    if op.startswith("v_cmp"):
        return sregs(ops[0]) or frozenset(("vcc",))
    return sregs(ops[1]) if op.startswith(_CARRY) and len(ops) > 1 else frozenset()


def fewest_waits(insts, labels):
    """The fewest wait states found, and how many accesses have a scalar base."""
    best, bases = NEED, 0
    for op, args in insts:
        bases += op.startswith(("global_", "buffer_", "flat_")) and bool(sregs(args))
    for i, (op, args) in enumerate(insts):
        stack = [(s, 0, written(op, args)) for s in H.successors(i, insts, labels)] if op.startswith("v_") else []
        seen = set()
        while stack:
            j, ws, live = stack.pop()
            if ws >= best or not live or j >= len(insts) or (j, ws, live) in seen:
                continue
            seen.add((j, ws, live))
            op2, args2 = insts[j]
            if op2.startswith(("global_", "buffer_", "flat_", "scratch_")) and sregs(args2) & live:
                best = ws
                continue
            ops = H.operands(args2)
            if ops and op2.startswith(("s_mov", "s_add", "s_sub", "s_lshl", "s_lshr", "s_and", "s_or", "s_mul",
                                       "s_load", "s_cselect", "v_readlane", "v_readfirstlane")):
                live = live - sregs(ops[0])
            cost = int(args2.split()[0], 0) + 1 if op2 == "s_nop" else 1
            stack.extend((s, ws + cost, live) for s in H.successors(j, insts, labels))
    return best, bases


def check(kernels):
    total = 0
    for name, lines in kernels.items():
        best, bases = fewest_waits(*H.parse(lines))
        total += bases
        assert best >= NEED, f"{name}: {best} wait states"
    assert total > 0


@pytest.mark.parametrize("source", ["decode.hip", "tree_verify.hip"])
def test_scalar_bases_are_waited_for(source, compiled_kernels):
    check(compiled_kernels[source])


def test_scalar_bases_of_the_chunk_kernels_are_waited_for(compiled_kernels, tmp_path):
    check(H.kernels(H.compile_device_asm(H.CSRC / "chunk.hip", tmp_path)))


def test_the_scan_finds_a_missing_wait():
    def at(text):
        return fewest_waits(*H.parse(text.split("\n")))

    near = "k:\n\tv_readlane_b32 s5, v1, 0\n\ts_mov_b32 m0, s9\n\ts_nop 0\n\tglobal_load_lds_dwordx4 v2, s[4:5]\n\ts_endpgm"
    assert at(near) == (2, 1)
    assert at(near.replace("s_nop 0", "s_nop 3")) == (NEED, 1)
    assert at(near.replace("\ts_nop 0", "\ts_mov_b32 s5, 0\n\ts_nop 0")) == (NEED, 1)  # written again
    loop = ("k:\n.LBB0_1:\n\tglobal_load_dword v3, v2, s[6:7]\n\ts_add_u32 s8, s8, 1\n\tv_cmp_eq_u32_e64 s[6:7], v1, v2\n"
            "\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm")
    assert at(loop) == (1, 1)
