"""Build check for the kernels that issue vector-memory instructions from inline asm (LDS-DMA in csrc/attn_impl.h,
csrc/lds_dma.h, csrc/attn_decode_mx.hip): such an instruction may read a scalar register that the vector ALU wrote
(v_readfirstlane, or v_readlane of a spilled scalar) only five wait states after that write. The compiler keeps the
distance for instructions that it knows; inside an asm statement nothing does, and the registers are its choice. Walks
the compiler's assembly backwards from every vector-memory instruction of an asm statement, over branches too.

    python tools/audit_asm_waits.py file.s ...
"""
import re
import sys

STATES = 5
CARRY = re.compile(r"_co_|div_scale|mad_[ui]64")      # a second result, in a scalar register


def registers(operand):
    """Numbers of the scalar registers of an operand."""
    m = re.match(r"s\[(\d+):(\d+)\]|s(\d+)\b", operand.strip())
    if not m:
        return set()
    return {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def functions(lines):
    """Per function a list of ("label", name) and ("op", mnemonic, operands, in an asm statement, line number)."""
    code, in_asm = None, False
    for n, line in enumerate(lines, 1):
        text = line.strip()
        m = re.match(r"([\w.$]+):", line)
        if m:
            if not m[1].startswith("."):
                if code:
                    yield code
                code = []
            elif code is not None:
                code.append(("label", m[1]))
        elif "#ASMSTART" in text:
            in_asm = True
        elif "#ASMEND" in text:
            in_asm = False
        else:
            text = text.split(";")[0].strip()
            if text and not text.startswith(".") and code is not None:
                op, _, rest = text.partition(" ")
                op, rest = (op, rest) if "\t" not in op else op.split("\t", 1)
                code.append(("op", op, [x.strip() for x in rest.split(",")] if rest else [], in_asm, n))
    if code:
        yield code


def violations(lines):
    """(line number, wait states) of every vector-memory instruction of an asm statement that comes too early."""
    found = []
    for code in functions(lines):
        label = {c[1]: i for i, c in enumerate(code) if c[0] == "label"}
        jumps = {}
        for i, c in enumerate(code):
            if c[0] == "op" and c[1].startswith(("s_branch", "s_cbranch")) and c[2] and c[2][-1] in label:
                jumps.setdefault(label[c[2][-1]], []).append(i)
        for i, c in enumerate(code):
            if c[0] != "op" or not c[3] or not c[1].startswith(("buffer_", "global_", "flat_", "scratch_")):
                continue
            needs = set().union(*map(registers, c[2]))
            walk, seen = [(i, 0)], {}
            while walk:
                j, states = walk.pop()
                if seen.get(j, STATES) <= states:
                    continue
                seen[j] = states
                before = list(jumps.get(j, []))
                if j > 0 and not (code[j - 1][0] == "op" and code[j - 1][1] in ("s_branch", "s_endpgm", "s_setpc_b64")):
                    before.append(j - 1)
                for k in before:
                    p = code[k]
                    if p[0] == "label":
                        walk.append((k, states))
                    elif p[1].startswith("v_") and set().union(*map(registers, p[2][:2 if CARRY.search(p[1]) else 1])) & needs:
                        found.append((c[4], states))
                    else:
                        walk.append((k, states + (int(p[2][0], 0) + 1 if p[1] == "s_nop" else 1)))
    return found


def main(paths):
    bad = 0
    for path in paths:
        with open(path) as f:
            got = violations(f)
        for n, states in got[:20]:
            print(f"audit_asm_waits: {path}:{n}: a scalar register written by the vector ALU {states} wait states before")
        print(f"audit_asm_waits: {path}: {len(got)} violations")
        bad += len(got)
    return 1 if bad else 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
