"""Static check of gfx950 assembly for matrix instructions written in inline asm, whose wait states the compiler
does not insert: no vector instruction writes an operand within the two wait states before one, and nothing but
another matrix instruction touches its result within 18 of it (16 passes of a 32x32 product, and two).

Instructions are walked in file order; each counts one wait state, ``s_nop N`` N + 1 and a matrix instruction 8 (the
least that one takes to issue behind another)."""
import re

_TOKEN = re.compile(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b")


def _regs(text: str) -> set:
    out = set()
    for k, lo, hi, k1, n in _TOKEN.findall(text):
        out |= {(k, r) for r in range(int(lo), int(hi) + 1)} if k else {(k1, int(n))}
    return out


def mfma_hazards(instrs: list) -> list:
    """``instrs``: (instruction, from inline asm) pairs of one kernel; the compiler's own matrix instructions are its care."""
    issues, written, live = [], [], []  # live: [registers, wait states since, text]
    for s, ours in instrs:
        op, _, rest = s.partition(" ")
        args = rest.split(",")
        mfma = op.startswith("v_mfma")
        if mfma and ours:
            sources, states = _regs(",".join(args[1:])), 0
            for count, regs, text in reversed(written):
                if states >= 2:
                    break
                if regs & sources:
                    issues.append(f"{s}  reads what [{text}] has just written")
                states += count
        elif not op.startswith("s_"):
            for regs, since, text in live:
                if regs & _regs(rest):
                    issues.append(f"{s}  touches the result of [{text}] after {since}")
        count = int(args[0]) + 1 if op == "s_nop" else 8 if mfma else 1
        live = [[r, n + count, t] for r, n, t in live if n + count < 18]
        if mfma and ours:
            live.append([_regs(args[0]), 0, s])
        plain = op.startswith("v_") and not mfma and not op.startswith("v_cmp")
        written = (written + [(count, _regs(args[0]) if plain else set(), s)])[-4:]
    return issues
