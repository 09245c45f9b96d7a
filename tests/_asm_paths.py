"""The checks of ``_mfma_hazards`` and ``_asm_waits`` along every path of a kernel: over loops' ends and branches too.

From each instruction that leaves something pending (a matrix instruction of inline asm its result, a vector instruction an
operand, an LDS read of inline asm its registers) the paths that follow are walked until it is there."""
import re

from _mfma_hazards import _regs

_LABEL = re.compile(r"^([.\w$]+):")
RESULT, OPERAND = 18, 2  # wait states


def kernels(asm: str) -> dict:
    """Kernel symbol -> (instructions [(text, from inline asm)], label -> index of the instruction behind it)."""
    out, cur, ours = {}, None, False
    for line in asm.splitlines():
        if re.match(r"^_Z\w+:", line):
            cur = line.split(":")[0]
            out[cur] = ([], {})
            continue
        if cur is None:
            continue
        if line.startswith(".Lfunc_end"):
            cur = None
            continue
        if ";;#ASMSTART" in line or ";;#ASMEND" in line:
            ours = ";;#ASMSTART" in line
            continue
        s = line.split(";")[0].strip()
        label = _LABEL.match(s)
        if label:
            out[cur][1][label.group(1)] = len(out[cur][0])
        elif s and not s.startswith("."):
            out[cur][0].append((s, ours))
    return out


class _Instr:
    def __init__(self, s, ours, n, labels):
        self.text, self.ours = s, ours
        self.op, _, rest = s.partition(" ")
        args = rest.split(",")
        self.scalar = self.op.startswith("s_")
        self.mfma = self.op.startswith("v_mfma")
        self.regs = _regs(rest)
        self.dst = _regs(args[0])
        self.sources = _regs(",".join(args[1:]))
        self.states = int(args[0]) + 1 if self.op == "s_nop" else 8 if self.mfma else 1
        self.writes = self.dst if self.op.startswith("v_") and not self.mfma and not self.op.startswith("v_cmp") else set()
        self.lds_read = ours and self.op.startswith("ds_read")
        self.counts = self.op.startswith(("ds_", "s_load", "s_buffer_load"))
        m = re.search(r"lgkmcnt\((\d+)\)", s) if self.op == "s_waitcnt" else None
        self.left = int(m.group(1)) if m else None
        ends = self.op in ("s_endpgm", "s_branch", "s_setpc_b64", "s_trap")
        self.next = [] if ends else [n + 1]
        if self.op == "s_branch" or self.op.startswith("s_cbranch"):
            self.next.append(labels[rest.strip()])


def _walk(instrs, start, pending, step, issues):
    """Follows every path behind ``start``.  step(instruction, pending) -> pending there after, None: no more."""
    todo, seen = [(n, pending) for n in instrs[start].next], set()
    while todo:
        at = todo.pop()
        if at in seen or at[0] >= len(instrs):
            continue
        seen.add(at)
        i = instrs[at[0]]
        after = step(i, at[1])
        if isinstance(after, str):
            issues.append(f"{i.text}  {after} [{instrs[start].text}]")
        elif after is not None:
            todo += [(n, after) for n in i.next]


def path_hazards(kernel) -> list:
    """``kernel``: a value of ``kernels()``."""
    texts, labels = kernel
    instrs = [_Instr(s, ours, n, labels) for n, (s, ours) in enumerate(texts)]
    issues = []
    for n, i in enumerate(instrs):
        if i.mfma and i.ours:
            def result(j, states, i=i):
                if not j.mfma and not j.scalar and j.regs & i.dst:
                    return f"after {states} states touches the result of"
                return states + j.states if states + j.states < RESULT else None
            _walk(instrs, n, 0, result, issues)
        elif i.writes:
            def operand(j, states, i=i):
                if j.mfma and j.ours and j.sources & i.writes:
                    return "reads what has just been written by"
                return states + j.states if states + j.states < OPERAND else None
            _walk(instrs, n, 0, operand, issues)
        elif i.lds_read:
            def landed(j, behind, i=i):
                if j.left is not None and j.left <= behind:
                    return None
                if not j.scalar and j.regs & i.dst:
                    return "touches registers of the read in flight"
                return min(behind + j.counts, 16)  # (the counter holds 15)
            _walk(instrs, n, 0, landed, issues)
    return issues
