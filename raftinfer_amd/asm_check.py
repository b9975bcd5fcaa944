"""Build-time checks of the prefill kernels' inline-asm MFMAs.

`prefill_mfma_kernel` issues its PV MFMAs as inline asm (so that the O^T
accumulators stay in AGPRs), `prefill_wide_kernel` and `paged_stream_kernel` all of
theirs.  The compiler cannot see an MFMA inside asm, so it neither inserts the wait states
the MFMA needs around it nor avoids placing a register copy right behind it.
The build therefore scans the kernels' gfx950 assembly and fails on

* any read of an inline-asm MFMA's destination registers, or (vector registers)
  any write to them, within the MFMA's result latency: a copy of an accumulator
  placed there once computed wrong prefill outputs;
* any vector instruction that writes an operand of an inline-asm MFMA, its
  accumulator among them, within the two wait states before it;
* in kernels that address the accumulation registers by number (`owned_agprs`),
  any use of one outside asm: it would overwrite an accumulator;
* any memory instruction that reads a scalar register within the five wait states
  behind a vector instruction that writes it, and any load into LDS right behind a
  write of M0: around inline asm the compiler leaves these waits out too.
"""
from __future__ import annotations

import re

# Wait states a v_mfma_f32_32x32x16_bf16 result (16 passes) needs before a
# VALU or v_accvgpr read of it; the kernels' drains give 20 (s_nop 7, s_nop 7,
# s_nop 3).
RESULT_WAIT_STATES = 19
# Wait states between a VALU write of a register and an MFMA that reads it.
OPERAND_WAIT_STATES = 2

# Wait states between a VALU write of a scalar register and a memory instruction that
# reads it, and between a write of M0 and a load into LDS.
SCALAR_WAIT_STATES = 5
M0_WAIT_STATES = 1

_INDEX = r"(0x[0-9a-f]+|\d+)"
_REGISTER = re.compile(rf"\b([av])\[{_INDEX}:{_INDEX}\]|\b([av])\[?{_INDEX}\b")
_SCALAR = re.compile(rf"\bs\[{_INDEX}:{_INDEX}\]|\bs{_INDEX}\b|\b(vcc|m0)\b")
_LABEL = re.compile(r"^([\w.$]+):")
_NOP = re.compile(r"^s_nop\s+(\d+)")


def _registers(operand: str):
    """(file, first, last) of every vector / accumulation register named."""
    found = []
    for m in _REGISTER.finditer(operand):
        if m.group(1):
            found.append((m.group(1), int(m.group(2), 0), int(m.group(3), 0)))
        else:
            found.append((m.group(4), int(m.group(5), 0), int(m.group(5), 0)))
    return found


def _vector_writes(opcode: str, operands):
    """The registers that a vector instruction writes: its first operand, both of a swap."""
    if not opcode.startswith("v_"):
        return []
    return operands[0] + (operands[1] if "swap" in opcode else [])


def _overlap(x, y) -> bool:
    return x[0] == y[0] and x[1] <= y[2] and y[1] <= x[2]


def asm_mfma_hazards(assembly: str, owned_agprs: bool = False) -> list[str]:
    """The violations of the rules above (s_nop n counts n + 1 wait states, any
    other instruction 1), along every path: what is under way at a branch reaches
    its label too, and nothing falls through an unconditional one.  Reads by other
    MFMAs are not checked: an accumulator feeds only the next MFMA of its own chain,
    which the hardware's dependency check covers."""
    arrivals: dict[str, tuple[dict, dict]] = {}
    while True:
        hazards, found = _one_pass(assembly, owned_agprs, arrivals)
        if found == arrivals:
            return hazards
        arrivals = found


def _merge(into: dict, entries) -> None:
    for register, left, line in entries:
        into[register, line] = max(into.get((register, line), 0), left)


def _one_pass(assembly: str, owned_agprs: bool, arrivals):
    """The hazards in listing order, entering each label with what falls into it and
    with its arrivals; and the arrivals that this pass saw (a label's only grow)."""
    found = {label: (dict(p), dict(w)) for label, (p, w) in arrivals.items()}
    hazards: list[str] = []
    pending: list[list] = []  # [destination, wait states left, line] of asm MFMAs
    written: list[list] = []  # [register, wait states left, line] of VALU writes
    in_asm = False
    for number, raw in enumerate(assembly.splitlines(), 1):
        text = raw.strip()
        if text.startswith(";;#ASMSTART"):
            in_asm = True
            continue
        if text.startswith(";;#ASMEND"):
            in_asm = False
            continue
        label = _LABEL.match(text)
        if label and label.group(1) in arrivals:
            both = ({}, {})
            _merge(both[0], [(tuple(r), left, line) for r, left, line in pending])
            _merge(both[1], [(tuple(r), left, line) for r, left, line in written])
            for mine, more in zip(both, arrivals[label.group(1)]):
                _merge(mine, [(r, left, line) for (r, line), left in more.items()])
            pending, written = ([[r, left, line] for (r, line), left in mine.items()] for mine in both)
        text = text.split(";")[0].strip()
        if not text or text.startswith(".") or text.endswith(":"):
            continue
        issued = None  # the destination of an asm MFMA on this line
        opcode = text.split()[0]
        operands = [_registers(x) for x in text[len(opcode):].split(",")]
        nop = _NOP.match(text)
        if opcode.startswith("v_mfma"):
            if in_asm and operands[0]:
                for source in operands[1] + operands[2] + operands[3]:
                    for register, left, line in written:
                        if left > 0 and _overlap(register, source):
                            hazards.append(f"line {number}: '{text}' reads a register written at line {line}, "
                                           f"{OPERAND_WAIT_STATES - left} wait states before")
                issued = operands[0][0]
        elif nop is None:
            stores = opcode.startswith("ds_write") or "store" in opcode
            reads = [r for x in (operands if stores else operands[1:]) for r in x]
            writes = [r for r in _vector_writes(opcode, operands) if r[0] == "v" and r not in reads]
            for verb, registers in (("reads", reads), ("writes", writes)):
                for register in registers:
                    for dest, left, line in pending:
                        if left > 0 and _overlap(dest, register):
                            hazards.append(f"line {number}: '{text}' {verb} {dest[0]}[{dest[1]}:{dest[2]}], written by "
                                           f"the inline-asm MFMA at line {line}, after "
                                           f"{RESULT_WAIT_STATES - left} wait states")
            if owned_agprs and not in_asm and any(r[0] == "a" for x in operands for r in x):
                hazards.append(f"line {number}: '{text}' uses an accumulation register outside asm")
        step = int(nop.group(1)) + 1 if nop else 1
        for entry in pending + written:
            entry[1] -= step
        if opcode.startswith(("s_branch", "s_cbranch")):
            to = found.setdefault(text.split()[1], ({}, {}))
            _merge(to[0], [(tuple(r), left, line) for r, left, line in pending if left > 0])
            _merge(to[1], [(tuple(r), left, line) for r, left, line in written if left > 0])
        if opcode.startswith(("s_branch", "s_endpgm")):
            pending, written = [], []
        pending = [e for e in pending if e[1] > 0]
        if issued is not None:
            pending.append([issued, RESULT_WAIT_STATES, number])
        written = [e for e in written if e[1] > 0]
        if not opcode.startswith("v_mfma"):
            written += [[r, OPERAND_WAIT_STATES, number] for r in _vector_writes(opcode, operands)]
    return hazards, found


def _scalars(text: str):
    """(name, first, last) of every scalar register named; vcc and m0 by their names."""
    found = []
    for m in _SCALAR.finditer(text):
        if m.group(4):
            found.append((m.group(4), 0, 0))
        else:
            first = m.group(1) or m.group(3)
            found.append(("s", int(first, 0), int(m.group(2) or first, 0)))
    return found


def scalar_wait_hazards(assembly: str) -> list[str]:
    """The memory instructions that read a scalar register, or M0, too soon after it is
    written, along every path as above."""
    arrivals: dict[str, dict] = {}
    while True:
        hazards, found = _one_scalar_pass(assembly, arrivals)
        if found == arrivals:
            return hazards
        arrivals = found


def _one_scalar_pass(assembly: str, arrivals):
    found = {label: dict(entries) for label, entries in arrivals.items()}
    hazards: list[str] = []
    pending: dict = {}  # (register, line): wait states left
    for number, raw in enumerate(assembly.splitlines(), 1):
        text = raw.strip()
        label = _LABEL.match(text)
        if label and label.group(1) in arrivals:
            _merge(pending, [(r, left, line) for (r, line), left in arrivals[label.group(1)].items()])
        text = text.split(";")[0].strip()
        if not text or text.startswith(".") or text.endswith(":"):
            continue
        opcode, _, rest = text.partition(" ")
        operands = rest.split(",")
        if opcode.startswith(("global_", "buffer_", "flat_", "scratch_")):
            reads = _scalars(rest) + ([("m0", 0, 0)] if "lds" in opcode or rest.endswith(" lds") else [])
            hazards += [f"line {number}: {text}: reads {r[0]} {left} wait states too soon after line {line}"
                        for (r, line), left in pending.items() if any(_overlap(r, x) for x in reads)]
        nop = _NOP.match(text)
        step = int(nop.group(1)) + 1 if nop else 1
        pending = {key: left - step for key, left in pending.items() if left > step}
        if opcode.startswith("v_"):
            if rest.lstrip().startswith("v") and "s[" not in rest and "vcc" not in rest and not opcode.startswith("v_cmp"):
                continue  # (most: no scalar result)
            # a scalar result: the first operand, of carries and scaled divisors the second; vcc unnamed
            results = _scalars(operands[0]) + (_scalars(operands[1]) if re.search("_co_|div_scale|v_mad_[iu]64", opcode) else [])
            results += [("vcc", 0, 0)] if opcode.startswith("v_cmp") and opcode.endswith("_e32") else []
            pending.update({(r, number): SCALAR_WAIT_STATES for r in results})
        elif opcode.startswith("s_") and not opcode.startswith(("s_cmp", "s_bitcmp")) and rest:
            written = _scalars(operands[0])
            pending = {key: left for key, left in pending.items() if not any(key[0][0] == w[0] and w[1] <= key[0][1] and key[0][2] <= w[2] for w in written)}
            if ("m0", 0, 0) in written:
                pending[("m0", 0, 0), number] = M0_WAIT_STATES
        if opcode.startswith(("s_branch", "s_cbranch")):
            _merge(found.setdefault(rest.strip(), {}), [(r, left, line) for (r, line), left in pending.items()])
        if opcode.startswith(("s_branch", "s_endpgm", "s_setpc")):
            pending = {}
    return hazards, found
