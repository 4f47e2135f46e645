"""Waits around the instructions that the GEMMs write in assembly.  The hardware does not hold back an
MFMA whose operand a vector instruction wrote less than two wait states earlier, nor a load whose scalar
base one wrote less than five earlier.  For its own instructions the compiler inserts the idle slots; it
does not look into assembly.  Read from the compiled kernels (no GPU needed): every path of up to that
many wait states that leads to such an instruction is followed backwards."""
import os
import re

import pytest

from tests.test_kernel_isa import ROOT, _compile

CSRC = os.path.join(ROOT, "symm-mem-recipes_amd", "csrc")


def _registers(operand):
    m = re.fullmatch(r"([vas])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m.group(1), i) for i in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.fullmatch(r"([vas])(\d+)", operand)
    return {(m.group(1), int(m.group(2)))} if m else set()


class Instruction:
    def __init__(self, text, in_assembly):
        self.text, self.in_assembly = text, in_assembly
        self.op, _, rest = text.partition(" ")
        operands = [t for t in re.split(r"[,\s]+", rest) if t]
        self.registers = [_registers(t) for t in operands]
        self.states = int(operands[0]) + 1 if self.op == "s_nop" else 1
        self.target = operands[0] if re.match(r"s_(c?branch)", self.op) else None
        self.vector = self.op.startswith("v_") and not self.op.startswith("v_mfma")

    def writes(self):
        """What a vector instruction writes: its first operand, and the scalar carry behind it."""
        if not self.registers:
            return set()
        return self.registers[0] | (self.registers[1] if re.search(r"_co_|div_scale", self.op) else set())


def kernels(asm):
    """{name: ([instructions], {label: index})} in program order."""
    out = {}
    for m in re.finditer(r"^(_ZN3smr\w+):[^\n]*\n(.*?)^\.Lfunc_end", asm, re.S | re.M):
        code, labels, inside = [], {}, False
        for line in m.group(2).splitlines():
            inside = True if "#ASMSTART" in line else False if "#ASMEND" in line else inside
            text = line.split(";")[0].strip()
            label = re.match(r"(\.LBB\w+):", text)
            if label:
                labels[label.group(1)] = len(code)
            elif re.match(r"[a-z]\w+", text):
                code.append(Instruction(text, inside))
        out[m.group(1)] = (code, labels)
    return out


def too_close(code, labels, at, needed, states):
    """A vector instruction that writes one of the registers `needed` less than `states` wait states before
    instruction `at`, on any path, or None."""
    sources = {}
    for i, ins in enumerate(code):
        if ins.target in labels:
            sources.setdefault(labels[ins.target], []).append(i)
    todo, seen = [(at, 0)], set()
    while todo:
        i, passed = todo.pop()
        if (i, passed) in seen or passed >= states:
            continue
        seen.add((i, passed))
        before = list(sources.get(i, []))
        if i > 0 and code[i - 1].op not in ("s_branch", "s_endpgm"):
            before.append(i - 1)
        for j in before:
            if code[j].vector and code[j].writes() & needed:
                return code[j].text
            todo.append((j, passed + code[j].states))
    return None


@pytest.fixture(scope="module", params=["mxfp4_matmul.hip", "ag_matmul.hip"])
def compiled(request, tmp_path_factory):
    return kernels(_compile(os.path.join(CSRC, request.param), tmp_path_factory.mktemp("isa") / "kernels.s"))


def test_no_operand_of_an_assembly_mfma_is_written_right_before_it(compiled):
    seen, bad = 0, []
    for name, (code, labels) in compiled.items():
        for i, ins in enumerate(code):
            if ins.in_assembly and ins.op.startswith("v_mfma"):
                seen += 1
                writer = too_close(code, labels, i, set().union(*ins.registers), 2)
                if writer is not None:
                    bad.append((name, writer, ins.text))
    assert seen > 100
    assert not bad, (len(bad), bad[:3])


def test_no_base_of_an_assembly_load_is_written_by_a_vector_instruction_right_before_it(compiled):
    seen, bad = 0, []
    for name, (code, labels) in compiled.items():
        for i, ins in enumerate(code):
            if ins.in_assembly and ins.op.startswith(("global_load", "buffer_load")):
                seen += 1
                base = {r for operand in ins.registers for r in operand if r[0] == "s"}
                writer = too_close(code, labels, i, base, 5)
                if writer is not None:
                    bad.append((name, writer, ins.text))
    assert seen > 20
    assert not bad, (len(bad), bad[:3])


def test_no_result_of_an_assembly_mfma_is_touched_right_behind_it(compiled):
    """A vector instruction that reads or writes an MFMA's result has to be up to 19 wait states behind it (16
    passes); the kernels leave 32 in front of their epilogue, and nothing of the compiler's may come sooner."""
    seen, bad = 0, []
    for name, (code, labels) in compiled.items():
        for i, ins in enumerate(code):
            if not (ins.in_assembly and ins.op.startswith("v_mfma")):
                continue
            seen += 1
            result, todo, visited = ins.registers[0], [(i + 1, 0)], set()
            while todo:
                j, passed = todo.pop()
                if j >= len(code) or passed >= 19 or (j, passed) in visited:
                    continue
                visited.add((j, passed))
                if code[j].vector and set().union(*code[j].registers) & result:
                    bad.append((name, ins.text, code[j].text))
                    break
                if code[j].op == "s_endpgm":
                    continue
                if code[j].target in labels:
                    todo.append((labels[code[j].target], passed + code[j].states))
                if code[j].op != "s_branch":
                    todo.append((j + 1, passed + code[j].states))
    assert seen > 100
    assert not bad, (len(bad), bad[:3])
