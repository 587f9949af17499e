"""The device code in the library, read instruction by instruction: results of matrix instructions are there before anything else takes them.

A matrix instruction hands its result over some cycles after it was issued; the hardware does not hold back an ordinary instruction that
reads or overwrites it earlier, so other instructions have to stand between them.  The compiler counts them along the order in which the
code stands, and was seen to miss ways through a branch."""
import os
import re
import shutil
import struct
import subprocess

import pytest

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cubert_amd", "libcuBERT.so")
OBJDUMP = next((p for p in ("/opt/rocm/llvm/bin/llvm-objdump", shutil.which("llvm-objdump")) if p and os.path.exists(p)), None)

# States (an instruction is one, s_nop n is n + 1) between a matrix instruction and an ordinary one that takes its result, on gfx950:
# passes of four cycles and 2 for fp32's own (8 and 16), 4 for the others (4 and 8)
STATES = {"v_mfma_f32_32x32x16_f16": 12, "v_mfma_f32_32x32x16_bf16": 12, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x32_bf16": 8,
          "v_mfma_i32_16x16x32_i8": 8, "v_mfma_f32_32x32x2_f32": 18, "v_mfma_f32_16x16x4_f32": 10}


def code_objects(data):
    """The gfx950 code objects of a library: entries of its offload bundles."""
    magic, at = b"__CLANG_OFFLOAD_BUNDLE__", 0
    while True:
        at = data.find(magic, at)
        if at < 0:
            return
        entry = at + len(magic) + 8
        for _ in range(struct.unpack_from("<Q", data, at + len(magic))[0]):
            offset, size, name = struct.unpack_from("<QQQ", data, entry)
            if b"gfx950" in data[entry + 24:entry + 24 + name]:
                yield data[at + offset:at + offset + size]
            entry += 24 + name
        at += len(magic)


def registers(text):
    found = set()
    for kind, one, low, high in re.findall(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])", text):
        found.update((kind, i) for i in (range(int(low), int(high) + 1) if one == "" else (int(one),)))
    return frozenset(found)


class Instruction(object):
    def __init__(self, address, text):
        self.address, self.text = address, text
        self.op, _, operands = text.partition(" ")
        self.operands = [o.strip() for o in operands.split(",")] if operands else []
        self.target, self._taken = None, None

    @property
    def taken(self):
        """What an ordinary instruction reads or overwrites, and a matrix instruction reads as its factors."""
        if self._taken is None:
            operands = self.operands
            if self.op.startswith("v_mfma"):
                operands = operands[1:3]
            elif re.match(r"(ds_read|ds_bpermute|ds_permute|global_load|buffer_load|flat_load|scratch_load)", self.op):
                operands = operands[1:]                    # (their result comes later still)
            elif not re.match(r"(v_|ds_|global_|buffer_|flat_|scratch_)", self.op):
                operands = []
            self._taken = registers(",".join(operands))
        return self._taken


def kernels(listing):
    """Functions of a listing as lists of instructions, whose branches name the index they go to."""
    line = re.compile(r"^\t(.+?)\s*// 0*([0-9A-F]+):(?:[^<]*<(.+)\+0x([0-9a-f]+)>)?")
    name, start, body = None, 0, []
    for text in listing.splitlines() + ["0 <>:"]:
        head = re.match(r"^([0-9a-f]+) <(.*)>:$", text)
        if head:
            if body:
                index = {x.address: i for i, x in enumerate(body)}
                for x in body:
                    x.target = index.get(x.target)
                yield name, body
            start, name, body = int(head.group(1), 16), head.group(2), []
            continue
        m = line.match(text)
        if m:
            x = Instruction(int(m.group(2), 16), m.group(1).strip())
            if x.op in ("s_branch",) or x.op.startswith("s_cbranch"):
                x.target = start + int(m.group(4), 16) if m.group(4) else start
            body.append(x)


def too_early(body, states=None):
    """(matrix instruction, one that takes its result, states that it needs, states between them) along every way through the code."""
    found = []
    for i, product in enumerate(body):
        if not product.op.startswith("v_mfma"):
            continue
        need = (states or STATES)[product.op]
        ways, seen = [(i + 1, 0, registers(product.operands[0]))], {}
        while ways:
            j, passed, live = ways.pop()
            while j < len(body) and passed < need and live:
                if seen.get(j, need) <= passed:
                    break
                seen[j] = passed
                x = body[j]
                if x.taken & live:
                    found.append((product.text, x.text, need, passed))
                    break
                if x.op.startswith("v_mfma"):
                    live = live - registers(x.operands[0])  # (a sum carried on is handed over inside the unit)
                if x.op == "s_endpgm":
                    break
                passed += int(x.operands[0], 0) + 1 if x.op == "s_nop" else 1
                if x.target is not None:
                    if x.op == "s_branch":
                        j = x.target
                        continue
                    ways.append((x.target, passed, live))
                j += 1
    return found


def listings():
    if OBJDUMP is None:
        pytest.skip("no llvm-objdump")
    if not os.path.exists(LIB):
        from cubert_amd import build
        build.build()
    import tempfile
    for code in code_objects(open(LIB, "rb").read()):
        with tempfile.NamedTemporaryFile(suffix=".co") as f:
            f.write(code)
            f.flush()
            yield subprocess.run([OBJDUMP, "-d", f.name], stdout=subprocess.PIPE, check=True, text=True).stdout


@pytest.fixture(scope="module")
def functions():
    return [f for listing in listings() for f in kernels(listing)]


def code(*lines):
    """A listing of instructions at 4 bytes each; a line may be (text, index it goes to)."""
    out = ["0000000000000100 <f>:"]
    for i, x in enumerate(lines):
        text, to = x if isinstance(x, tuple) else (x, None)
        out.append("\t%s // %012X: 00000000%s" % (text, 0x100 + 4 * i, "" if to is None else " <f+0x%x>" % (4 * to)))
    return next(kernels("\n".join(out)))[1]


def test_the_reader_finds_what_comes_too_early():
    product = "v_mfma_f32_32x32x2_f32 v[0:15], v20, v21, v[0:15]"
    assert not too_early(code(product, "s_nop 15", "s_nop 1", "v_add_f32_e32 v30, v3, v31", "s_endpgm"))
    for last in ("v_add_f32_e32 v30, v3, v31", "v_mov_b32_e32 v15, 0", "ds_write_b128 v40, v[4:7]", "global_store_dword v2, v40, s[0:1]",
                 "v_mfma_f32_32x32x2_f32 v[40:55], v3, v60, 0", "ds_read_b32 v50, v9", "v_accvgpr_write_b32 a3, v9"):
        found = too_early(code(product, "s_nop 15", "s_nop 0", last, "s_endpgm"))
        assert [f[2:] for f in found] == [(18, 17)], last
    for last in ("v_add_f32_e32 v30, v16, v31", "v_mfma_f32_32x32x2_f32 v[0:15], v22, v23, v[0:15]", "ds_read_b32 v3, v16"):
        assert not [f for f in too_early(code(product, last, "s_endpgm")) if f[1] == last], last
    # along a branch that is taken: 1 and 3 states; on the way straight on enough
    found = too_early(code(product, ("s_cbranch_vccnz 20", 4), "s_nop 15", "s_nop 1", "s_nop 2", "v_max_f32_e32 v1, v1, v2", "s_endpgm"))
    assert [f[2:] for f in found] == [(18, 4)]
    found = too_early(code(product, ("s_branch 2", 3), "v_mov_b32_e32 v1, 0", "s_nop 9", ("s_cbranch_scc0 65533", 2), "s_endpgm"))
    assert [f[2:] for f in found] == [(18, 12)]


def test_the_guard_alone_is_long_enough(functions):
    """products_done() stands where the compiler's count was seen to fail, so it counts on nothing else."""
    for kind in ("attention_window_spread_kernel", "attention_window_shared_kernel", "attention_window_terms_kernel"):
        bodies = [body for name, body in functions if kind in name]
        assert bodies
        for body in bodies:
            runs = []                                      # of s_nop instructions that begin with the longest there is
            for x, y in zip(body, body[1:]):
                if x.text == "s_nop 15":
                    runs.append(16 + (int(y.operands[0], 0) + 1 if y.op == "s_nop" else 0))
            assert max(runs, default=0) > max(STATES.values()), kind


def test_copies_to_lds_count_on_nothing_else(functions):
    """Their statement has the five states that a scalar base written by a vector instruction needs, and gives m0 back."""
    copies = 0
    for name, body in functions:
        if "attention_window" not in name:
            continue
        for i, x in enumerate(body):
            if x.op == "global_load_lds_dwordx4" and x.operands[1].startswith("s["):
                copies += 1
                states, j = 0, i - 1
                while body[j].op in ("s_nop", "s_mov_b32") and body[j].operands[-1] != "m0":
                    states += int(body[j].operands[0], 0) + 1 if body[j].op == "s_nop" else 1
                    j -= 1
                kept = body[j].operands
                assert body[j].op == "s_mov_b32" and kept[1] == "m0" and states + 1 >= 5, (name, x.text)
                assert body[i + 1].op == "s_mov_b32" and body[i + 1].operands == ["m0", kept[0]], (name, x.text)
    assert copies > 100


def test_results_of_matrix_instructions_are_waited_for(functions):
    assert sum(any(x.op.startswith("v_mfma") for x in body) for _, body in functions) > 50
    unknown = {x.op for _, body in functions for x in body if x.op.startswith("v_mfma")} - set(STATES)
    assert not unknown, "states of %s" % sorted(unknown)
    wrong = [(name,) + f for name, body in functions for f in too_early(body)]
    assert not wrong, "%d ways, such as %s" % (len(wrong), "; ".join("%s: %s -> %s, %d states and %d" % w for w in wrong[:4]))
