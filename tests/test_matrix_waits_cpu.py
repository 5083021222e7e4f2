"""Results of matrix instructions are read when they are there: on every way through the compiled attention kernels as many wait states lie between a product and the first
vector, LDS or memory instruction that touches its sum as the instruction asks for.  The compiler sees to that, but behind branches over a few instructions it has counted the
longer way only.  No GPU needed."""
import os
import re
import subprocess
from concurrent.futures import ProcessPoolExecutor

from ratchet_amd import build
from test_kernel_resources_cpu import code_objects

OBJDUMP = os.path.join(os.path.dirname(os.path.dirname(build.HIPCC)), "llvm", "bin", "llvm-objdump")
LINE = re.compile(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+): ")
REGISTERS = re.compile(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+)\b)")
TOUCH = ("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")


def wait_states(op):
    """for vectors' reads: two more than the passes of an f32 product, four more than those of a 16-bit one"""
    if "x2_f32" in op or "32x32x2f32" in op:
        return 16 + 2
    if "x4_f32" in op or "16x16x4f32" in op:
        return 8 + 2
    return (8 if "32x32" in op else 4) + 4


def registers(text):
    out = set()
    for kind, low, high, one in REGISTERS.findall(text):
        out.update((kind, n) for n in range(int(low or one), int(high or one) + 1))
    return out


def too_early(code):
    """[(product, wait states, reader)] of one kernel, whose code is [(address, mnemonic, operands)]"""
    index = {at: i for i, (at, _, _) in enumerate(code)}
    touched, out = {}, []

    def touches(i):
        if i not in touched:
            touched[i] = frozenset(registers(code[i][2])) if code[i][1].startswith(TOUCH) else frozenset()
        return touched[i]

    for i, (_, op, text) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        result, need, best, ways = registers(text.split(",")[0]), wait_states(op), {}, [(i + 1, 0)]
        while ways:
            j, states = ways.pop()
            if j >= len(code) or states >= need or best.get(j, need) <= states:
                continue
            best[j] = states
            at, name, operands = code[j]
            if touches(j) & result:
                if not name.startswith("v_mfma"):
                    out.append((op, states, name + " " + operands))
                    continue
                if registers(operands.split(",")[0]) >= result:  # the next product of the same sum
                    continue
            if name in ("s_endpgm", "s_setpc_b64"):
                continue
            if name.startswith(("s_branch", "s_cbranch")):
                offset = int(operands.split()[0])
                ways.append((index[at + 4 + 4 * (offset - 65536 if offset >= 32768 else offset)], states + 1))
                if name == "s_branch":
                    continue
            ways.append((j + 1, states + (int(operands, 0) + 1 if name == "s_nop" else 1)))
    return out


def check(path):
    """(kernels with products, products, those whose result is read too early) of a code object's attention kernels"""
    kernels, products, bad, code, name = 0, 0, [], [], None

    def finish():
        nonlocal kernels, products
        n = sum(op.startswith("v_mfma") for _, op, _ in code)
        if n:
            kernels, products = kernels + 1, products + n
            bad.extend((name,) + x for x in too_early(code))

    with subprocess.Popen([OBJDUMP, "-d", "--mcpu=gfx950", path], stdout=subprocess.PIPE, text=True) as dump:
        for line in dump.stdout:
            head = re.match(r"^[0-9a-f]+ <(.*)>:", line)
            if head:
                finish()
                name, code = head.group(1), []
            elif name and "attention" in name:
                m = LINE.match(line)
                if m:
                    code.append((int(m.group(3), 16), m.group(1), m.group(2)))
    finish()
    return kernels, products, bad


def test_the_check_finds_a_short_way():
    """a product, a branch over what waits, and a read"""
    code = [(0, "v_mfma_f32_16x16x16_f16", "a[0:3], v[0:1], v[2:3], a[0:3]"), (8, "s_cbranch_scc1", "3"), (12, "s_nop", "7"), (16, "s_nop", "7"), (20, "s_nop", "0"),
            (24, "s_nop", "0"), (28, "v_accvgpr_read_b32", "v5, a3"), (36, "s_endpgm", "")]
    assert too_early(code) == [("v_mfma_f32_16x16x16_f16", 2, "v_accvgpr_read_b32 v5, a3")]
    code[5] = (24, "s_nop", "6")
    assert too_early(code) == []


def test_products_are_waited_for(tmp_path):
    paths = []
    for k, co in enumerate(code_objects()):
        if b"attention" in co:
            paths.append(str(tmp_path / ("%d.co" % k)))
            open(paths[-1], "wb").write(co)
    with ProcessPoolExecutor(4) as pool:
        results = list(pool.map(check, paths))
    assert sum(r[0] for r in results) >= 200 and sum(r[1] for r in results) >= 10000, results
    bad = [x for r in results for x in r[2]]
    assert not bad, (len(bad), bad[:10])
