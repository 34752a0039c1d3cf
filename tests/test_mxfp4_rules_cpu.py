"""Sizes, addresses and waits of the MXFP4 row kernels, asked of what they are built from.  No GPU needed."""
import ctypes
import os
import random
import re
import subprocess

import pytest

from nn_amd import _lib, build


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


# ---- which form a shape takes -----------------------------------------------------------

BF16, F32, QUANT_BF16, QUANT_F32, CODES = range(5)  # kinds of x (MxInput)


def form(lib, m, n, k, x):
    """("rows", kind, pairs of a wave) or ("gemm", operands, 32-row tiles, 128-column tiles)"""
    lib.nnq_rule_mx.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    f = (ctypes.c_int * 4)()
    if lib.nnq_rule_mx(m, n, k, x, f):
        kind = {BF16: "X_BF16", F32: "X_TRI" if m <= 5 else "X_PLANES", QUANT_BF16: "X_Q16", QUANT_F32: "X_Q32", CODES: "X_CODES"}[x]
        return "rows", kind, f[0]
    return ("gemm16", f[0], f[1], 3 if x == F32 else 1) if x in (BF16, F32) else ("gemm4", f[0], f[1])


def built_forms():
    """the kernels' instantiations, from the calls that launch them"""
    gemm = open(os.path.join(build.CSRC, "nnq_mxfp4_gemm.hip")).read()
    rows = open(os.path.join(build.CSRC, "nnq_mxfp4.hip")).read()
    forms = {("gemm16", *map(int, g)) for g in re.findall(r"launch16<(\d), (\d), (\d)>\(", gemm)}
    forms |= {("gemm4", *map(int, g)) for g in re.findall(r"launch4<(\d), (\d)>\(", gemm)}
    counts = [int(c) for c in re.findall(r"launch_rows_t<XF, (\d)>\(", rows)]
    for kind in re.findall(r"launch_rows_x<(X_\w+)>\(", rows):
        forms |= {("rows", kind, c) for c in counts if kind != "X_PLANES" or c <= 2}
    assert "if constexpr (XF != X_PLANES)" in rows
    return forms


def test_every_built_form_is_some_shapes(lib):
    """and every shape's form is built"""
    rng = random.Random(5)
    log = lambda lo, hi: round(lo * (hi / lo) ** rng.random())
    seen = set()
    for _ in range(150000):
        m = rng.choice((log(1, 16), log(17, 9000)))
        seen.add(form(lib, m, log(1, 300000), 32 * log(1, 1 << 15), rng.randrange(5)))
    assert seen == built_forms(), (seen ^ built_forms())


# ---- addresses ----------------------------------------------------------------------------


@pytest.mark.parametrize("planes", [1, 3])
def test_copies_of_x_stay_in_its_planes(lib, planes):
    """The GEMM with bf16 operands copies 16 bytes at (offset of a lane) + (plane and unit, a scalar offset).  A buffer's range
    check is only documented to count the lane's offset, so that one has to keep every copy in the planes by itself: of all rows of
    the last row block, those past m too, and all columns of a unit that K ends in."""
    lib.nnq_rule_mx_x_offset.argtypes = [ctypes.c_int] * 5
    rng = random.Random(planes)
    cases = [(17, 32, 64), (33, 2880, 64), (64, 384, 64), (65, 1056, 64), (1, 160, 32), (129, 4096, 128)]
    cases += [(rng.randint(1, 300), 32 * rng.randint(1, 40), rng.choice((32, 64))) for _ in range(12)]
    for m, k, tile in cases:
        total = planes * m * k * 2
        units = (k + 127) // 128
        read = set()
        for row in range((m + tile - 1) // tile * tile):
            for u in {0, units // 2, units - 1}:
                for col in range(0, 128, 8):
                    off = lib.nnq_rule_mx_x_offset(row, m, k, u, col)
                    if off >= total:
                        assert off >= 0x7FFFFFF0 and (row >= m or 128 * u + col >= k)
                        continue
                    for plane in range(planes):
                        at = off + plane * m * k * 2 + 256 * u
                        assert at == 2 * ((plane * m + row) * k + 128 * u + col) and at + 16 <= total, (m, k, row, u, col, plane)
                    read.add((row, u, col))
        assert len(read) == m * sum(min(128, k - 128 * u) // 8 for u in {0, units // 2, units - 1})


# ---- counted waits ------------------------------------------------------------------------


def kernel_blocks(asm):
    """(kernel, its blocks) of both GEMMs; a block: [what it does in order], a copy into LDS "copy", another load "load", a
    barrier "barrier", a wait for memory its count, a jump the label"""
    for m in re.finditer(r"^(\S*mx_gemm(16|4)_kernelILi(\d)ELi(\d)E(?:Li(\d)E)?\S*):(.*?)^\.Lfunc_end", asm, re.S | re.M):
        blocks = {"": []}
        for line in m.group(6).splitlines():
            t = line.strip()
            if label := re.match(r"(\.LBB\w+):", t):
                blocks[label.group(1)] = ops = []
                continue
            ops = blocks[list(blocks)[-1]]
            if re.match(r"buffer_load_\w+ .*\blds\b", t):
                ops.append("copy")
            elif re.match(r"(buffer|global)_load_", t):
                ops.append("load")
            elif t.startswith("s_barrier"):
                ops.append("barrier")
            elif w := re.match(r"s_waitcnt.*vmcnt\((\d+)\)", t):
                ops.append(int(w.group(1)))
            elif jump := re.match(r"s_c?branch\w* (\.LBB\w+)", t):
                ops.append(jump.group(1))
        yield tuple(int(g) for g in m.group(2, 3, 4, 5) if g), list(blocks.items())


def early_reads(kernel, blocks):
    """Stages whose barrier is passed with a copy of theirs in flight: the prologue, the loop (two stages) so many times, and
    the stage of an odd number, as a wave's loads and copies return in order.  Waits that the compiler adds for a load's value may
    go with it, and do not count."""
    bits, mt, nt = kernel[:3]
    copies = mt + 1 if bits == 4 else 2 * mt * kernel[3]  # of a wave and stage
    at = next(i for i, (label, ops) in enumerate(blocks) if label in ops and ops.count("barrier") == 2)
    loop = blocks[at][1]
    wait = max(o for o in loop if isinstance(o, int) and loop[loop.index(o) + 1] == "barrier")
    tail = next(ops for _, ops in blocks[at + 1:] if any(a == wait and b == "barrier" for a, b in zip(ops, ops[1:])))
    prologue = [o for _, ops in blocks[:at] for o in ops if o in ("copy", "load")]
    found = []
    for turns in (0, 1, 3):
        flight, issued, stage = [], 0, 0
        path = prologue + turns * loop + tail
        for op, then in zip(path, path[1:] + [None]):
            if op == "copy":
                flight.append(issued // copies)  # the stage it is for
                issued += 1
            elif op == "load":
                flight.append(None)
            elif op == "barrier":
                if any(f is not None and f <= stage for f in flight):
                    found.append((kernel, turns, stage))
                stage += 1
            elif isinstance(op, int) and then == "barrier":
                flight = flight[max(0, len(flight) - op):]
        assert stage == 2 * turns + 1
    # the outputs pass through what held the copies: behind the last stage the next barrier follows a wait for all of them
    behind = [o for _, ops in blocks[[b for _, b in blocks].index(tail) + 1:] for o in ops]
    if behind[behind.index("barrier") - 1] != 0:
        found.append((kernel, "outputs", None))
    return found


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="needs hipcc")
def test_gemm_waits_cover_their_copies(tmp_path):
    """A stage's copies are waited for by a count of what is issued behind them, so the compiler must neither move a load of
    the weights in front of a copy nor delete one.  Nothing on the GPU shows that reliably: the assembly is read."""
    out = str(tmp_path / "gemm.s")
    subprocess.run([build.HIPCC, f"--offload-arch={build.ARCH}", *build.COMMON, *build.DEVICE_FLAGS,
                    *build.EXTRA_FLAGS.get("nnq_mxfp4_gemm.hip", []), "--cuda-device-only", "-S",
                    os.path.join(build.CSRC, "nnq_mxfp4_gemm.hip"), "-o", out], check=True, stdout=subprocess.DEVNULL,
                   stderr=subprocess.DEVNULL)
    kernels = list(kernel_blocks(open(out).read()))
    assert {k[0] for k, _ in kernels} == {16, 4} and len(kernels) >= 10
    for kernel, blocks in kernels:
        assert early_reads(kernel, blocks) == []
        # a load in front of the copies of a stage would be seen
        for i, (_, ops) in enumerate(blocks):
            if ops.count("barrier") == 2:
                first, last = ops.index("copy"), len(ops) - 1 - ops[::-1].index("copy")
                later = next(j for j in range(last, len(ops)) if ops[j] == "load")
                moved = ops[:]
                moved.insert(first, moved.pop(later))
                assert early_reads(kernel, blocks[:i] + [(blocks[i][0], moved)] + blocks[i + 1:])
                break
    # nothing but the fences keeps that order: one stands behind every call that issues copies
    text = open(os.path.join(build.CSRC, "nnq_mxfp4_gemm.hip")).read()
    calls = re.findall(r"^ *copy_a\([^;]*\);\n(.*\n)?(.*)$", text, re.M)
    assert len(calls) == 4
    for between, line in calls:
        assert "__builtin_amdgcn_sched_barrier(0);" in between + line, (between, line)
