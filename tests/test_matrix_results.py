"""Listings of the library that is built: no instruction reads the result of a matrix product before it is there.

The hardware does not wait for that; the compiler counts the instructions in between, but where a branch skips a block it
counts those of the block on the path without them too, and rows come out wrong now and then.  The kernels wait
before such branches themselves (``settle`` in ``csrc/ftc_delta_kernel.h``).  Every path behind every product is followed here."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from fast_transformers_amd import _native

# Instructions (s_nop n is n + 1 of them) between a product and the first use of its result, as the compiler keeps them
# within a block: passes + 4 of bf16 and fp16 products, passes + 2 of fp32 ones.
BETWEEN = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_32x32x16_bf16": 12,
           "v_mfma_f32_32x32x16_f16": 12, "v_mfma_f32_16x16x4_f32": 10}
BRANCH = 2  # a wavefront issues nothing until its branch is decided

REGISTERS = re.compile(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(text):
    found = set()
    for kind, first, last, one in REGISTERS.findall(text):
        found.update((kind, i) for i in range(int(one or first), int(one or last) + 1))
    return found


def operands(line):
    parts = line.split(None, 1)
    return parts[0], [x.strip() for x in re.split(r",(?![^\[]*\])", parts[1])] if len(parts) > 1 else []


def functions(listing):
    """(name, instructions, {label: index}) of a disassembly with labels."""
    name, lines, labels = None, [], {}
    for line in listing.splitlines():
        line = line.split("//")[0].rstrip()
        head = re.match(r"<(\S+)>:", line)
        if head and re.fullmatch(r"L\d+", head.group(1)):
            labels[head.group(1)] = len(lines)
        elif head:
            if name:
                yield name, lines, labels
            name, lines, labels = head.group(1), [], {}
        elif name and line[:1].isspace() and line.strip():
            lines.append(line.strip())
    if name:
        yield name, lines, labels


def too_early(lines, labels):
    """(product, user, instructions in between) of every result that is used too early on some path."""
    split = [operands(line) for line in lines]
    found = []
    for i, (op, args) in enumerate(split):
        if not op.startswith("v_mfma"):
            continue
        assert op in BETWEEN, "how long %s takes is not known here" % op
        result = registers(args[0])
        todo, seen = [(i + 1, 0)], {}
        while todo:
            at, passed = todo.pop()
            while at < len(split) and passed < BETWEEN[op]:
                if seen.get(at, 1 << 30) <= passed:
                    break
                seen[at] = passed
                other, given = split[at]
                if other.startswith("v_mfma"):
                    if (registers(given[1]) | registers(given[2])) & result:
                        found.append((lines[i], lines[at], passed))
                        break
                    if registers(given[0]) & result:  # (adds to it, or replaces it: products stay in order)
                        break
                elif re.match(r"v_|ds_|global_|buffer_|flat_|scratch_", other) and registers(" ".join(given)) & result:
                    found.append((lines[i], lines[at], passed))
                    break
                if other.startswith(("s_branch", "s_cbranch")):
                    passed += BRANCH
                    todo.append((labels[given[0]], passed))
                    if other == "s_branch":
                        break
                elif other == "s_endpgm":
                    break
                else:
                    passed += int(given[0], 0) + 1 if other == "s_nop" else 1
                at += 1
    return found


def tool(name):
    for folder in ("/opt/rocm/llvm/bin", "/opt/rocm/lib/llvm/bin"):
        if os.path.exists(os.path.join(folder, name)):
            return os.path.join(folder, name)
    return shutil.which(name)


def device_code(fat):
    """The gfx950 objects in a library's section of bundles."""
    for found in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", fat):
        at = found.end()
        (count,) = struct.unpack_from("<Q", fat, at)
        at += 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", fat, at)
            target = fat[at + 24:at + 24 + length]
            at += 24 + length
            if b"gfx950" in target and size:
                yield fat[found.start() + offset:found.start() + offset + size]


def test_no_result_of_a_matrix_product_is_read_early(tmp_path):
    objdump, objcopy = tool("llvm-objdump"), tool("llvm-objcopy")
    if not (objdump and objcopy):
        pytest.skip("needs llvm-objdump and llvm-objcopy")
    fat = tmp_path / "fat"
    subprocess.check_call([objcopy, "--dump-section", ".hip_fatbin=%s" % fat, _native.LIB_PATH, os.devnull])
    running = []
    for i, code in enumerate(device_code(fat.read_bytes())):
        path, listing = tmp_path / ("%d.o" % i), tmp_path / ("%d.s" % i)
        path.write_bytes(code)
        with open(listing, "w") as out:
            running.append((listing, subprocess.Popen(
                [objdump, "-d", "--symbolize-operands", "--no-show-raw-insn", "--no-leading-addr", str(path)], stdout=out)))
    products, early = 0, []
    for listing, process in running:
        assert process.wait() == 0
        for name, lines, labels in functions(listing.read_text()):
            products += sum(line.startswith("v_mfma") for line in lines)
            early += [(name, *found) for found in too_early(lines, labels)]
    assert products > 10000
    assert not early, early[:5]


PRODUCT = "v_mfma_f32_16x16x32_bf16 a[0:3], v[2:5], v[6:9], a[0:3]"


@pytest.mark.parametrize("between, early", [
    (["s_nop 6"], True), (["s_nop 7"], False), (["v_add_f32_e32 v20, v21, v22"] * 7, True),
    (["v_mfma_f32_16x16x32_bf16 a[16:19], v[2:5], v[6:9], a[16:19]"] * 8, False),
    (["s_cbranch_vccz L0"] + ["v_add_f32_e32 v20, v21, v22"] * 8 + ["L0", "s_nop 4"], True),   # what a branch skips does not count
    (["s_cbranch_vccz L0"] + ["v_add_f32_e32 v20, v21, v22"] * 8 + ["L0", "s_nop 5"], False),
    (["s_branch L0", "L1", "s_nop 7", "s_endpgm", "L0", "s_nop 2"], True),
    (["s_branch L0", "L1", "v_accvgpr_read_b32 v4, a1", "s_endpgm", "L0", "s_nop 7"], False),
])
@pytest.mark.parametrize("use", ["v_accvgpr_read_b32 v9, a2", "global_store_dwordx4 v[10:11], a[0:3], off",
                                 "v_mfma_f32_16x16x32_bf16 a[8:11], a[2:5], v[6:9], a[8:11]"])
def test_the_check_itself(between, early, use):
    body = [PRODUCT] + between + [use, "s_endpgm"]
    listing = "<kernel>:\n" + "\n".join("<%s>:" % l if re.fullmatch(r"L\d", l) else "\t" + l for l in body) + "\n"
    ((name, lines, labels),) = functions(listing)
    assert name == "kernel" and bool(too_early(lines, labels)) == early


def test_sums_in_place_are_no_use():
    ((_, lines, labels),) = functions("<kernel>:\n\t%s\n\t%s\n\ts_nop 7\n\tv_accvgpr_read_b32 v9, a2\n\ts_endpgm\n" % (PRODUCT, PRODUCT))
    assert not too_early(lines, labels)
