"""Wait states of the assembly blocks in the 8-bit products and in differential attention's chunk kernel, in the device code the compiler makes of
them: those of the copies into LDS (test_wait_states.py), and those of the score products, matrix instructions of 32 x 32 x 16 whose sums vector
instructions read.  Such a read wants 18 wait states behind the last product into those registers; a product of that size holds
the matrix pipe for eight, so that it counts as eight where it is issued behind another one.  And a product wants two behind a vector
instruction that writes one of its operands."""
import os
import re
import shutil
import subprocess

import pytest

from tests.test_wait_states import _missing
from tinytitan_amd import build

pytestmark = pytest.mark.skipif(shutil.which(build.HIPCC) is None, reason="no hipcc")

ENOUGH, PRODUCT, OPERAND = 18, 8, 2


def _vectors(operand):
    """The vector registers that an operand names."""
    m = re.match(r"\s*-?\|?v\[(\d+):(\d+)\]|\s*-?\|?v(\d+)\b", operand)
    if not m:
        return set()
    return set(range(int(m[1]), int(m[2]) + 1)) if m[1] else {int(m[3])}


def early_reads(listing):
    """Instructions that read or write a score product's registers too early, and how many such products there are.  A product may take the
    registers of the one before it as its own sum."""
    function, found, products, in_block = "", [], 0, False
    written, now = {}, 0  # register -> states at the last product into it
    made = {}             # ... behind the last vector instruction that wrote it
    for line in listing.splitlines():
        label = re.match(r"(_Z\w+):", line)
        if label:
            function, written, made = label[1], {}, {}
        if "#ASMSTART" in line or "#ASMEND" in line:
            in_block = "#ASMSTART" in line
        text = line.split(";")[0].strip()
        if not text or text.startswith(".") or text.endswith(":"):
            continue
        op, _, operands = text.partition(" ")
        parts = operands.split(",")
        if op.startswith("v_mfma") and in_block:
            target = _vectors(parts[0])
            assert target, text  # (a score product's sum is in vector registers)
            for part in parts[1:3]:
                found += [(function, text) for reg in _vectors(part) if now - written.get(reg, -99) < ENOUGH]
            found += [(function, text) for part in parts[1:] for reg in _vectors(part) if now - made.get(reg, -99) < OPERAND]
            third = _vectors(parts[3])
            assert not third or third == target, text
            if not third:  # (the first of a sum: nobody may still be reading the old one, which was read behind its own products)
                found += [(function, text) for reg in target if now - written.get(reg, -99) < ENOUGH]
            now += PRODUCT
            written.update({reg: now - PRODUCT + 1 for reg in target})
            products += 1
            continue
        if op.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")):
            for part in parts:
                found += [(function, text) for reg in _vectors(part) if now - written.get(reg, -99) < ENOUGH]
        now += PRODUCT if op.startswith("v_mfma") else int(operands, 0) + 1 if op == "s_nop" else 1
        if op.startswith("v_"):
            made.update({reg: now for reg in _vectors(parts[0])})
    return found, products


def _listing(tmp_path, source):
    listing = tmp_path / "device.s"
    subprocess.run([build.HIPCC, *build.FLAGS, "--cuda-device-only", "-S", os.path.join(build.CSRC, source), "-o", str(listing)], check=True,
                   capture_output=True)
    return listing.read_text()


@pytest.fixture(scope="module")
def int8_listing(tmp_path_factory):
    return _listing(tmp_path_factory.mktemp("int8"), "int8_proj.hip")


@pytest.mark.parametrize("source", ["attn_maps_chunk.hip", "int8_proj.hip"])
def test_copies_into_lds_wait_for_what_they_read(tmp_path, source):
    missing, copies, clobbered = _missing(_listing(tmp_path, source))
    assert copies > 20
    assert not clobbered
    assert not missing, f"{len(missing)}, e.g. {missing[0]}"


def test_scores_are_read_behind_their_products(tmp_path):
    listing = _listing(tmp_path, "attn_maps_chunk.hip")
    found, products = early_reads(listing)
    assert products == (2 * 2 + 4 + 8 * 2) * 2  # heads of 64, 128 and 256, two tiles or one, in front of the loop and in it
    assert not found, f"{len(found)}, e.g. {found[0]}"
    assert "v_cmpx" not in listing  # (a product behind a change of the lanes at work would want wait states, too)


def test_the_check_sees_an_early_read():
    product = "\t;;#ASMSTART\n\tv_mfma_f32_32x32x16_f16 v[0:15], v[20:23], v[24:27], 0\n\t;;#ASMEND\n"
    read = "\tv_max3_f32 v30, v3, v31, v32\n"
    other = "\tv_mfma_f32_32x32x16_f16 a[0:15], v[40:43], v[44:47], a[0:15]\n"
    assert early_reads("_Zf:\n" + product + read)[0]
    assert early_reads("_Zf:\n" + product + other + read)[0]
    assert not early_reads("_Zf:\n" + product + other * 2 + "\ts_nop 1\n" + read)[0]
    assert not early_reads("_Zf:\n" + product + "\ts_nop 15\n\ts_nop 7\n" + read)[0]
    operand = "\tv_accvgpr_read_b32 v22, a3\n"
    assert early_reads("_Zf:\n" + operand + product)[0]
    assert early_reads("_Zf:\n" + operand + "\ts_nop 0\n" + product)[0]
    assert not early_reads("_Zf:\n" + operand + "\ts_nop 1\n" + product)[0]


# The chunk kernel's copies of V, in the order that one wavefront issues them, along every way through its code: by the n-th barrier those of the
# walk's first n blocks have landed, whatever else is on its way.  (Vector memory operations end in order, as far as a wait counts them.)
COPIES = {256: 4, 128: 1, 64: 1}  # a wavefront's of a block


def late_copies(listing, name, copies, barriers):
    """Places of the first `barriers` barriers that some way reaches with a copy of an earlier block on its way, and how many barriers were reached."""
    body = listing[re.search(r"^%s:" % re.escape(name), listing, re.M).end():].split(".Lfunc_end")[0].partition("\n")[2]
    code, labels = [], {}
    for line in body.splitlines():
        text = line.split(";")[0].strip()
        if text.endswith(":"):
            labels[text[:-1]] = len(code)
        elif text and not text.startswith("."):
            code.append(text)
    late, reached, seen, ways = [], 0, set(), [(0, (), 0, 0)]
    while ways:
        at, flying, copied, passed = way = ways.pop()
        if way in seen or at >= len(code):
            continue
        seen.add(way)
        op, _, operands = code[at].partition(" ")
        if op == "s_endpgm":
            continue
        if op == "s_waitcnt":
            m = re.search(r"vmcnt\((\d+)\)", operands)
            if m:
                flying = flying[max(len(flying) - int(m[1]), 0):]
                while flying and flying[0] < 0:
                    flying = flying[1:]
        elif op.startswith(("global_", "buffer_", "flat_", "scratch_")):
            lds = "lds" in op
            if lds or flying:  # (what is older than every copy on its way changes nothing for them)
                flying = flying + (copied if lds else -1,)
            copied += lds
        elif op == "s_barrier":
            passed += 1
            reached = max(reached, passed)
            late += [at for c in flying if 0 <= c < passed * copies]
            if passed == barriers:
                continue
        target = operands.strip() if op.startswith(("s_branch", "s_cbranch")) else None
        if target is not None:
            ways.append((labels[target], flying, copied, passed))
        if op != "s_branch":
            ways.append((at + 1, flying, copied, passed))
    return late, reached


@pytest.mark.parametrize("dim", [256, 128, 64])
def test_values_have_landed_by_the_barrier_in_front_of_them(tmp_path, dim):
    listing = _listing(tmp_path, "attn_maps_chunk.hip")
    name = re.search(r"^(_ZN2tt\w*attn_maps_chunk_kernelILi%dE\w*):" % dim, listing, re.M)[1]
    late, reached = late_copies(listing, name, COPIES[dim], 5)
    assert reached == 5
    assert not late


@pytest.mark.parametrize("kernel,tm,tn", [("int8_gemm", 256, 256), ("int8_gemm", 128, 256), ("int8_gemm", 128, 128), ("int8_gemm", 128, 64),
                                          ("int8_gemm", 64, 128), ("int8_steps", 64, 64)])
def test_stages_of_a_product_have_landed_by_their_barriers(int8_listing, kernel, tm, tn):
    name = re.search(r"^(_ZN2tt\w*%s_kernelILi%dELi%dE\w*):" % (kernel, tm, tn), int8_listing, re.M)[1]
    late, reached = late_copies(int8_listing, name, (tm + tn) // 32, 4)
    assert reached == 4
    assert not late


def test_the_check_sees_a_late_copy():
    def listing(wait):
        return "k:\n\tglobal_load_lds_dwordx4 v1, s[0:1]\n\tbuffer_load_dwordx4 v[0:3], v9, s[4:7], 0 offen\n\ts_cbranch_scc1 .LBB0_1\n\ts_waitcnt vmcnt(0)\n" \
               ".LBB0_1:\n\ts_waitcnt vmcnt(%d)\n\ts_barrier\n\ts_endpgm\n.Lfunc_end0:\n" % wait
    assert late_copies(listing(2), "k", 1, 1) == ([6 - 1], 1)
    assert late_copies(listing(1), "k", 1, 1) == ([], 1)
