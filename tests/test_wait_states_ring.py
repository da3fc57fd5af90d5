"""The waits that the few tokens' 8-bit products count by hand, in the device code the compiler makes of them: a wavefront keeps a ring of stages in LDS,
copied there from memory, without a barrier.  Along every way through a kernel: a stage's copies have landed where its operands are read, the operands
of a stage have been read where the copies into its place begin, tokens as they come (the kernels that quantise them) have landed where they
are read, and nothing is on its way to LDS where the sums take the rings' place."""
import os
import re
import shutil
import subprocess
from typing import NamedTuple

import pytest

from tinytitan_amd import build

pytestmark = pytest.mark.skipif(shutil.which(build.HIPCC) is None, reason="no hipcc")

# row tiles, token tiles, wavefronts, stages of a ring, whether the kernel quantises the tokens
KERNELS = [(1, 1, 8, 2, 0), (1, 2, 8, 3, 0), (1, 3, 4, 4, 0), (1, 4, 4, 4, 0), (2, 1, 8, 2, 0), (2, 2, 8, 2, 0), (2, 3, 8, 2, 0), (2, 4, 4, 3, 0), (4, 1, 4, 3, 0),
           (4, 2, 4, 3, 0), (4, 3, 4, 2, 0), (1, 1, 8, 4, 1), (2, 1, 8, 3, 1), (4, 1, 4, 3, 1)]


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    out = tmp_path_factory.mktemp("ring") / "device.s"
    subprocess.run([build.HIPCC, *build.FLAGS, "--cuda-device-only", "-S", os.path.join(build.CSRC, "int8_proj.hip"), "-o", str(out)], check=True,
                   capture_output=True)
    return out.read_text()


def _body(listing, rt, nt, waves, depth, fused):
    name = re.search(r"^(_ZN2tt\w*int8_ring_kernelILi%dELi%dELi%dELi%dELb%dE\w*):" % (rt, nt, waves, depth, fused), listing, re.M)
    return listing[name.end():].split(".Lfunc_end")[0].partition("\n")[2]


def _scalars(operand):
    """The scalar registers that an operand names."""
    m = re.match(r"\s*s\[(\d+):(\d+)\]|\s*s(\d+)\b", operand)
    return set() if not m else set(range(int(m[1]), int(m[2]) + 1)) if m[1] else {int(m[3])}


class Way(NamedTuple):
    """A way through a kernel up to an instruction."""
    at: int = 0
    flying: tuple = ()    # copies on their way to LDS, in order: their stages, -1 of tokens
    lds: int = 0          # LDS operations on their way
    truths: tuple = ()    # (a scalar pair's first register, the truth value in it)
    vcc: str = ""         # "0", "-1": none or all of the lanes at work
    tokens: int = 0       # copies of tokens
    front: int = 0        # copies in front of the loop
    turn: int = -1
    made: int = 0         # copies of this turn
    stages: int = 0       # stages copied
    ended: bool = False   # a turn has copied none: there are no further stages


def faults(body, copies, depth):
    """(what is read or written too early on some way, and where; how many reads of a stage were looked at), for stages of `copies` copies each.

    Which ways there are follows from the number of a wavefront's stages: depth - 1 of them, or all if there are fewer, are copied in front of the loop;
    turn i reads stage i and copies stage i + depth - 1 where there is one.  What a way waits for is read from the code."""
    code, labels, header, block = [], {}, [], None
    for line in body.splitlines():
        text = line.split(";")[0].strip()
        if text.endswith(":"):
            labels[text[:-1]] = len(code)
            inner = re.search(r"in Loop: Header=(BB\w+)", line)
            block = inner[1] if inner else text[2:-1] if "Loop Header" in line else None
        elif text and not text.startswith("."):
            code.append(text)
            header.append(block)
    into_lds = [i for i, text in enumerate(code) if text.startswith("global_load_lds")]
    in_turn, in_front = into_lds[-copies:], into_lds[-2 * copies:-copies]
    head, in_loop = labels[".L" + header[in_turn[0]]], [h == header[in_turn[0]] for h in header]
    assert all(in_loop[i] for i in in_turn) and len(in_front) == copies and not any(in_loop[i] for i in in_front)
    found, looked, seen, ways = set(), set(), set(), [Way()]
    while ways:
        w = ways.pop()
        if w in seen:
            continue
        seen.add(w)
        op, _, operands = code[w.at].partition(" ")
        parts = [part.strip() for part in operands.split(",")]
        if op == "s_endpgm":
            continue
        if w.at == head:
            w = w._replace(turn=w.turn + 1, made=0)
            if w.turn >= w.stages or w.turn == 3 * depth:
                continue  # (no stage to read; far enough)
        full = w.front == copies * (depth - 1)
        if op.startswith("ds_read"):
            if w.turn < 0 and -1 in w.flying:
                found.add(("reads tokens on their way", w.at))
            if in_loop[w.at]:
                w = w._replace(ended=w.ended or not w.made)
                looked.add((w.at, w.turn))
                if any(s <= w.turn for s in w.flying):
                    found.add(("reads a stage on its way", w.at))
        if op.startswith("ds_"):
            w = w._replace(lds=min(w.lds + 1, 16))  # (what a wait counts to)
        elif w.at in in_front:
            if full:
                continue
            w = w._replace(flying=w.flying + (w.front // copies,), front=w.front + 1, stages=(w.front + 1) // copies)
        elif w.at in in_turn:
            if not full or w.ended:
                continue
            if w.lds:
                found.add(("copies over what is being read", w.at))
            w = w._replace(flying=w.flying + (w.turn + depth - 1,), made=w.made + 1, stages=w.stages + (w.made + 1 == copies))
        elif op.startswith("global_load_lds"):
            if w.tokens == 2:
                continue
            w = w._replace(flying=w.flying + (-1,), tokens=w.tokens + 1)
        elif op.startswith(("global_", "buffer_", "flat_", "scratch_", "s_load", "s_buffer")):
            assert not in_loop[w.at], code[w.at]  # (counts of their own)
        elif op == "s_waitcnt":
            m, n = re.search(r"vmcnt\((\d+)\)", operands), re.search(r"lgkmcnt\((\d+)\)", operands)
            if m and int(m[1]) and w.turn < 0 and not full:
                continue  # (the wait of a ring that is full)
            w = w._replace(flying=w.flying[max(len(w.flying) - int(m[1]), 0):] if m else w.flying, lds=min(w.lds, int(n[1])) if n else w.lds)
        elif op == "s_barrier" and w.at > in_turn[-1]:
            if w.stages == w.turn + 1 and w.flying:
                found.add(("the sums' place has copies on their way", w.at))
            continue
        if op == "s_andn2_b64" and parts[:2] == ["vcc", "exec"]:
            known = [value for register, value in w.truths if register in _scalars(parts[2])]
            w = w._replace(vcc={"0": "-1", "-1": "0"}[known[0]] if known else "")
        elif parts[0].startswith("vcc") or op.startswith("v_cmp"):
            w = w._replace(vcc="")
        written = _scalars(parts[0])
        if written and op.startswith(("s_", "v_readfirstlane", "v_cmp")):
            truths = tuple(t for t in w.truths if not {t[0], t[0] + 1} & written)
            w = w._replace(truths=truths + ((min(written), parts[1]),) if op == "s_mov_b64" and parts[1] in ("0", "-1") else truths)
        target = labels[parts[0]] if op.startswith(("s_branch", "s_cbranch")) else None
        taken = op == "s_branch" or (w.vcc == "-1" if w.vcc and op == "s_cbranch_vccnz" else w.vcc == "0" if w.vcc and op == "s_cbranch_vccz" else None)
        if target is not None and taken is not False:
            ways.append(w._replace(at=target))
        if target is None or taken in (None, False):
            ways.append(w._replace(at=w.at + 1))
    return found, len(looked)


@pytest.mark.parametrize("rt,nt,waves,depth,fused", KERNELS)
def test_stages_land_before_they_are_read_and_are_read_before_they_are_replaced(listing, rt, nt, waves, depth, fused):
    copies = 2 * rt + (0 if fused else 2 * nt)
    found, looked = faults(_body(listing, rt, nt, waves, depth, fused), copies, depth)
    assert looked >= 2 * depth * (rt + nt)
    assert not found


def test_every_ring_is_looked_at(listing):
    names = re.findall(r"^_ZN2tt\w*int8_ring_kernelILi(\d)ELi(\d)ELi(\d)ELi(\d)ELb(\d)E\w*:", listing, re.M)
    assert sorted(tuple(map(int, name)) for name in names) == sorted(KERNELS)


def _kinds(body, copies, depth):
    return {what for what, _ in faults(body, copies, depth)[0]}


def test_the_check_sees_what_is_too_early(listing):
    for rt, nt, waves, depth, fused in ((1, 2, 8, 3, 0), (2, 1, 8, 2, 0), (1, 1, 8, 4, 1)):
        body, copies = _body(listing, rt, nt, waves, depth, fused), 2 * rt + (0 if fused else 2 * nt)
        wait = "s_waitcnt vmcnt(%d)" % ((depth - 1) * copies)
        at = body.rindex(wait)
        one_more = body[:at] + wait.replace("(%d)" % ((depth - 1) * copies), "(%d)" % ((depth - 1) * copies + 1)) + body[at + len(wait):]
        assert _kinds(one_more, copies, depth) == {"reads a stage on its way"}
        # (the loop's wait for everything, which comes with the last stages)
        last = body.rindex("s_waitcnt vmcnt(0)", 0, at)
        assert "reads a stage on its way" in _kinds(body[:last] + "s_nop 0" + body[last + len("s_waitcnt vmcnt(0)"):], copies, depth)
        # (the operands' waits, behind the last of which the next turn's copies go)
        late = re.sub(r"s_waitcnt lgkmcnt\(\d+\)", "s_nop 0", body)
        assert "copies over what is being read" in _kinds(late, copies, depth)
    body = _body(listing, 1, 1, 8, 4, 1)
    wait = "s_waitcnt vmcnt(6)"
    assert "reads tokens on their way" in _kinds(body.replace(wait, "s_waitcnt vmcnt(7)", 1), 2, 4)
