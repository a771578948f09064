"""Every wait of a kernel ends: what a wait that gave up leads to is read from the sources (a timeout
cannot be tried out without one)."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "dcu-video-dit-turbo_b200" / "csrc"
KERNELS = sorted(p.name for p in CSRC.glob("*.cu") if "mbar_wait" in p.read_text())


def source(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def blocks(text):
    """(header, start, end) of every brace block: the text between the statement before and its brace,
    and the positions of the braces."""
    out, stack = [], []
    for i, c in enumerate(text):
        if c == "{":
            # the header of `for (a; b; c) {` holds semicolons: look back to its keyword's parenthesis
            depth, j = 0, i - 1
            while j >= 0 and (depth > 0 or text[j] not in ";{}"):
                depth += (text[j] == ")") - (text[j] == "(")
                j -= 1
            stack.append((text[j + 1:i].strip(), i))
        elif c == "}":
            header, start = stack.pop()
            out.append((header, start, i))
    return out


def enclosing(all_blocks, at):
    """Blocks around a position, the innermost first."""
    return sorted((b for b in all_blocks if b[1] < at < b[2]), key=lambda b: b[2] - b[1])


def is_loop(header):
    return re.search(r"\b(for|while)\s*\(", header) is not None


@pytest.mark.parametrize("name", KERNELS)
def test_no_thread_leaves_a_loop_that_passes_a_named_barrier(name):
    """A named barrier has no limit: a thread that leaves such a loop on a timeout, while another
    warp's wait succeeded, leaves that one at the barrier for ever."""
    text = source(name)
    all_blocks = blocks(text)
    for m in re.finditer(r"bar\.sync 1", text):
        loops = [b for b in enclosing(all_blocks, m.start()) if is_loop(b[0])]
        for _, start, end in loops:
            body = list(text[start + 1:end])
            for header, s, e in all_blocks:                 # a nested loop's own break stays in it
                if start < s and e < end and is_loop(header):
                    body[s - start - 1:e - start] = " " * (e - s + 1)
            body = "".join(body)
            assert not re.search(r"\b(break|return)\b", body), (name, re.findall(r"[^\n]*\b(?:break|return)\b[^\n]*", body))


ONE_LANE = re.compile(r"\blane == 0\b|elect_one\(\) != 0|threadIdx\.x == ")
WARP_WIDE = re.compile(r"\b(?:mbar_wait_warp\(|wait_warp[(,)]|__all_sync\(|__any_sync\(|__shfl\w*_sync\(|__syncwarp\(|__reduce\w*_sync\(|tmem_(?:ld|st)_)")


def line_at(text, at):
    return text[text.rfind("\n", 0, at) + 1:text.find("\n", at)].strip()


@pytest.mark.parametrize("name", KERNELS + ["flash_common.cuh"])
def test_warps_leave_their_waits_together(name):
    """Lanes that wait each for themselves can disagree on a timeout.  Outside of a single lane's code, where
    warp-wide instructions follow, no lane leaves on its own answer: the wait is the whole warp's
    (mbar_wait_warp), or every lane goes on whatever its wait said until a vote."""
    text = source(name)
    all_blocks = blocks(text)
    for m in re.finditer(r"(?<!auto )\b(?:mbar_wait|wait)\(|if \(!ok\) (?:break|continue|return)", text):
        line = line_at(text, m.start())
        if re.match(r"auto wait(_warp)? = ", line):         # a kernel's own names for the two
            continue
        around = enclosing(all_blocks, m.start())
        if any(ONE_LANE.search(b[0]) for b in around):
            continue
        roles = [b for b in around if re.search(r"\bwarp (==|>=) ", b[0])]
        if roles and not WARP_WIDE.search(text[roles[0][1]:roles[0][2]]):
            continue                                        # the warp does not meet before the kernel's end
        if line.startswith("if (!ok)"):
            assert re.search(r"wait_warp\(|__all_sync\(", text[max(0, m.start() - 900):m.start()]), (name, line)
        else:
            assert re.match(r"if \(ok\b.*\) ok = (mbar_wait|wait)\(", line), (name, line)


@pytest.mark.parametrize("name", KERNELS + ["flash_common.cuh"])
def test_a_single_lane_makes_no_wait_of_a_warp(name):
    """A warp-wide instruction in one lane's code waits for lanes that never come."""
    text = source(name)
    all_blocks = blocks(text)
    for m in WARP_WIDE.finditer(text):
        line = line_at(text, m.start())
        assert not any(ONE_LANE.search(b[0]) for b in enclosing(all_blocks, m.start())), (name, line)
        assert not re.match(r"if \(.*(lane == 0|threadIdx\.x == )", line), (name, line)
