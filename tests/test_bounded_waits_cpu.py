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
