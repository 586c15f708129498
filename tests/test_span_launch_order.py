"""A kernel launched as a programmatic dependent one may end before the kernel
before it has, unless its threads wait for that one (griddepcontrol.wait).  What
the stream runs next is ordered behind the whole call only if no block can leave
without the wait: read off the kernels' source, as a run shows nothing but luck."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "vllm_b200/csrc"


def body(file, name):
    """The text between the braces of kernel `name`, without comments."""
    text = re.sub(r"//[^\n]*", "", (CSRC / file).read_text())
    at = text.index("{", text.index(")", text.index(f" {name}(")))
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[at + 1:i]
    raise AssertionError(name)


def blocks_left(text, at):
    """Starts of the brace blocks that are open at `at`."""
    stack = []
    for i in range(at):
        if text[i] == "{":
            stack.append(i)
        elif text[i] == "}":
            stack.pop()
    return stack


def exits_without_wait(text):
    """Returns of the kernel (not of its lambdas) that no wait precedes, in a block that is
    open at the return (or in the condition line before the block)."""
    waits = [(m.start(), blocks_left(text, m.start())) for m in re.finditer(r"griddepcontrol\.wait", text)]
    bad = []
    for m in re.finditer(r"\breturn\b", text):
        open_blocks = blocks_left(text, m.start())
        if any(re.search(r"\][^;{}]*$", text[max(0, b - 80):b]) and "[&]" in text[max(0, b - 80):b]
               for b in open_blocks):
            continue  # a lambda's
        if not any(at < m.start() and blocks == open_blocks[:len(blocks)] for at, blocks in waits):
            bad.append(text[:m.start()].count("\n"))
    return bad


@pytest.mark.parametrize("name", ["prefix_merge_kernel", "span_decode_kernel"])
def test_no_exit_without_the_wait(name):
    text = body("tvp_span_decode.cu", name)
    assert text.count("griddepcontrol.wait") >= 2
    if name == "span_decode_kernel":
        # SHARED is launched behind the kernel before it as a whole: its exits need no wait
        assert re.search(r"cfg\.numAttrs = SHARED \? 0 : 1;", (CSRC / "tvp_span_decode.cu").read_text())
        text = re.sub(r"if \(SHARED && [^{]*\{.*?\n  \}", "", text, count=1, flags=re.S)
        text = text.replace("if (!SHARED) asm", "asm")
    assert exits_without_wait(text) == []


def test_the_tiles_last_block_waits_whatever_the_groups_are():
    """The merge kernel waits for the tile grid alone, whose last block stands for the decode kernel."""
    text = body("tvp_span_tiles.cu", "span_tiles_kernel")
    last = text.index("blockIdx.x == gridDim.x - 1")
    assert "griddepcontrol.wait" in text[last:text.index("return", last)]
    assert last < re.search(r"groups_(in_order|usable)\(", text).start()
    early = text[:last]
    assert early.count("return") == 1 and early.index("griddepcontrol.wait") < early.index("return")


def test_the_search_sees_an_exit_without_wait():
    text = 'if (a) { return; } asm("griddepcontrol.wait;"); if (b) return; auto f = [&](int i) { return i; };'
    assert len(exits_without_wait(text)) == 1
    assert exits_without_wait('if (a) { asm("griddepcontrol.wait;"); return; } asm("griddepcontrol.wait;");') == []
