"""What the source of the paged tree attention has to keep, read from its text (no GPU needed)."""

import os
import re

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fa4-cp_b200", "csrc",
                   "attn_paged_tree.cu")
COLLECTIVE = re.compile(r"\btmem_(?:ld|st|wait_ld|wait_st)\w*\(")
PER_LANE = {"valid", "lane", "t", "key", "row", "node", "head", "tok"}


def _close(text, at, pair):
    """Index behind the bracket that closes the one at `at`."""
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == pair[0]) - (text[i] == pair[1])
        if depth == 0:
            return i + 1
    raise ValueError("unbalanced")


def _loops(text):
    for m in re.finditer(r"\b(?:for|while) \(", text):
        end = _close(text, m.end() - 1, "()")
        body = re.match(r"\s*\{", text[end:])
        if body:
            start = end + body.end() - 1
            yield text[start:_close(text, start, "{}")]


def _jumps(body):
    """(condition, jump) of every `if (...) continue;` and `if (...) { ...; break; }`."""
    for m in re.finditer(r"\bif \(", body):
        end = _close(body, m.end() - 1, "()")
        jump = re.match(r"\s*(?:\{[^{}]*)?\b(continue|break)\s*;", body[end:])
        if jump:
            yield body[m.end():end - 1], jump.group(1)


def test_no_lane_leaves_a_loop_of_warp_collective_accesses():
    """tcgen05.ld and .st are .sync.aligned: all lanes of a warp execute each of them together.  So
    no loop that holds one may be left or gone on with under a condition that differs by lane."""
    text = re.sub(r"//[^\n]*", "", open(SRC).read())
    loops = [b for b in _loops(text) if COLLECTIVE.search(b)]
    assert len(loops) >= 3  # the items, their tiles, the columns of a result
    for body in loops:
        for cond, jump in _jumps(body):
            names = set(re.findall(r"[A-Za-z_]\w*", cond))
            assert not names & PER_LANE, f"`if ({cond}) {jump}` parts the lanes of a warp"


def test_the_grid_is_of_the_device_of_the_call():
    """The number of SMs is asked of the device that the call runs on, not kept from the first one."""
    text = re.sub(r"//[^\n]*", "", open(SRC).read())
    at = text.index("int launch_tree(")
    body = text[text.index("{", at):_close(text, text.index("{", at), "{}")]
    assert "cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)" in body
    assert text.count("MultiProcessorCount") == 1
