"""Bounded waits of the block-scaled e4m3 kernels: that each wait's result decides what follows, read off the sources, and on a GPU the
path of a wait that runs out, on barriers that nothing arrives on."""
import os
import re
import time

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paddock_b200", "csrc")


def code(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def call_at(text, start):
    """The call that starts at `start`, with its arguments."""
    depth, i = 0, text.index("(", start)
    while True:
        depth += {"(": 1, ")": -1}.get(text[i], 0)
        i += 1
        if depth == 0:
            return text[start:i]


def unused_waits(text):
    """Lines of waits whose result is not an operand of a vote of the whole warp that `ok` takes, or whose `ok` is not looked at next."""
    bad = []
    votes = [(m.start(), call_at(text, m.end() - len("__all_sync("))) for m in re.finditer(r"ok = __all_sync\(", text)]
    for m in re.finditer(r"\bwait_soon\(", text):
        line = text.count("\n", 0, m.start()) + 1
        named = re.search(r"const bool (\w+) = (?:f8blk::)?$", text[:m.start()])
        inside = [v for at, v in votes if at < m.start() < at + len("ok = ") + len(v)]
        behind = [(at, v) for at, v in votes if at > m.start()][:1]
        vote = inside[:1] or ([behind[0][1]] if named and behind and re.search(rf"&& {named.group(1)}\b|\b{named.group(1)} &&", behind[0][1]) else [])
        if not vote:
            bad.append(line)
            continue
        at = text.index(vote[0], m.start() if not inside else text.rindex("ok = __all_sync(", 0, m.start()))
        if not text[at + len(vote[0]):].lstrip("; \n").startswith("if (!ok) break;"):
            bad.append(line)
    return bad


@pytest.mark.parametrize("name,waits", [("f8blk_split.cu", 4), ("f8blk_wide.cu", 5)])
def test_every_wait_decides_whether_its_loop_goes_on(name, waits):
    text = code(name)
    assert len(re.findall(r"\bwait_soon\(", text)) == waits and not unused_waits(text)


def test_a_wait_that_is_not_looked_at_is_found():
    """The check itself, on sources with one wait's result dropped."""
    for name, was, now in (("f8blk_wide.cu", " && empty);", ");"), ("f8blk_wide.cu", "if (!ok) break;\n                tc5::fence_after_sync();", ""),
                           ("f8blk_split.cu", "if (!ok) break;\n            tc5::fence_after_sync();", ""),
                           ("f8blk_split.cu", "ok = __all_sync(0xffffffffu, wait_soon(&sh->empty", "(void)__all_sync(0xffffffffu, wait_soon(&sh->empty")):
        text = code(name)
        assert was in text
        assert unused_waits(text.replace(was, now, 1)), (name, was)


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_given_up_and_reported(pack):
    import torch
    scratch = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert pack.device_error() == 0
    t0 = time.perf_counter()
    assert pack.status("pdk_selftest_f8blk_wait", 2000, scratch) == 0
    took = time.perf_counter() - t0
    assert 0.001 < took < 0.5                      # the second warp's own limit is a second
    assert scratch.tolist() == [1, 1]
    assert pack.device_error() == (5 << 8 | 8) and pack.device_error() == 0
    assert float((torch.ones(8, device="cuda") * 2).sum()) == 16.0


def test_selftest_refusals():
    import ctypes as C

    import paddock_b200 as pb
    fn = C.CDLL(pb.lib_path()).pdk_selftest_f8blk_wait
    fn.argtypes, fn.restype = [C.c_uint32, C.c_void_p, C.c_void_p], C.c_int
    for budget, scratch in ((0, 0x7000_0000_0000), (100001, 0x7000_0000_0000), (1000, None), (1000, 0x7000_0000_0002)):
        assert fn(budget, scratch, None) == 1
