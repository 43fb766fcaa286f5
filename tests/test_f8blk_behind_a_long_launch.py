"""Block-scaled e4m3 products behind a launch that takes longer than their own waits may: programmatic dependents are resident while the launch
before them still runs, so a limit that starts then would run out although nothing is wrong."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paddock_b200", "csrc")


@pytest.mark.parametrize("name,roles", [("f8blk_split.cu", 3), ("f8blk_wide.cu", 4)])
def test_no_limit_starts_before_the_launch_in_front_has_ended(name, roles):
    """Each role waits for the launch in front before its first bounded wait."""
    text = open(os.path.join(CSRC, name)).read()
    body = text[re.search(r"^f8blk_\w+_kernel\(", text, re.M).start():]
    parts = [re.sub(r"//[^\n]*", "", p) for p in re.split(r"// -{20,} ", body[:body.index("\n}\n")])[1:]]     # a line of dashes heads each role
    assert len(parts) == roles
    for p in parts:
        assert "pdk_pdl_wait();" in p and p.index("pdk_pdl_wait();") < p.index("wait_soon("), p[:300]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(5, 272, 2048), (1000, 2304, 1024)])
def test_a_product_behind_a_wait_of_more_than_a_second(pack, m, n, k):
    """In front: the pack's wait for a flag that nothing sets, given up after 1.5 s, which lets its dependents in at once."""
    import torch

    from test_gpu_f8blk import Operands
    o = Operands(m, n, k, 990, planes=2)
    (g, gs, _), (u, us, _) = o.w
    flags = torch.zeros(16, dtype=torch.int32, device="cuda")
    assert pack.device_error() == 0
    outs = []
    for late in (False, True):
        y, hq, hs = torch.zeros(m, n, device="cuda"), torch.zeros(m, n, dtype=torch.uint8, device="cuda"), torch.zeros(m, -(-n // 128), device="cuda")
        torch.cuda.synchronize()
        for name, args in (("pdk_f8blk_gemm", (g, gs, o.xq, o.xs, y, k, n, m)), ("pdk_f8blk_gate_up", (g, gs, u, us, o.xq, o.xs, hq, hs, k, n, m))):
            if late:
                pack.call("pdk_peer_flags_wait", flags, 1, 1, 1500000)
            pack.call(name, *args)
        assert pack.device_error() == (0x16 << 8 if late else 0)          # rank 0 is late, and nothing else
        outs.append((y, hq, hs))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
