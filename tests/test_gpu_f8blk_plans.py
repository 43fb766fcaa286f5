"""The gated front with 64 tokens a tile and all of K in one CTA: the plan of some tens of tokens through wide planes, whose meeting is one CTA's own.
Ragged tokens, a last channel tile that is not full and a last block of K that is not."""
import ctypes

import pytest
import torch

from test_gpu_f8blk import Operands, blocks, check_gate_up, guarded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,ff,k", [(41, 19472, 2064), (60, 19456, 5120), (64, 20816, 4112), (33, 22544, 2576)])
def test_gated_front_of_whole_tiles_of_64_tokens(pack, m, ff, k):
    plan = (ctypes.c_uint32 * 3)()
    assert pack._lib.pdk_f8blk_plan(2, k, ff, m, plan) == 0 and tuple(plan) == (1, 64, 1)
    o = Operands(m, ff, k, 960 + m, planes=2)
    hq, q_kept = guarded(m * ff, torch.uint8)
    hs, s_kept = guarded(m * blocks(ff), torch.float32)
    (g, gs, _), (u, us, _) = o.w
    kept = []
    for _ in range(2):                                        # and the same bits again
        pack.call("pdk_f8blk_gate_up", g, gs, u, us, o.xq, o.xs, hq, hs, k, ff, m)
        assert pack.device_error() == 0 and q_kept() and s_kept()
        kept.append((hq.clone(), hs.clone()))
    assert torch.equal(kept[0][0], kept[1][0]) and torch.equal(kept[0][1], kept[1][1])
    check_gate_up(o, hq, hs)
