"""What orders the scale warps' stores in front of the product warps' loads in the wide block-scaled e4m3 kernel, read off its source: the product
warps wait for `done` alone, so a thread that has waited for `full`, on which the scale warps arrive behind their stores, has to arrive on `done`
itself.  The tensor core's own arrival (tcgen05.commit) orders what the tensor core did."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paddock_b200", "csrc", "f8blk_wide.cu")


def test_the_issuer_hands_the_scales_on():
    text = re.sub(r"//[^\n]*", "", open(SOURCE).read())
    # done: the tensor core's arrival and the issuer's
    assert re.search(r"mbar_init\(&sh->done\[s\], 2u?\);", text)
    issuer = text[text.index("warp <= C::kIssuers"):]
    issuer = issuer[:issuer.index("} else {")]
    waited = issuer.index("wait_soon(&sh->full[stage]")
    assert waited < issuer.index("mbar_arrive_elect(&sh->done[stage])") and waited < issuer.index("mma_commit_elect(&sh->done[stage])")
    # full: behind the stores of every lane of a scale warp
    stored = text.index("slot[h][row0")
    assert stored < text.index("__syncwarp();", stored) < text.index("if (lane == 0u) tc5::mbar_arrive(&sh->full[stage]);", stored)
    # and the product's lanes each wait for done before they load
    product = text[text.index("for (uint32_t tile = blockIdx.x; tile < n_tiles; tile += gridDim.x)"):]
    assert product.index("wait_soon(&sh->done[stage]") < product.index("sh->scale[block % kSlots]")
