"""Refusals of the normed and the plain position rotation that need no GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from oscar_amd.kernels import rotary


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("dual", ["query", "key", "query_weight", "key_weight", None])
def test_forward_mode_is_refused(dual, given):
    """A tangent would be lost without a word; tensors without one are taken inside a level too."""
    args = {"query": torch.ones(3, 2, 64), "key": torch.ones(3, 1, 64), "query_weight": torch.ones(64),
            "key_weight": torch.ones(64)}
    out = {"query_out": torch.empty(3, 2, 64), "key_out": torch.empty(3, 1, 64)} if given else {}
    turn, pos = rotary.Rotary(rotary.rotary_table(8, 32)), torch.arange(3)
    with forward_ad.dual_level():
        if dual:
            args[dual] = forward_ad.make_dual(args[dual], torch.ones_like(args[dual]))
        match = "tangents" if dual else "device tensors"
        with pytest.raises(ValueError, match=match):
            rotary.norm_rotate(*args.values(), pos, turn, **out)
        with pytest.raises(ValueError, match=match if dual in ("query", "key") else "device tensors"):
            rotary.rotate(args["query"], args["key"], pos, turn, **out)
    with pytest.raises(ValueError, match="device tensors"):
        rotary.rotate(torch.ones(3, 2, 64), None, pos, turn)
