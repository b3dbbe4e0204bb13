"""CPU: the ops without a gradient refuse forward mode, function transforms and
tracers, which do not see what a kernel computes."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx


def calls():
    """Name, call of one float (or of no) tensor, that tensor."""
    from asrback_amd.drafts import accept_drafts, commit_drafts, tree_attention, tree_masks
    from asrback_amd.linear4 import Linear4, linear4, pack4

    weight = pack4(torch.zeros(8, 64, dtype=torch.uint8), torch.ones(8, 2))
    ints = torch.zeros(2, 3, dtype=torch.int64)
    count = torch.zeros(2, dtype=torch.int64)
    q, k, draft = torch.zeros(2, 3, 4, 64), torch.zeros(2, 8, 2, 64), torch.zeros(2, 3, 2, 64)
    cache, drafts = torch.zeros(4, 2, 16, 2, 64), torch.zeros(4, 2, 3, 2, 64)
    return [
        ("linear4", lambda x: linear4(x, weight), torch.zeros(3, 64)),
        ("linear4", lambda x: linear4(torch.zeros(3, 64), weight, x), torch.zeros(8)),
        ("linear4", Linear4(weight), torch.zeros(3, 64)),
        ("tree_attention", lambda x: tree_attention(x, k, k, draft, draft, ints), q),
        ("tree_attention", lambda x: tree_attention(q, k, x, draft, draft, ints), k),
        ("tree_attention", lambda x: tree_attention(q, k, k, draft, x, ints), draft),
        ("commit_drafts", lambda x: commit_drafts(x, cache, drafts, drafts, ints, count, count), cache.clone()),
        ("commit_drafts", lambda x: commit_drafts(cache, cache.clone(), x, drafts, ints, count, count), drafts),
        ("tree_masks", tree_masks, ints),
        ("accept_drafts", lambda x: accept_drafts(x, ints, ints), ints),
    ]


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
@pytest.mark.parametrize("index", range(10))
def test_refused(index):
    name, call, x = calls()[index]
    with pytest.raises(RuntimeError, match="GPU only"):
        call(x)
    if x.is_floating_point():
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match=f"{name} has no gradient"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
            with torch.no_grad(), pytest.raises(RuntimeError, match=f"{name} has no gradient"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
            # Tensors without a tangent are ordinary ones.
            with pytest.raises(RuntimeError, match="GPU only"):
                call(x)
        with pytest.raises(RuntimeError, match=f"{name} takes no part"):
            torch.func.jvp(call, (x,), (x,))
    with torch.no_grad():
        with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
            torch.jit.trace(call, (x,))
        with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
            make_fx(call)(x)
