"""CPU tests of what a delta-net layer and the copies of pages refuse before anything is launched, and of what they take."""
import numpy as np
import pytest
import torch

from saber_engine_amd import gdn, iu8
from tests.test_attn_host import cache, refused
from tests.test_gdn_host import P, built, ctx  # noqa: F401


class Calls:
    """A context that notes what it is asked for."""

    def __init__(self):
        self.names = []

    def __getattr__(self, name):
        return lambda *a, **k: self.names.append(name)


def test_counts_of_accepted_rows_that_do_not_fit():
    c, s = Calls(), gdn.GdnState(3, 2, 8, device="cpu")
    n = gdn.GdnLayerIU8(c, s, 3, 256)
    bf = dict(dtype=torch.bfloat16)
    n.set_weights(*(None,) * 6, conv=torch.ones(s.channels, 4, **bf), a_log=torch.ones(8), dt_bias=torch.ones(8), norm=torch.ones(128, **bf), had_t=torch.ones(1024))
    for bad in (torch.zeros(2, dtype=torch.int32), torch.zeros(3), torch.zeros(3, dtype=torch.int64), torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(iu8.IU8Error, match="kept"):
            n.accept(bad)
        with pytest.raises(iu8.IU8Error, match="kept"):
            n._core(bad, n.core, 0)
    with pytest.raises((iu8.IU8Error, AttributeError)):
        n.accept(np.zeros(3, np.int32))
    assert not c.names
    n.accept(torch.zeros(3, dtype=torch.int32))
    assert c.names == ["gdn_conv", "gdn"]


@pytest.mark.parametrize("kv_heads", [1, 3, 5, 7, 32767])
def test_pages_of_any_count_of_heads_may_be_copied(ctx, kv_heads):  # noqa: F811
    """No query heads stand beside them: what is refused is only that the context is not open."""
    refused(lambda: ctx.kv_copy(cache(kv_heads=kv_heads), P, P, 3), iu8.E_ARG, "null argument")


@pytest.mark.parametrize("kv_heads", [0, 32768, (1 << 32) - 1])
def test_pages_of_counts_that_no_cache_has_are_not(ctx, kv_heads):  # noqa: F811
    refused(lambda: ctx.kv_copy(cache(kv_heads=kv_heads), P, P, 3), iu8.E_RULE, "whole groups")


def test_a_layer_keeps_a_workspace_for_prompts_alone():
    s = gdn.GdnState(4, 2, 8, device="cpu")
    assert gdn.GdnLayerIU8(None, s, 4, 256)._gdn_ws is None and gdn.GdnLayerIU8(None, s, 40, 256, max_q=10)._gdn_ws is None
    assert gdn.GdnLayerIU8(None, s, 100, 256, max_q=90)._gdn_ws.numel() == (100 // 64 + 4) * (2 * 32768 + 8 * 19456)
