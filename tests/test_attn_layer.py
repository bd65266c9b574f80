"""CPU tests of what the attention layer and its cache refuse (saber_engine_amd/attn.py): tensors that a kernel would read past."""
import pytest
import torch

from saber_engine_amd import attn, iu8


def test_caches_of_scales_that_do_not_fit():
    f = lambda *n, **kw: torch.ones(*n, **kw)  # noqa: E731
    make = lambda **kw: attn.PagedKvCache(3, 2, 64, 200, kind=iu8.KV_E4M3, device="cpu", **kw)  # noqa: E731
    assert make(k_scale=f(2), v_scale=f(2)).desc.k_scale
    for bad in (dict(), dict(k_scale=f(2)), dict(k_scale=f(1), v_scale=f(2)), dict(k_scale=f(2), v_scale=f(2, dtype=torch.float64)), dict(k_scale=f(4)[::2], v_scale=f(2)),
                dict(k_scale=f(2, device="meta"), v_scale=f(2))):
        with pytest.raises(iu8.IU8Error, match="k_scale") as e:
            make(**bad)
        assert e.value.code == iu8.E_ARG


def test_layers_of_tensors_that_do_not_fit():
    c = attn.PagedKvCache(3, 2, 64, 200, device="cpu")
    f64 = dict(dtype=torch.float64)
    for bad in (torch.ones(8), torch.ones(64, **f64), torch.ones(16, **f64)[::2], torch.ones(8, device="meta", **f64)):
        with pytest.raises(iu8.IU8Error, match="inv_freq"):
            attn.AttnLayerIU8(None, c, 3, 4, 256, inv_freq=bad)
    n = attn.AttnLayerIU8(None, c, 3, 4, 256, inv_freq=torch.ones(8, **f64))
    had = torch.ones(256)
    for bad, words in ((dict(had_t=torch.ones(128)), "had_t"), (dict(had_t=had.double()), "had_t"), (dict(had_t=had, q_norm=torch.ones(64)), "head norms"),
                       (dict(had_t=had, k_norm=torch.ones(32, dtype=torch.bfloat16)), "head norms")):
        with pytest.raises(iu8.IU8Error, match=words):
            n.set_weights(None, None, None, None, **bad)
    for dtype in (torch.bfloat16, torch.int16):
        n.set_weights(None, None, None, None, had_t=had, q_norm=torch.ones(64, dtype=dtype), k_norm=None)
    for bad in (torch.zeros((3, 256)), torch.zeros((256, 3), dtype=torch.int16).t(), torch.zeros((3, 256), dtype=torch.int16, device="meta")):
        with pytest.raises(iu8.IU8Error, match="in one piece"):
            n.forward(bad)
