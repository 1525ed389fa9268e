"""CPU: a model whose projections the 8-bit products do not take is refused when it is
built, not at its first step."""
from dataclasses import replace

import pytest
import torch

from test_decode_step import TINY, DenseCache
from zoomkv_revision_amd import decode_step as ds
from zoomkv_revision_amd import fp8


@pytest.mark.parametrize("changed,name", [(dict(ffn=fp8.MAX_K + 1), "ffn"), (dict(hidden=fp8.MAX_K + 128), "hidden"),
                                          (dict(heads=130, kv_heads=2), "heads")])
def test_projections_too_wide_for_8_bits(changed, name):
    """(The check stands before the first use of the device.)"""
    with pytest.raises(ValueError, match=f"at most 16384 channels; got {name}"):
        ds.RandomQwen3(replace(TINY, **changed), "cuda", weights="fp8")


def test_the_torch_ops_take_any_width():
    geo = replace(TINY, layers=1, ffn=fp8.MAX_K + 128)
    m = ds.RandomQwen3(geo, "cpu", seed=1, max_position=64, weights="fp8")
    assert torch.isfinite(m.decode_step(torch.tensor([1]), DenseCache(1, 1, geo.kv_heads))).all()
