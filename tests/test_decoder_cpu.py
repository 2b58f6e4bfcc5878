"""What a decoder refuses, without a GPU."""
from types import SimpleNamespace

import pytest
import torch

from sketchpad_b200.decoder import Decoder, DecoderConfig


def test_layers_and_caches():
    c = DecoderConfig(hidden=64, intermediate=64, heads=1, kv_heads=1, head_dim=16,
                      max_positions=8)
    norm, layer = torch.ones(64), object()
    cache = lambda pages, size: SimpleNamespace(pages=pages, page_size=size)  # noqa: E731
    assert len(Decoder(c, [layer] * 2, norm, [cache(4, 8)] * 2).layers) == 2
    for layers, caches in (([], []), ([layer], []), ([layer], [cache(4, 8)] * 2),
                           ([layer] * 2, [cache(4, 8), cache(4, 16)]),
                           ([layer] * 2, [cache(4, 8), cache(5, 8)])):
        with pytest.raises(ValueError):
            Decoder(c, layers, norm, caches)
