"""RecurrentLayer.repack() writes into the words that captured calls hold (CPU only)."""
import numpy as np
import pytest
import torch

from reimagined_amd import ops
from reimagined_amd.layers import BitLinear, RecurrentLayer


def test_repack_stays_in_place():
    rng = np.random.default_rng(1)
    n = lambda *s: rng.standard_normal(s).astype(np.float32)
    layer = RecurrentLayer(dict(w_in=n(96, 48), w_out=n(48, 32), lam=n(32)), "cpu")
    held = [(p.packed, p.packed.data_ptr()) for p in (layer.in_proj, layer.out_proj)]
    layer.w_in.neg_()
    layer.w_out.mul_(3.0).add_(0.2)
    layer.repack()
    for (words, at), p, scale, w in zip(held, (layer.in_proj, layer.out_proj), (layer.in_scale, layer.out_scale),
                                        (layer.w_in, layer.w_out)):
        packed, ws = ops.pack_ternary(w)
        assert p.packed.data_ptr() == at == words.data_ptr()
        assert np.array_equal(words.numpy().view(np.uint32), packed)
        assert p.weight_scale == ws and scale.tolist() == [ws]


def test_load_refuses_another_shape():
    lin = BitLinear(np.ones((4, 16), np.float32), "cpu")
    with pytest.raises(ValueError, match="weights must be"):
        lin.load(np.ones((16, 4), np.float32))
