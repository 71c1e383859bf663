"""A prompt prefix kept in 4 bits, rebuilt for another prompt."""

import warnings

import pytest
import torch

from tfimage import kv4, mmdit

pytestmark = pytest.mark.gpu


def test_a_rebuilt_prefix_warns_of_values_past_its_scales(dev):
    cfg = mmdit.DitConfig(layers=2, dim=512, heads=4, mlp=1024)
    m = mmdit.SynthMMDiT(cfg, device="cuda", seed=3)
    g = torch.Generator().manual_seed(4)
    ctx = torch.randn((1, 70, cfg.txt_dim), generator=g).cuda()
    prefix = m.build_prefix(ctx, cache="nvfp4")
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        m.build_prefix(ctx, into=prefix, cache="nvfp4")       # its own prompt, with room to spare
    old = prefix.caches[1]
    small = kv4.Kv4Cache(old.k_codes, old.k_sf, old.v_codes, old.v_sf, old.k_global, old.v_global / (2 * mmdit.CACHE_MARGIN))
    prefix.caches[1] = small                                  # holds half of this prompt's largest value
    with pytest.warns(UserWarning, match=r"2\.0\d? times .* saturates"):
        assert m.build_prefix(ctx, into=prefix, cache="nvfp4") is prefix
    rows = torch.empty((2, 70, cfg.heads, cfg.head_dim), dtype=torch.bfloat16, device=dev)
    kv4.read(small, prefix.table, torch.zeros_like(prefix.lengths), rows[0], rows[1])
    top = 2688 * small.v_global
    assert abs(float(rows[1].abs().max()) / top - 1) <= 2.0 ** -8          # saturated, at half a step of bf16
