"""What the oracle takes for a 4-bit cache's keys and values (CPU)."""
import numpy as np
import pytest
import torch

from kv4_util import quantised


@pytest.mark.parametrize("sel,dim", [(0, 3), (1, 40)], ids=["key", "value"])
def test_the_oracle_refuses_a_cache_that_is_a_step_off(O, sel, dim):
    """The oracle takes the stored form of its own keys and values, and not one that is 1.3 steps from it."""
    ctx, kv, d, n = 32, 2, 64, 6
    cfg = O.config(hidden=256, layers=4, vocab=4096, q_heads=4, kv_heads=kv, head_dim=d, key_heads=2, value_heads=4,
                   key_dim=64, value_dim=64, experts=16, top=2, intermediate=128, shared=128, context=ctx, rope_dims=16,
                   theta=1e7)
    model = O.Model(cfg, 5)
    toks = np.arange(n, dtype=np.uint32) * 7
    logits, state, _, route = model.forward(toks, 0)
    own = state[-2 * kv * ctx * d:].reshape(2, kv, ctx, d)[:, :, :n].astype(np.float64)
    held = quantised(torch.from_numpy(own.copy()))[0].float().numpy()
    got = model.forward(toks, 0, cached_kv=held[None])[0]
    assert got.shape == logits.shape and np.isfinite(got).all() and not np.array_equal(got, logits)
    step = (own[sel, 1, 4].max() - own[sel, 1, 4].min()) / 15
    held[sel, 1, 4, dim] = own[sel, 1, 4, dim] + 1.3 * step
    with pytest.raises(Exception, match="not near"):
        model.forward(toks, 0, cached_kv=held[None])
