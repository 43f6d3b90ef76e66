"""How exactly the softmax weights of a shared prefix count, on prefixes of any length: as bf16 pairs, as the decode
kernel's do.

The rows of V are zero but for a few, of either sign, so that a weight's own rounding is not averaged away and the
output's rounding is small against it.  Tolerance, with share_j the weights and S = max_j scale log2(e) sum_d |q_d K_jd|
(at least 1): a score is off by at most 2^-16 S, a share by 2^-15 S of itself; a weight as a bf16 pair is off by at
most 2^-16 of itself; L / 16 additions of at most 2^-23 each; all relative to sum_j share_j |V_j|.  The output is
rounded to bf16: 2^-8 of it.  (Weights rounded to bf16 alone would be off by up to 2^-8.)
"""
import pytest
import torch

from test_shared_prefix_gpu import Case, DEV

pytestmark = pytest.mark.gpu


def few_rows(batch, prefix, seed):
    c = Case([batch], [prefix], [0] * batch, seed=seed, q_std=0.5)
    c.rows_k.mul_(0.25)
    c.rows_v.zero_()
    chosen = torch.randperm(prefix, generator=c.g, device=DEV)[:8]
    c.rows_v[chosen] = torch.randint(0, 2, (8, 8, 128), generator=c.g, device=DEV).bfloat16() * 2 - 1
    c.put()
    return c


@pytest.mark.parametrize("batch", [3, 32, 33, 64, 70])
@pytest.mark.parametrize("prefix", [600, 1023, 1024, 1100, 2500, 9000])
def test_weights_are_not_rounded_to_bf16(batch, prefix):
    c = few_rows(batch, prefix, seed=batch + prefix)
    out, lse = c.run()
    assert c.status == 0
    ref, size, ref_lse, _, slack = c.expect()
    tol = slack + 2.0 ** -16 + prefix / 16 * 2.0 ** -23
    off = (out.double() - ref).abs()
    bound = 2.0 ** -8 * ref.abs() + tol[..., None] * size
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-30)).max())
    c.check(out, lse)
