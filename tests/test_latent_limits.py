"""latent_append and latent_attention at the limits of a call: latents that are not finite far ahead of the new tokens."""
import math

import pytest
import torch

from latent_util import RANK, draw
from ktransformers_b200.operators.latent_attention import latent_attention

gpu = pytest.mark.gpu
FORMS = pytest.mark.parametrize("form", ["expanded", "absorbed"])


def call(d, form, **kw):
    return latent_attention(d.q, d.q_rot, d.kv, d.w, d.batch, d.cache, d.heads, d.nope, d.vdim, d.scale, form=form, **kw)


# ------------------------------------------------------------------------------------------------ latents that are not finite
@gpu
@FORMS
@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("page", [64, 48, 16])
def test_a_latent_that_is_not_finite_far_ahead(form, what, page):
    """One of a sequence's first latents reaches all of a portion behind 400 keys, whatever the pages, and no other sequence."""
    d = draw([(400, 70), (0, 90)], heads=2, page=page, seed=31)
    clean = call(d, form)
    d.kv[d.cache.page_table[0, 5 // page].long(), 5 % page, 300] = what
    got = call(d, form)
    assert not torch.isfinite(got[:70]).any() and torch.equal(got[70:], clean[70:])


@gpu
@FORMS
def test_a_latent_that_is_not_finite_beside_one_key_with_all_the_weight(form):
    """A part of the keys whose scores are far below those of another still hands on that one of its latents is infinite."""
    d = draw([(600, 3)], heads=2, seed=32)
    d.q_rot.zero_()
    d.q_rot[:, :, 0] = 64.0
    d.kv[..., RANK:] = 0
    d.kv[d.cache.page_table[0, 6].long(), 16, RANK] = 64.0      # 64 * 64 / sqrt(192) = 296 above the others
    assert torch.isfinite(call(d, form)).all()
    d.kv[d.cache.page_table[0, 0].long(), 5, 300] = math.inf
    assert not torch.isfinite(call(d, form)).any()
