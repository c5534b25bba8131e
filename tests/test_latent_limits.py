"""latent_append, latent_attention and the layer on them at the limits of a call: latents that are not finite far ahead of the new tokens, positions behind the page table, portions and pages that are not there, layers that
were built without memory or are captured before their first call, configurations that come back from a file."""
import ctypes as C
import math
from types import SimpleNamespace

import pytest
import torch

from latent_util import HALF, RANK, ROT, draw, near
from test_latent_portions import YARN, Exact, layer
from ktransformers_b200 import native
from ktransformers_b200.models.modeling_deepseek_v3 import DeepseekV3Attention, DeepseekV3Config, DeepseekV3RotaryEmbedding, DeepseekV3YarnRotaryEmbedding, yarn_get_mscale, yarn_inv_freq
from ktransformers_b200.operators.attention import KDeepseekV2Attention
from ktransformers_b200.operators.latent_attention import LatentRotation, latent_append, latent_attention

gpu = pytest.mark.gpu
FORMS = pytest.mark.parametrize("form", ["expanded", "absorbed"])


def call(d, form, **kw):
    return latent_attention(d.q, d.q_rot, d.kv, d.w, d.batch, d.cache, d.heads, d.nope, d.vdim, d.scale, form=form, **kw)


def definition(d):
    """(out, bound) in 64 bits with latent_util.attention's bound, over the keys that are there: up to the token's position, in a column of the page table, in a page of the pool.  A row without any is zero"""
    outs, bounds, at = [], [], 0
    w = d.w.view(d.heads, d.nope + d.vdim, RANK).double()
    room = d.cache.page_table.shape[1] * d.page
    for i, (b, n) in enumerate(d.lens):
        key = torch.arange(min(b + n, room), device=d.kv.device)
        page = d.cache.page_table[i].long()[key // d.page]
        there = (page >= 0) & (page < d.kv.shape[0])
        rows = d.kv[page.clamp(0, d.kv.shape[0] - 1), key % d.page].double().masked_fill(~there[:, None], 0.0)
        lat, rot = rows[:, :RANK], rows[:, RANK:]
        q = d.q.view(-1, d.heads, d.nope + ROT)[at:at + n, :, :d.nope].double()
        see = (key[None, :] <= torch.arange(b, b + n, device=rows.device)[:, None]) & there[None, :]
        some = see.any(1, keepdim=True)
        o, e = [], []
        for h in range(d.heads):
            wk, wv = w[h, :d.nope], w[h, d.nope:]
            s = (q[:, h] @ wk @ lat.t() + d.q_rot[at:at + n, h].double() @ rot.t()) * d.scale
            p = torch.where(some, torch.softmax(s.masked_fill(~see, -math.inf), 1), torch.zeros_like(s))
            k, v = lat @ wk.t(), lat @ wv.t()
            off = torch.maximum(q[:, h].abs() @ k.abs().t(), (q[:, h] @ wk).abs() @ lat.abs().t()).masked_fill(~see, 0.0).amax(1) * (HALF * d.scale)
            mass = torch.maximum(p @ v.abs(), (p @ lat).abs() @ wv.abs().t() + (p @ lat.abs()) @ wv.abs().t() * HALF)
            o.append(p @ v)
            e.append(mass * (torch.expm1(2 * off)[:, None] * (1 + 4 * HALF) + 4 * HALF) + o[-1].abs() * HALF)
        outs.append(torch.stack(o, 1).flatten(1))
        bounds.append(torch.stack(e, 1).flatten(1))
        at += n
    return torch.cat(outs), torch.cat(bounds)


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


# ------------------------------------------------------------------------------------------------ positions behind the page table
def short_table(page, before, tokens, shift, heads=2, seed=0, **kw):
    """A portion whose positions go on behind the last column of its page table"""
    d = draw([(before, tokens)], heads=heads, page=page, seed=seed, **kw)
    columns = (before + tokens + page - 1) // page
    d.cache = SimpleNamespace(page_table=d.cache.page_table[:, :columns].contiguous(), max_pages_per_seq=columns, page_size=page)
    d.batch.pos += shift
    d.lens = [(before + shift, tokens)]
    d.batch.max_kv = before + shift + tokens
    return d


SHORT = pytest.mark.parametrize("page,before,tokens,shift", [
    (16, 34, 30, 16),        # 64 positions, the portion at 50 .. 79
    (64, 290, 30, 20),       # 320 positions, two and a half key tiles; 310 .. 339
    (64, 98, 30, 200),       # 128 positions, all tokens behind them
    (48, 250, 134, 10),      # 384 positions, three key tiles; 260 .. 393
    (64, 500, 140, 1000),    # 640 positions, all tokens far behind them
    (16, 79, 1, 1),          # 80 positions, a decoded token at the first that is not there
])


@gpu
@FORMS
@SHORT
def test_attention_behind_the_page_table(form, page, before, tokens, shift):
    """Tokens at positions that have no column see the keys that have one, as the one-token step of the layer does."""
    d = short_table(page, before, tokens, shift, seed=41)
    want, bound = definition(d)
    near(call(d, form), want, bound)
    d.batch.max_kv = 4 * d.batch.max_kv
    near(call(d, form), want, bound)


def append(d, rot):
    kva = torch.randn((d.batch.n_tokens, RANK + ROT), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).bfloat16()
    weight = torch.linspace(0.5, 1.5, RANK, device="cuda").bfloat16()
    return latent_append(d.q, kva, weight, 1e-6, d.batch, d.cache, d.kv, d.heads, d.nope, rot=rot)


@gpu
@SHORT
def test_append_behind_the_page_table(page, before, tokens, shift):
    """Tokens at positions that have no column are turned and written nowhere."""
    d = short_table(page, before, tokens, shift, seed=42)
    rot = LatentRotation(10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64).cuda())
    start, room = d.kv.clone(), d.cache.page_table.shape[1] * page
    got = append(d, rot)
    after, d.kv = d.kv, start.clone()
    stay = max(0, room - before - shift)      # tokens that have a column
    d.batch.seqs[1, 0] = stay
    first = append(d, rot)
    assert torch.equal(after.view(torch.int16), d.kv.view(torch.int16)) and torch.equal(got[:stay], first[:stay])
    key = torch.arange(before + shift, before + shift + stay, device="cuda")
    at = d.cache.page_table[0].long()[key // page], key % page
    start[at] = after[at]
    assert torch.equal(after.view(torch.int16), start.view(torch.int16))


@gpu
def test_append_of_a_portion_longer_than_its_table():
    """More tokens than the table has positions: the first ones are written, each once, whatever the order of the warps."""
    d = draw([(0, 1000)], heads=2, page=16, seed=43)
    rot = LatentRotation(10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64).cuda())
    whole, start = d.kv.clone(), d.kv.clone()
    d.kv = whole
    append(d, rot)
    table = d.cache.page_table
    d.cache, d.kv = SimpleNamespace(page_table=table[:, :5].contiguous(), max_pages_per_seq=5, page_size=16), start.clone()
    append(d, rot)
    used = table[0, :5].long()
    start[used] = whole[used]
    assert torch.equal(d.kv.view(torch.int16), start.view(torch.int16))


# ------------------------------------------------------------------------------------------------ portions that are not there
@gpu
@FORMS
@pytest.mark.parametrize("first,count", [(5, 100), (5, 36), (-1, 20), (2000000000, 2000000000)])
def test_portions_that_reach_past_the_call(form, first, count):
    """A portion with tokens that the call does not have is not there: its rows stay, and nothing is appended for it."""
    d = draw([(90, 5), (10, 35)], heads=3, seed=51)
    want, bound = definition(d)
    d.batch.seqs[:, 1] = torch.tensor([first, count], dtype=torch.int32, device="cuda")
    got = call(d, form, out=torch.full((40, 384), 7.0, dtype=torch.bfloat16, device="cuda"))
    near(got[:5], want[:5], bound[:5])
    assert (got[5:] == 7).all()
    start = d.kv.clone()
    append(d, None)
    page, row = d.cache.page_table[0, 1].long(), slice(90 - 64, 95 - 64)
    assert not torch.equal(d.kv[page, row], start[page, row])
    start[page, row] = d.kv[page, row]
    assert torch.equal(d.kv.view(torch.int16), start.view(torch.int16))


@gpu
@FORMS
def test_portions_whose_first_token_is_not_there(form):
    """The first token's slot and position are the portion's: where they are not there, none of its rows is written, in either form."""
    d = draw([(90, 5), (10, 35)], heads=3, seed=52)
    want, bound = definition(d)
    for name, what in (("slot", 9), ("pos", -1), ("pos", 0x7ffffff0)):
        held = getattr(d.batch, name)[5].clone()
        getattr(d.batch, name)[5] = what
        got = call(d, form, out=torch.full((40, 384), 7.0, dtype=torch.bfloat16, device="cuda"))
        near(got[:5], want[:5], bound[:5])
        assert (got[5:] == 7).all()
        getattr(d.batch, name)[5] = held
    near(call(d, form), want, bound)


# ------------------------------------------------------------------------------------------------ pages that are not there
@gpu
@FORMS
@pytest.mark.parametrize("lens,heads,page,gone", [
    ([(400, 70), (30, 60)], 2, 64, [(0, 0), (0, 3), (1, 1)]),
    ([(400, 70), (30, 60)], 2, 16, [(0, 0), (0, 7), (0, 8), (0, 26), (1, 2)]),
    ([(400, 70), (30, 60)], 3, 48, [(0, 2), (0, 8), (1, 0)]),
    ([(1000, 3), (0, 1)], 16, 32, [(0, i) for i in range(8, 20)] + [(0, 31)]),
    ([(4000, 5)], 128, 64, [(0, i) for i in range(0, 40)]),      # whole runs of tiles without a key
    ([(3000, 2)], 4, 64, [(0, i) for i in range(47)]),            # no key at all, in several parts
    ([(0, 5), (100, 20)], 2, 64, [(0, 0)]),                       # no key at all
    ([(0, 5), (100, 20)], 2, 16, [(0, 0)]),
    ([(5000, 70)], 4, 64, [(0, i) for i in range(0, 79)]),        # parts of the keys, most of them empty
    ([(200, 5), (700, 9)], 4, 256, [(0, 0), (1, 1)]),             # pages of several tiles, of which the first tokens see some whole
])
def test_keys_of_pages_that_are_not_there(form, lens, heads, page, gone):
    """Keys in pages outside the pool are not seen; a row that sees no key becomes zero."""
    d = draw(lens, heads=heads, page=page, seed=61)
    for k, (i, column) in enumerate(gone):
        d.cache.page_table[i, column] = -1 if k % 2 else d.kv.shape[0] + k
    want, bound = definition(d)
    got = call(d, form)
    empty = (bound == 0).all(1)
    assert (got[empty] == 0).all()
    near(got[~empty], want[~empty], bound[~empty])


# ------------------------------------------------------------------------------------------------ calls without tokens, and very many sequences
def test_calls_without_tokens_or_portions_need_no_keys():
    """(host code only)"""
    base = dict(q=64, q_stride=2 * 192, q_rot=64, heads=2, nope_dim=128, vdim=128, w=64, scale=0.1, form=0, pos=64, slot=64, seqs=64, seqs_stride=1, n_seqs=1, page_table=64, n_slots=1, max_pages=4,
                page_size=64, n_pages=9, cache=64, out=64, out_stride=256)
    lib, p = native.lib(), native.LatentAttnParams(**base)
    assert lib.ktb200_latent_attn(C.byref(p), 0, 0, None, 0, None) == native.OK
    assert lib.ktb200_latent_attn(C.byref(native.LatentAttnParams(**{**base, "n_seqs": 0})), 4, 0, None, 0, None) == native.OK
    assert lib.ktb200_latent_attn(C.byref(p), 4, 0, None, 0, None) == native.EINVAL
    assert lib.ktb200_latent_attn(C.byref(p), 0, -1, None, 0, None) == native.EINVAL


@gpu
def test_a_call_without_tokens():
    d = draw([(30, 0)], heads=2, seed=71)
    d.batch.max_kv = 0
    assert call(d, None).shape == (0, 256)


@gpu
def test_decoded_tokens_of_very_many_sequences():
    """Sequences times max_kv above 2^30: the absorbed form has no rows of all keys to make room for."""
    d = draw([(5, 1)] * 9000, heads=1, seed=72)
    near_keys = call(d, "absorbed")
    d.batch.max_kv = 131072
    assert torch.equal(call(d, None), near_keys) and torch.isfinite(near_keys).all()


# ------------------------------------------------------------------------------------------------ a scheduler's step
@gpu
@pytest.mark.parametrize("form", ["expanded", "absorbed", None])
@pytest.mark.parametrize("page", [64, 16])
def test_portions_and_decoded_tokens_in_one_call(form, page):
    """A long portion beside decoded tokens and drafts over contexts of very different lengths, an empty portion among them: one form for all of them, each right."""
    d = draw([(900, 1), (0, 700), (3000, 1), (17, 0), (40, 3), (0, 1), (500, 130)], heads=4, page=page, seed=81)
    want, bound = definition(d)
    near(call(d, form), want, bound)
    start = d.kv.clone()
    rot = LatentRotation(10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64).cuda())
    append(d, rot)
    key = torch.cat([torch.arange(b, b + n, device="cuda") for b, n in d.lens])
    at = d.cache.page_table[d.batch.slot.long(), key // page].long(), key % page
    assert (d.kv[at] != start[at]).any(-1).all()
    start[at] = d.kv[at]
    assert torch.equal(d.kv.view(torch.int16), start.view(torch.int16))


# ------------------------------------------------------------------------------------------------ the layer
@gpu
@pytest.mark.parametrize("scaling", [None, YARN])
def test_layer_at_the_end_of_its_cache(scaling):
    """A portion that crosses the end of the static cache, and a decoded token behind it: what the cache holds stays, tokens that fit are right, those that do not see what is there."""
    from ktransformers_b200.models.custom_cache import StaticCache
    from ktransformers_b200.operators.flashinfer_wrapper import MLAWrapper
    cfg, plain = layer(16, 128, scaling, seed=6)
    exact = Exact(cfg, plain)
    op = KDeepseekV2Attention("blk.0.self_attn", None, cfg, plain, "cuda", "cuda")
    cache = StaticCache(cfg, max_batch_size=3, max_cache_len=200, device="cuda")      # 256 positions
    op.mla_wrapper = MLAWrapper(2, cache.max_pages * 2)
    rows = cache.key_cache[0].view(3, 256, 576)
    where = lambda at, n: torch.arange(at, at + n, device="cuda")
    x = torch.randn(2, 263, 512, device="cuda").bfloat16()
    run = lambda at, n: op(x[:, at:at + n], position_ids=where(at, n)[None].expand(2, n), past_key_value=cache, cache_position=where(at, n))[0]
    with torch.no_grad():
        run(0, 250)
        before = rows.clone()
        y = run(250, 12)
        want = exact(x[:, :256], where(0, 256)[None].expand(2, 256))[:, 250:]
        # some ten roundings of 1.65e-3 (root of mean square) one behind the other are 5.2e-3, three times that
        assert (y[:, :6].float() - want).norm() <= 1.6e-2 * want.norm() and torch.isfinite(y).all()
        assert torch.equal(rows[:, :250], before[:, :250]) and (rows[2] == 0).all() and (rows[:2, 250:] != 0).any(-1).all()
        full = rows.clone()
        token = run(262, 1)
        again = op._portion(x[:, 262:], where(262, 1)[None].expand(2, 1), cache, where(262, 1))
        assert torch.equal(rows, full) and (token.float() - again.float()).norm() <= 2 * 1.6e-2 * again.float().norm()      # (both are that far off at most)


@gpu
def test_one_token_step_behind_the_end_of_its_cache():
    """A decoded token behind the static cache, by the layer's fused step and module by module (a rotation of another class): neither writes it anywhere, and both see what is there."""
    from ktransformers_b200.models.custom_cache import StaticCache
    from ktransformers_b200.operators.flashinfer_wrapper import MLAWrapper

    class OtherRotary(DeepseekV3RotaryEmbedding):
        pass

    cfg, plain = layer(16, 128, None, seed=10)
    x, past, outs = torch.randn(2, 3, 1, 512, device="cuda").bfloat16(), torch.randn(3, 128, 576, device="cuda").bfloat16(), []
    for rot in (DeepseekV3RotaryEmbedding(64), OtherRotary(64)):
        plain.rotary_emb = rot.to("cuda")
        op = KDeepseekV2Attention("blk.0.self_attn", None, cfg, plain, "cuda", "cuda")
        cache = StaticCache(cfg, max_batch_size=3, max_cache_len=128, device="cuda")
        cache.key_cache[0].view(3, 128, 576).copy_(past)
        op.mla_wrapper = MLAWrapper(2, cache.max_pages * 2)
        with torch.no_grad():      # (the first call plans, the second does not)
            for i, pos in enumerate((128, 150)):
                outs.append(op(x[:, i], position_ids=torch.full((2, 1), pos, device="cuda"), past_key_value=cache, cache_position=torch.tensor([pos], device="cuda"))[0].float())
        assert torch.equal(cache.key_cache[0].view(3, 128, 576), past)
    for a, b in zip(outs[:2], outs[2:]):
        assert torch.isfinite(a).all() and (a - b).norm() <= 2 * 1.6e-2 * b.norm()      # (some ten roundings of 1.65e-3 in each, three times that)


@gpu
@pytest.mark.parametrize("heads", [4, 128])
def test_layer_with_a_cache_much_longer_than_its_context(heads):
    """Parts of the keys, passes over the heads and workspaces follow the cache's size; results do not."""
    from ktransformers_b200.models.custom_cache import StaticCache
    cfg, plain = layer(heads, 128, YARN, seed=9)
    exact = Exact(cfg, plain)
    op = KDeepseekV2Attention("blk.0.self_attn", None, cfg, plain, "cuda", "cuda")
    cache, at = StaticCache(cfg, max_batch_size=2, max_cache_len=100000, device="cuda"), 0
    for n in (200, 1, 100, 3):
        x, where = torch.randn(2, n, 512, device="cuda").bfloat16(), torch.arange(at, at + n, device="cuda")[None].expand(2, n)
        with torch.no_grad():
            y, want = op(x, position_ids=where, past_key_value=cache, cache_position=where[0])[0], exact(x, where)
        at += n
        assert (y.float() - want).norm() <= 1.6e-2 * want.norm()      # (some ten roundings of 1.65e-3 one behind the other are 5.2e-3, three times that)


def test_scaled_rotation_of_a_layer_built_without_memory():
    """Models are built on the meta device before their weights are loaded: the frequencies are there all the same."""
    cfg = DeepseekV3Config(hidden_size=64, num_attention_heads=2, q_lora_rank=None, num_hidden_layers=1, rope_scaling=dict(YARN))
    with torch.device("meta"):
        rot = DeepseekV3Attention(cfg).rotary_emb
        f = rot.inv_freq_on("cpu")
    assert f.device.type == "cpu" and torch.equal(f, yarn_inv_freq(64, 10000.0, 40, 4096))
    cos, _ = rot(torch.zeros(1), torch.tensor([[0, 7]]))
    assert cos.device.type == "cpu" and torch.equal(cos[0, 1, :32], ((7 * f).cos() * rot.gain).float())


@gpu
def test_scaled_layer_captured_before_its_first_call():
    """Nothing of a scaled rotation is copied from the host by the first call: it may be a captured one.  The same bits as eagerly."""
    from ktransformers_b200.models.custom_cache import StaticCache
    cfg, plain = layer(4, 64, YARN, seed=8)
    op = KDeepseekV2Attention("blk.0.self_attn", None, cfg, plain, "cuda", "cuda")
    x, at = torch.randn(2, 1, 512, device="cuda").bfloat16(), torch.full((1,), 3000, device="cuda")
    run = lambda cache: op(x, position_ids=at[None].expand(2, 1), past_key_value=cache, cache_position=at)[0]
    make = lambda: StaticCache(cfg, max_batch_size=2, max_cache_len=3010, device="cuda")
    with torch.no_grad():
        eager = make()
        want = run(eager)
        plain.rotary_emb = DeepseekV3YarnRotaryEmbedding(64, scaling_factor=40, mscale=1.0, mscale_all_dim=1.0)
        cache, g = make(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            y = run(cache)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(cache.key_cache[0], eager.key_cache[0])
        assert torch.equal(run(cache), want)      # and eagerly behind the captured call


@pytest.mark.parametrize("given", [dict(rope_scaling=YARN), dict(rope_scaling=YARN, rope_theta=50000.0), dict(rope_parameters={**YARN, "rope_type": "yarn", "rope_theta": 50000.0}),
                                   dict(rope_parameters={"rope_type": "default", "rope_theta": 50000.0}), dict()])
def test_a_scaled_configuration_comes_back(given, tmp_path):
    """A configuration whose rotation is scaled is the same after to_dict and after a file, and has the same layer, under either name that checkpoints give the scaling; the caller's dict stays."""
    held = {k: dict(v) if isinstance(v, dict) else v for k, v in given.items()}
    first = DeepseekV3Config(hidden_size=64, num_attention_heads=2, q_lora_rank=None, num_hidden_layers=1, **given)
    assert given == held
    first.save_pretrained(tmp_path)
    base = 50000.0 if "rope_parameters" in given or "rope_theta" in given else 10000.0
    for cfg in (first, DeepseekV3Config.from_dict(first.to_dict()), DeepseekV3Config.from_pretrained(tmp_path)):
        rot, wanted = DeepseekV3Attention(cfg).rotary_emb, next((v for v in given.values() if isinstance(v, dict)), None)
        if wanted is None or wanted.get("rope_type") == "default":
            assert type(rot) is DeepseekV3RotaryEmbedding and rot.base == base
        else:
            assert {k: cfg.rope_scaling[k] for k in YARN} == YARN
            assert torch.equal(rot.inv_freq_on("cpu"), yarn_inv_freq(64, base, 40, 4096))
            assert math.isclose(DeepseekV3Attention(cfg).softmax_scale, 192 ** -0.5 * yarn_get_mscale(40, 1.0) ** 2)
