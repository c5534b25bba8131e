"""latent_append and latent_attention against their definitions in 64 bits: forms, head layouts, lengths, pages, strides, portions without tokens, rows that are not finite, streams and graphs."""
import ctypes as C
import math
from types import SimpleNamespace

import pytest
import torch

from latent_util import HALF, RANK, ROT, attention, batch_of, draw, near, turned
from ktransformers_b200 import native
from ktransformers_b200.operators.latent_attention import LatentRotation, latent_append, latent_attention, yarn_inv_freq

gpu = pytest.mark.gpu


def call(d, form=None, **kw):
    return latent_attention(d.q, d.q_rot, d.kv, d.w, d.batch, d.cache, d.heads, d.nope, d.vdim, d.scale, form=form, **kw)


# ------------------------------------------------------------------------------------------------ attention
@gpu
@pytest.mark.parametrize("form", ["expanded", "absorbed"])
@pytest.mark.parametrize("lens,heads,nope,vdim,page", [
    ([(0, 1)], 4, 128, 128, 64),                       # one token, nothing before
    ([(0, 128)], 3, 128, 128, 64),                     # one whole row tile
    ([(0, 257)], 2, 128, 128, 64),                     # a tile of one token behind a whole one
    ([(127, 2)], 4, 128, 128, 64),                     # across a key tile
    ([(1000, 130)], 5, 128, 128, 64),                  # heads that are no power of two
    ([(300, 90), (0, 200), (77, 1)], 4, 64, 128, 32),  # portions of different lengths
    ([(45, 60), (512, 64)], 16, 128, 64, 16),          # pages that end inside a tile
    ([(700, 333)], 2, 64, 64, 48),                     # pages that are no power of two
    ([(5000, 70)], 4, 128, 128, 64),                   # few tiles, many keys: parts
    ([(2000, 3)] * 5, 128, 128, 128, 64),              # drafts
])
def test_attention_against_64_bits(form, lens, heads, nope, vdim, page):
    d = draw(lens, heads, nope, vdim, page, seed=len(lens) + heads)
    want, bound = attention(d)
    near(call(d, form), want, bound)


@gpu
@pytest.mark.parametrize("form", ["expanded", "absorbed"])
def test_attention_leaves_other_rows_and_columns(form):
    """Portions without tokens, a portion in a slot that is not there, tokens in no portion, an output inside a wider one, queries of a wider row."""
    d = draw([(100, 40), (30, 0), (200, 70)], heads=3, idle=9, seed=3)
    T = d.batch.n_tokens
    wide = torch.full((T, 3 * 128 + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    rows = torch.full((T, 3 * 192 + 8), math.nan, dtype=torch.bfloat16, device="cuda")
    rows[:, :3 * 192] = d.q
    want, bound = attention(d)
    out = latent_attention(rows, d.q_rot, d.kv, d.w, d.batch, d.cache, 3, 128, 128, d.scale, form=form, out=wide[:, 8:8 + 384])
    assert out.data_ptr() == wide[:, 8:].data_ptr()
    near(out[:110], want, bound)
    assert (wide[110:] == 7).all() and (wide[:, :8] == 7).all() and (wide[:, 392:] == 7).all()
    d.batch.slot[:40] = 55
    again = torch.full((T, 384), 7.0, dtype=torch.bfloat16, device="cuda")
    latent_attention(d.q, d.q_rot, d.kv, d.w, d.batch, d.cache, 3, 128, 128, d.scale, form=form, out=again)
    assert (again[:40] == 7).all() and torch.equal(again[40:110], out[40:110]) and (again[110:] == 7).all()


@gpu
@pytest.mark.parametrize("form", ["expanded", "absorbed"])
@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("page", [64, 16])
def test_attention_rows_that_are_not_finite(form, what, page):
    """What lies behind a sequence's last token is never multiplied; a latent or rotated key that is not finite reaches the rows that see it and no others."""
    d = draw([(70, 100), (0, 90)], heads=2, page=page, seed=5)
    table = d.cache.page_table.long()
    clean = call(d, form)
    for i, n in enumerate((170, 90)):
        if n % page:
            d.kv[table[i, n // page], n % page:] = what
    d.kv[[p for p in range(d.kv.shape[0]) if p not in table[table >= 0].tolist()]] = what
    assert torch.equal(call(d, form), clean)
    d.kv[table[0, 120 // page], 120 % page, 300] = what
    d.kv[table[1, 5 // page], 5 % page, RANK + 3] = what
    got = call(d, form)
    assert torch.equal(got[:50], clean[:50]) and torch.equal(got[100:105], clean[100:105])
    assert not torch.isfinite(got[50:100]).any()
    # an infinite rotated key of a finite latent: its score is infinite, and where that is below zero it has no weight
    none = (d.q_rot[105:, :, 3] < 0)[..., None].expand(-1, -1, 128).reshape(-1, 256) if what == math.inf else torch.zeros_like(got[105:], dtype=torch.bool)
    assert torch.equal(torch.isfinite(got[105:]), none)


@gpu
@pytest.mark.parametrize("form", ["expanded", "absorbed"])
def test_attention_large_scores_and_one_key_with_all_the_weight(form):
    """Scores that grow along the keys raise the running maximum tile by tile; one key far above the others leaves its value alone."""
    d = draw([(600, 70)], heads=2, seed=7)
    grow = torch.linspace(0.05, 3.0, d.kv.shape[0] * 64, device="cuda")
    pages = d.cache.page_table[0, :11].long()
    d.kv[pages] = (d.kv[pages].float() * grow[:11 * 64].view(11, 64, 1)).bfloat16()
    want, bound = attention(d)
    near(call(d, form), want, bound, rel=2.5e-2)      # (a spread of scores of about three: 3 x 1.65e-3 of a weight, twice; and the sums' own)
    d.q.zero_()
    d.q_rot.zero_()
    d.q_rot[:, :, 0] = 64.0
    d.kv[..., RANK:] = 0
    d.kv[pages[2], 9, RANK] = 64.0                     # 64 * 64 / sqrt(192) = 296 above the others
    got = call(d, form)
    value = d.kv[pages[2], 9, :RANK].double() @ d.w.view(2, 256, RANK)[:, 128:].double().transpose(1, 2)
    assert ((got.double() - value.reshape(1, -1)).abs() <= value.abs().reshape(1, -1) * 2.1 * HALF + 1e-6).all()


@gpu
@pytest.mark.parametrize("form,page", [("expanded", 64), ("absorbed", 64), ("absorbed", 16)])
def test_attention_with_fewer_keys_than_there_are(form, page):
    """A max_kv that a portion's positions pass: that portion's rows are whatever they are, nothing else is touched, and the portion that keeps to it is right."""
    d = draw([(3000, 40), (50, 60)], heads=2, page=page, seed=21)
    want, bound = attention(d)
    d.batch.max_kv = 128
    got = torch.full((109, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    call(d, form, out=got[:100])
    near(got[40:100], want[40:], bound[40:])
    assert (got[100:] == 7).all()


@gpu
def test_one_row_of_any_width():
    d = draw([(130, 1)], heads=3, seed=22)
    want, bound = attention(d)
    wide = torch.full((1, 3 * 192 + 5), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, :576] = d.q
    d.q = wide
    for form in ("expanded", "absorbed"):
        near(call(d, form), want, bound)


@gpu
def test_attention_in_passes_over_the_heads():
    """More keys and values than one pass holds (40,000 keys of 128 heads are 2.6 GB); with a bound far above the keys there are, the passes behind the first find nothing to do."""
    d = draw([(39936, 64)], heads=128, seed=9)
    got = call(d, "expanded")
    for h in (0, 101, 127):
        one = SimpleNamespace(**{**vars(d), "heads": 1, "q": d.q.view(64, 128, 192)[:, h].contiguous(), "q_rot": d.q_rot[:, h:h + 1], "w": d.w.view(128, 256, RANK)[h].contiguous()})
        want, bound = attention(one)
        near(got.view(64, 128, 128)[:, h], want, bound)
    d = draw([(100, 70)], heads=128, seed=10, max_kv=150000)
    want, bound = attention(d)
    near(call(d, "expanded"), want, bound)


@gpu
def test_attention_beyond_32_bits_of_offset():
    """A pool whose last pages lie more than 2^31 elements behind its first."""
    pages = (1 << 31) // (64 * 576) + 40
    d = draw([(190, 66)], heads=2, seed=11)
    pool = torch.zeros((pages, 64, 576), dtype=torch.bfloat16, device="cuda")
    used = d.cache.page_table[0, :4].long()
    far = torch.arange(pages - 4, pages, device="cuda").flip(0)
    pool[far] = d.kv[used]
    want, bound = attention(d)
    d.kv = pool
    d.cache.page_table[0, :4] = far.int()
    for form in ("expanded", "absorbed"):
        near(call(d, form), want, bound)


@gpu
@pytest.mark.parametrize("form", ["expanded", "absorbed"])
def test_attention_again_on_another_stream_and_in_a_graph(form):
    """The same bits each time: eagerly, on a side stream, and replayed with other tokens, positions and pages in the captured call's tensors; two graphs next to each other."""
    a, b = draw([(130, 80), (0, 90)], heads=4, seed=13), draw([(64, 80), (70, 90)], heads=4, seed=14)
    first, other = call(a, form), call(b, form)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(call(a, form), first)
    torch.cuda.synchronize()
    a.batch.max_kv = b.batch.max_kv = 256
    graphs = []
    for d in (a, b):
        out = torch.zeros_like(first)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(d, form, out=out)
        graphs.append((g, out))
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], first) and torch.equal(graphs[1][1], other)
    n = min(a.kv.shape[0], b.kv.shape[0])
    for name in ("q", "q_rot", "w"):
        getattr(a, name).copy_(getattr(b, name))
    for name in ("pos", "slot", "seqs"):
        getattr(a.batch, name).copy_(getattr(b.batch, name))
    a.cache.page_table.zero_()
    used = b.cache.page_table[:, :3].long()
    for i in range(2):      # the same contents in other pages of a's pool (six of them hold both)
        for j in range(3):
            if int(used[i, j]) >= 0:
                a.kv[3 * i + j] = b.kv[used[i, j]]
                a.cache.page_table[i, j] = 3 * i + j
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], other) and n >= 6


# ------------------------------------------------------------------------------------------------ append
def append_case(lens, heads=3, nope=128, rank=RANK, rot_dim=ROT, page=64, seed=0, idle=0):
    batch, cache, total = batch_of(lens, page, seed=seed, idle=idle)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")
    T = batch.n_tokens
    return SimpleNamespace(batch=batch, cache=cache, lens=lens, heads=heads, nope=nope, page=page, q=rand(T, heads * (nope + rot_dim)).bfloat16(),
                           kva=torch.cat((rand(T, rank) * 3, rand(T, rot_dim)), 1).bfloat16(), weight=(1 + 0.2 * rand(rank)).bfloat16(), kv=rand(total, page, rank + rot_dim).bfloat16())


def check_append(d, rot, freq, q=None, kva=None, positions=None):
    q, kva = d.q if q is None else q, d.kva if kva is None else kva
    rank = d.weight.numel()
    before, width = d.kv.clone(), d.kv.shape[2]
    rot_dim = width - rank
    got = latent_append(q, kva, d.weight, 1e-5, d.batch, d.cache, d.kv, d.heads, d.nope, rot=rot, inv_freq=freq, positions=positions)
    T = sum(n for _, n in d.lens)
    at = (positions if positions is not None else d.batch.pos)[:T]
    hw = d.nope + rot_dim
    part = d.q[:T].reshape(T, d.heads, hw)[..., d.nope:]
    turn = lambda x: turned(x, at, rot, freq) if rot is not None else x.double()
    want = turn(part)
    # one rounding; the angle's remainder is a number of 32 bits of at most pi (2^-23 off), cosine, sine and products as much again: 2^-20 of the pair's length
    length = (turn(part).abs() + (part.double().abs().amax(-1, keepdim=True) if rot_dim else 0)) * 2.0 ** -20 * (rot.gain if rot is not None else 1)
    assert ((got[:T].double() - want).abs() <= want.abs() * HALF + length).all()
    x = d.kva[:T, :rank].double()
    latent = x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-5) * d.weight.double()
    key = turn(d.kva[:T, None, rank:width])[:, 0]
    p = d.batch.pos[:T].long()
    page = d.cache.page_table[d.batch.slot[:T].long(), p // d.page].long()
    row = d.kv[page, p % d.page].double()
    assert ((row[:, :rank] - latent).abs() <= latent.abs() * (HALF + 2.0 ** -20)).all()
    if rot_dim:
        assert ((row[:, rank:] - key).abs() <= key.abs() * HALF + (key.abs() + d.kva[:T, rank:width].double().abs().amax(1, keepdim=True)) * 2.0 ** -20 * (rot.gain if rot is not None else 1)).all()
    before[page, p % d.page] = d.kv[page, p % d.page]
    assert torch.equal(before.view(torch.int16), d.kv.view(torch.int16))      # nothing else was written
    return got


def rotation(layout, split, gain, dims, factor=1.0):
    freq = yarn_inv_freq(dims, 10000.0, factor, 4096) if factor > 1 else 10000.0 ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    return LatentRotation(freq.cuda(), layout, split, gain)


@gpu
@pytest.mark.parametrize("lens,heads,nope,rank,rot_dim,page,dims,layout,split,gain,factor", [
    ([(160000, 1)], 128, 128, 512, 64, 64, 64, "interleaved", True, 1.0, 40.0),      # far in a scaled context
    ([(5, 300)], 128, 128, 512, 64, 64, 64, "interleaved", True, 1.0, 1.0),
    ([(0, 40), (63, 2), (100, 0), (31, 65)], 5, 64, 512, 64, 16, 64, "interleaved", False, 1.3, 4.0),
    ([(10, 33)], 16, 128, 512, 64, 48, 32, "halves", False, 1.37, 40.0),             # half of the columns
    ([(7, 9), (70, 4)], 2, 33, 100, 30, 10, 18, "interleaved", True, 1.1, 1.0),      # no whole 16 bytes anywhere
    ([(7, 9)], 3, 0, 256, 20, 7, 20, "halves", False, 1.0, 1.0),
    ([(3, 5)], 2, 128, 512, 64, 64, 0, "halves", False, 1.0, 1.0),                   # nothing turned
    ([(3, 5)], 2, 64, 512, 0, 64, 0, "halves", False, 1.0, 1.0),                     # no rotated part
    ([(20, 1)] * 70, 16, 128, 512, 64, 32, 64, "halves", False, 1.0, 1.0),           # a decode batch
])
def test_append_against_64_bits(lens, heads, nope, rank, rot_dim, page, dims, layout, split, gain, factor):
    d = append_case(lens, heads, nope, rank, rot_dim, page, seed=heads)
    rot = rotation(layout, split, gain, dims, factor) if dims else None
    check_append(d, rot, rot.inv_freq if rot else None)


@gpu
def test_append_strides_other_positions_and_idle_tokens():
    d = append_case([(9, 20), (70, 30)], heads=4, seed=2, idle=6)
    rot = rotation("interleaved", True, 1.0, 64)
    T = d.batch.n_tokens
    q = torch.full((T, 4 * 192 + 5), math.nan, dtype=torch.bfloat16, device="cuda")
    kva = torch.full((T, 576 + 3), math.nan, dtype=torch.bfloat16, device="cuda")
    q[:, 3:3 + 768], kva[:, 1:577] = d.q, d.kva
    positions = torch.randint(0, 1 << 20, (T,), dtype=torch.int32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    check_append(d, rot, rot.inv_freq, q[:, 3:3 + 768], kva[:, 1:577], positions)
    a = check_append(d, rot, rot.inv_freq)
    b = check_append(d, rot, rot.inv_freq, q[:, 3:3 + 768], kva[:, 1:577])      # (the unaligned rows' path)
    assert torch.equal(a[:50], b[:50])


@gpu
def test_append_skips_what_is_not_there():
    """A slot outside the table, a page outside the pool and a position below zero: nothing is written."""
    d = append_case([(9, 20), (70, 30), (0, 4)], heads=2, seed=4)
    rot = rotation("interleaved", True, 1.0, 64)
    d.batch.slot[:20] = 77
    d.cache.page_table[1] = torch.tensor([-1, d.kv.shape[0]] * 8, dtype=torch.int32, device="cuda")[:d.cache.page_table.shape[1]]
    d.batch.pos[50:] = -3
    before = d.kv.clone()
    latent_append(d.q, d.kva, d.weight, 1e-5, d.batch, d.cache, d.kv, 2, 128, rot=rot)
    assert torch.equal(before.view(torch.int16), d.kv.view(torch.int16))
    got = latent_attention(d.q, d.q.new_zeros((54, 2, 64)), d.kv, d.q.new_zeros((512, 512)), d.batch, d.cache, 2, 128, 128, 1.0, form="expanded", out=torch.full((54, 256), 7.0, dtype=torch.bfloat16, device="cuda"))
    assert (got[:20] == 7).all() and (got[50:] == 7).all()


def test_yarn_frequencies():
    """The ends keep their frequency and are divided by the factor; between them the frequency falls with the column; a factor of one changes nothing."""
    plain = yarn_inv_freq(64, 10000.0, 1.0, 4096)
    i = torch.arange(32, dtype=torch.float64)
    assert torch.allclose(plain, 10000.0 ** (-i / 32), rtol=1e-14)
    f = yarn_inv_freq(64, 10000.0, 40.0, 4096)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(f[turns > 32 * 10000 ** (1 / 32)], plain[turns > 32 * 10000 ** (1 / 32)])
    slow = turns < 10000 ** (-1 / 32)
    assert torch.allclose(f[slow], plain[slow] / 40, rtol=1e-14) and (f[1:] < f[:-1]).all() and slow.any()


# ------------------------------------------------------------------------------------------------ refusals (host code only)
def test_calls_refuse_cpu_tensors():
    batch, cache, total = batch_of([(3, 4)], device="cpu")
    t = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        latent_append(t(4, 2 * 192), t(4, 576), t(512), 1e-6, batch, cache, t(total, 64, 576), 2, 128)
    with pytest.raises(ValueError, match="CUDA"):
        latent_attention(t(4, 2 * 192), t(4, 2, 64), t(total, 64, 576), t(512, 512), batch, cache, 2, 128, 128, 0.1)
    with pytest.raises(ValueError, match="bfloat16"):
        latent_append(t(4, 2 * 192), t(4, 576), t(512), 1e-6, batch, cache, t(total, 64, 576).float(), 2, 128)


def attn_params(**kw):
    base = dict(q=64, q_stride=2 * 192, q_rot=64, heads=2, nope_dim=128, vdim=128, w=64, scale=0.1, form=0, pos=64, slot=64, seqs=64, seqs_stride=1, n_seqs=1, page_table=64, n_slots=1, max_pages=4,
                page_size=64, n_pages=9, cache=64, out=64, out_stride=256)
    return native.LatentAttnParams(**{**base, **kw})


@pytest.mark.parametrize("wrong", [dict(heads=0), dict(nope_dim=96), dict(vdim=192), dict(form=3), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(q_stride=100), dict(q_stride=2 * 192 + 4),
                                   dict(out_stride=255), dict(page_size=0), dict(n_pages=0), dict(max_pages=0), dict(n_slots=0), dict(n_seqs=-1), dict(n_pages=1 << 30), dict(q=0), dict(w=0), dict(cache=8),
                                   dict(q_rot=2), dict(pos=0), dict(out=0)])
def test_attention_refuses_on_the_host(wrong):
    a = attn_params(**wrong)
    lib = native.lib()
    assert lib.ktb200_latent_attn(C.byref(a), 4, 100, None, 0, None) == native.EINVAL
    assert lib.ktb200_latent_attn(C.byref(attn_params()), 4, 0, None, 0, None) == native.EINVAL
    assert lib.ktb200_latent_attn(C.byref(attn_params()), 0, 100, None, 0, None) == native.OK
    assert lib.ktb200_latent_attn(C.byref(attn_params(n_seqs=0)), 4, 100, None, 0, None) == native.OK


def test_form_follows_the_tokens_a_sequence():
    form = lambda T, n, keys=9000, f=0: native.lib().ktb200_latent_attn_form(C.byref(attn_params(n_seqs=n, form=f)), T, keys)
    assert form(1, 1) == 1 and form(2000, 1) == 2 and form(40, 40) == 1 and form(4000, 4) == 2 and form(1, 1, f=2) == 2 and form(4000, 1, f=1) == 1
    assert form(100, 1, keys=1000) == 2 and form(100, 1) == 1 and form(63, 1, keys=1000) == 1


@pytest.mark.parametrize("wrong", [dict(heads=0), dict(kv_rank=0), dict(rot_dims=66), dict(rot_dims=7), dict(rot_layout=2), dict(inv_freq=0), dict(q_stride=1), dict(kva_stride=575), dict(page_size=0),
                                   dict(q=0), dict(cache=0), dict(seqs=0), dict(n_seqs=-1), dict(rot_dim=300, rot_dims=258, q_stride=4000, kva_stride=4000)])
def test_append_refuses_on_the_host(wrong):
    base = dict(q=64, q_stride=384, heads=2, nope_dim=128, kva=64, kva_stride=576, kv_rank=512, rot_dim=64, norm_weight=64, eps=1e-6, rot_dims=64, rot_layout=0, rot_split=1, rot_gain=1.0, inv_freq=64,
                angle_pos=0, pos=64, slot=64, seqs=64, seqs_stride=1, n_seqs=1, page_table=64, n_slots=1, max_pages=4, page_size=64, n_pages=9, cache=64, q_rot=64)
    lib = native.lib()
    assert lib.ktb200_latent_append(C.byref(native.LatentAppendParams(**{**base, **wrong})), 4, None) == native.EINVAL
    assert lib.ktb200_latent_append(C.byref(native.LatentAppendParams(**base)), 0, None) == native.OK


@gpu
def test_calls_refuse_on_the_gpu():
    d = draw([(3, 70)], heads=2)
    ok = dict(q=d.q, q_rot=d.q_rot, kv=d.kv, w=d.w, batch=d.batch, cache=d.cache, heads=2, nope=128, vdim=128, scale=0.1)
    latent_attention(**ok)
    other = lambda **kw: SimpleNamespace(**{**vars(d.batch), **kw})
    for wrong in (dict(q=d.q.float()), dict(q=d.q[:, :300]), dict(q=d.q[:50]), dict(q_rot=d.q_rot[:, :1]), dict(q_rot=d.q_rot.cpu()), dict(kv=d.kv.float()), dict(kv=d.kv[..., :512]), dict(kv=d.kv[:, ::2]),
                  dict(w=d.w[:-1]), dict(w=d.w.half()), dict(w=d.w.t()), dict(heads=3), dict(nope=96), dict(vdim=96), dict(scale=0.0), dict(form="both"), dict(batch=other(pos=d.batch.pos.long())),
                  dict(batch=other(pos=d.batch.pos[:9])), dict(batch=other(n_seqs=5)), dict(batch=other(seqs=d.batch.seqs.cpu())), dict(batch=other(max_kv=0)),
                  dict(cache=SimpleNamespace(page_table=d.cache.page_table, max_pages_per_seq=9, page_size=64)), dict(out=torch.empty((73, 256), dtype=torch.float32, device="cuda")),
                  dict(out=torch.empty((72, 256), dtype=torch.bfloat16, device="cuda")), dict(out=torch.empty((256, 73), dtype=torch.bfloat16, device="cuda").t())):
        with pytest.raises((ValueError, RuntimeError)):
            latent_attention(**{**ok, **wrong})
