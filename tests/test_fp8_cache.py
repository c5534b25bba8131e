"""The paged e4m3 cache: append (rotation, norms, codes, scales) and attention, against 64-bit forms (fp8_cache_util)."""
import ctypes as C
import math
from types import SimpleNamespace

import pytest
import torch

import fp8_cache_util as U
from ktransformers_b200 import native
from ktransformers_b200.models.custom_cache import Fp8CacheLayer, PagedStateCache
from ktransformers_b200.operators.attention import fp8_cache_append, fp8_cache_attention

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
ROT = lambda dims, layout: SimpleNamespace(dims=dims, layout_code=layout)
INV = lambda dims: 10000.0 ** (-torch.arange(0, dims, 2, dtype=torch.float64) / max(dims, 1))


def filled(total, G, ps, d, dv, seed, wide=0):
    """a pool that holds something everywhere; `wide`: scales over so many powers of two"""
    g = torch.Generator().manual_seed(seed)
    codes = lambda n: torch.randn((total, G, ps, n), generator=g).mul_(60).to(U.E4M3)
    return codes(d), codes(dv), torch.exp2(torch.randint(-6 - wide, -5 + wide, (total, G, 2), generator=g).float())


def on(x, device="cuda"):
    if isinstance(x, SimpleNamespace):
        return SimpleNamespace(**{k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in vars(x).items()})
    return x.to(device) if isinstance(x, torch.Tensor) else x


# ------------------------------------------------------------------------------------------------------------------------- CPU
def test_exponent_is_the_smallest_that_reaches():
    for top in (448.0, 448.0000305, 447.99997, 1.0, 1.75, 1.7500001, 3.5, 1e-30, 1e30, 0.0, 2.0 ** -56 * 448):
        e = U.exponent(top)
        assert -64 <= e <= 64
        if -64 < e < 64:
            assert 448.0 * 2.0 ** e >= top > 448.0 * 2.0 ** (e - 1)


def test_layer_refuses_other_tensors():
    k, v, s = filled(2, 2, 4, 8, 8, 0)
    Fp8CacheLayer(k, v, s)
    for bad in ((k.float(), v, s), (k, v[:, :, :2], s), (k, v, s[:, :, :1]), (k, v, s.double()), (k.transpose(2, 3), v, s), (k[0], v[0], s[0]), (k, v.to("meta"), s)):
        with pytest.raises(ValueError):
            Fp8CacheLayer(*bad)
    assert [tuple(x.shape) for x in Fp8CacheLayer(k, v, s).dequantize()] == [(2, 2, 4, 8)] * 2


def test_cache_manager_holds_layers_in_both_widths():
    c = PagedStateCache([0, 32, 32], 0, 64, 2, "cpu", page_size=16, fp8_heads=[None, (2, 8, 8), None])
    assert isinstance(c.key_cache[1], Fp8CacheLayer) and c.key_cache[1].k.shape == (c.num_pages, 2, 16, 8) and c.key_cache[2].shape == (c.num_pages, 16, 32)
    with pytest.raises(ValueError, match="one entry"):
        PagedStateCache([32, 32], 0, 64, 2, "cpu", page_size=16, fp8_heads=[None])


RotDims = lambda dims: SimpleNamespace(dims=dims, layout_code=0)


@pytest.mark.gpu
def test_wrappers_refuse_what_does_not_fit():
    batch, cache, total = U.batch_of([(5, 1)], 16)
    kv = Fp8CacheLayer(*filled(total, 2, 16, 32, 32, 0))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        fp8_cache_append(torch.zeros(1, 256), batch, cache, kv, 4, 2, 32, 32, (0, 128, 192))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        fp8_cache_attention(torch.zeros(1, 4, 32), kv, batch, cache, 4, 2, 32, 32, 0.1)


APPEND_OK = dict(proj=16, proj_stride=256, heads=4, kv_heads=2, dim=32, vdim=32, pos=16, slot=16, seqs=16, n_seqs=1, page_table=16, n_slots=1, max_pages=2, page_size=16, n_pages=2, k_codes=16, v_codes=16,
                 scales=16, q_out=16)
ATTN_OK = dict(q=16, heads=4, kv_heads=2, dim=32, vdim=32, scale=1.0, out_scale=1.0, pos=16, slot=16, seqs=16, n_seqs=1, page_table=16, n_slots=1, max_pages=2, page_size=16, n_pages=2, k_codes=16,
               v_codes=16, scales=16, out=16, out_stride=128)


@pytest.mark.parametrize("bad", [dict(kv_heads=3), dict(dim=257), dict(dim=0), dict(vdim=300), dict(rot_dims=3), dict(rot_dims=34), dict(rot_dims=8), dict(rot_layout=2), dict(qk_norm=2), dict(qk_norm=3),
                                 dict(page_size=0), dict(max_pages=0), dict(n_slots=0), dict(n_seqs=-1), dict(proj=None), dict(q_out=None), dict(scales=None), dict(k_codes=None), dict(seqs=None)])
def test_append_refuses(bad):
    a = native.Fp8AppendParams(**{**APPEND_OK, **bad})
    assert native.seq_lib().ktb200_fp8_cache_append(C.byref(a), 1, native.GGML_BF16, None) == native.EINVAL
    assert b"fp8_cache_append" in native.seq_lib().ktb200_last_error()


def test_append_refuses_types_and_takes_no_tokens():
    lib, a = native.seq_lib(), native.Fp8AppendParams(**APPEND_OK)
    assert lib.ktb200_fp8_cache_append(C.byref(a), 1, native.GGML_F16, None) == native.EINVAL
    assert lib.ktb200_fp8_cache_append(None, 1, native.GGML_BF16, None) == native.EINVAL
    assert lib.ktb200_fp8_cache_append(C.byref(a), 0, native.GGML_BF16, None) == native.OK


@pytest.mark.parametrize("bad,call", [(dict(kv_heads=3), {}), (dict(dim=257), {}), (dict(vdim=0), {}), (dict(page_size=0), {}), (dict(window=-1), {}), (dict(chunk=-4), {}), (dict(out_stride=127), {}),
                                      (dict(q=None), {}), (dict(out=None), {}), (dict(scales=None), {}), ({}, dict(part=-128)), ({}, dict(part=100)), ({}, dict(max_keys=-1)),
                                      ({}, dict(part=128, max_keys=128 * 129)), ({}, dict(part=128, max_keys=1000)), ({}, dict(part=128, max_keys=1000, ws=16, n=100)), ({}, dict(dtype=native.GGML_F16))])
def test_attention_refuses(bad, call):
    a = native.Fp8AttnParams(**{**ATTN_OK, **bad})
    lib, o = native.seq_lib(), {**dict(max_keys=32, part=0, ws=None, n=0, dtype=native.GGML_BF16), **call}
    assert lib.ktb200_fp8_cache_attn(C.byref(a), 1, o["max_keys"], o["part"], o["ws"], o["n"], o["dtype"], 1, None) == native.EINVAL
    assert b"fp8_cache_attn" in lib.ktb200_last_error()


def test_attention_takes_no_tokens():
    lib, a = native.seq_lib(), native.Fp8AttnParams(**ATTN_OK)
    assert lib.ktb200_fp8_cache_attn(C.byref(a), 0, 32, 0, None, 0, native.GGML_F32, 1, None) == native.OK


@pytest.mark.parametrize("dtype", [native.GGML_BF16, native.GGML_F32])
@pytest.mark.parametrize("heads,kv_heads", [(64, 8), (16, 2), (7, 7), (17, 1), (64, 1)])
@pytest.mark.parametrize("n_seqs,n_tokens", [(1, 1), (3, 3), (200, 200), (2, 50), (1, 3000)])
def test_attention_parts_of_any_range_are_few(n_seqs, n_tokens, heads, kv_heads, dtype):
    lib = native.seq_lib()
    for window, chunk in ((0, 0), (700, 0), (0, 4096)):
        a = native.Fp8AttnParams(**{**ATTN_OK, **dict(heads=heads, kv_heads=kv_heads, n_seqs=n_seqs, window=window, chunk=chunk)})
        for keys in (1, 300, 5000, 131072, 1 << 24, 2 ** 31 - 1):
            need = lib.ktb200_fp8_cache_attn_workspace(C.byref(a), n_tokens, keys, -1, dtype, 1)
            assert need % (n_tokens * heads * 34 * 4) == 0 and need // (n_tokens * heads * 34 * 4) <= 128
            assert lib.ktb200_fp8_cache_attn_workspace(C.byref(a), n_tokens, keys, 0, dtype, 1) == 0


def test_engine_refuses_an_8_bit_cache_where_there_is_none():
    from ktransformers_b200.util.engine import Engine
    model = SimpleNamespace(make_cache=lambda *a, **k: None)
    with pytest.raises(ValueError, match="has no 'fp8' cache"):
        Engine(model, kv_cache="fp8")


def test_lipadra_keeps_its_attention_rows_in_8_bits_where_asked():
    import lipadra_util as LU
    from ktransformers_b200.models.configuration_lipadra import LipadraConfig
    from ktransformers_b200.models.modeling_lipadra import LipadraForCausalLM
    cfg = LipadraConfig.from_dict(LU.config([(LU.attention(dim=16, vdim=16), None), (LU.retention(), None)]))
    model = LipadraForCausalLM(cfg, device="cpu")
    c = model.make_cache(64, max_slots=2, page_size=16, kv_cache="fp8")
    assert isinstance(c.key_cache[0], Fp8CacheLayer) and c.key_cache[0].k.shape[1:] == (2, 16, 16) and not isinstance(c.key_cache[1], Fp8CacheLayer)
    with pytest.raises(ValueError, match="no 'int4' cache"):
        model.make_cache(64, kv_cache="int4")


def test_prep_and_attention_refuse_what_8_bit_layers_do_not_have():
    from ktransformers_b200.operators.attention import paged_softmax_attention, qkv_prep
    batch, cache, total = U.batch_of([(5, 1)], 16)
    kv = Fp8CacheLayer(*filled(total, 2, 16, 32, 32, 0))
    with pytest.raises(ValueError, match="8 bits"):
        qkv_prep(torch.zeros(1, 256), batch, cache, kv, 4, 2, 32, 32, (0, 128, 192), maps=2)
    with pytest.raises(ValueError, match="8 bits"):
        paged_softmax_attention(torch.zeros(1, 4, 32), kv, batch, cache, 4, 2, 32, 32, 0.1, gate=torch.zeros(1, 128))


# ------------------------------------------------------------------------------------------------------------------------- append
# fp32 against 64 bits: the turn is two products and a sum (3 x 2^-24 of |x| + |y|) with sine and cosine 2^-22 off, a norm 13 roundings of a sum of squares (half of
# them in the root) and three more: in all below 32 x 2^-24 of a row's largest
FP32_OFF = 32 * 2.0 ** -24


def run_append(lens, ps, H, G, d, dv, dtype, rot=None, norm=0, seed=0, tail=0, gap=0, scale=None, held=None, times=1):
    """One append on the GPU beside its 64-bit form; checks everything that it returns and what it leaves alone"""
    g = torch.Generator().manual_seed(seed)
    batch, cache, total = U.batch_of(lens, ps, seed=seed, tail=tail)
    T, dt = batch.pos.shape[0], DT[dtype]
    offs = (gap, gap + H * d + gap, gap + H * d + gap + G * d + gap)
    proj = torch.randn((T, offs[2] + G * dv + gap), generator=g)
    if scale is not None:
        proj = proj * scale(T)
    proj = proj.to(dt)
    k, v, s = held or filled(total, G, ps, d, dv, seed)
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(dt) for _ in range(2)] if norm == 3 else [None, None]
    inv = INV(rot.dims) if rot is not None else None
    q_ref, k_ref, v_ref, s_ref, k_exact, v_exact = U.append(proj, batch, cache, k, v, s, H, G, d, dv, offs, rot, inv, norm, 1e-5, *w)
    kv = Fp8CacheLayer(*(x.cuda() for x in (k, v, s)))
    for _ in range(times):
        q = fp8_cache_append(proj.cuda(), on(batch), on(cache), kv, H, G, d, dv, offs, rot, on(inv), norm, 1e-5, *map(on, w))
    torch.cuda.synchronize()
    off = FP32_OFF * q_ref.abs().amax(-1, keepdim=True)
    assert ((q.cpu().double() - q_ref).abs() <= HALF_STEP[dt] * q_ref.abs() * (1 + 2.0 ** -6) + off).all()
    assert torch.equal(kv.scales.cpu().double(), s_ref)
    exact_k = norm == 0 and (rot is None or rot.dims == 0)
    for got, ahead, slack in ((kv.k, k_exact, 0.0 if exact_k else FP32_OFF), (kv.v, v_exact, 0.0)):
        got, near = got.cpu().double(), slack * ahead.abs().amax(-1, keepdim=True)
        lo, hi = U.to_codes(ahead - near), U.to_codes(ahead + near)
        assert ((got >= lo) & (got <= hi)).all()
    return kv, (k_ref, v_ref, s_ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,ps,H,G,d,dv,rot,norm", [
    ([(0, 1)], 64, 2, 1, 128, 128, ROT(128, 1), 0),                      # the first token of all
    ([(63, 1), (64, 1), (65, 1)], 64, 16, 2, 128, 128, ROT(128, 1), 3),    # the last row of a page, the first, the second
    ([(5, 1)] * 40, 16, 8, 8, 64, 64, ROT(32, 0), 1),                     # more portions than lanes
    ([(0, 200)], 64, 8, 2, 128, 128, ROT(64, 0), 0),
    ([(37, 150), (0, 1), (3, 77)], 64, 64, 8, 128, 128, ROT(128, 1), 1),
    ([(7, 30), (0, 5), (11, 64)], 7, 6, 2, 80, 80, ROT(40, 1), 3),         # odd pages, heads that are no whole vectors
    ([(1, 33)], 16, 7, 1, 96, 96, ROT(96, 0), 0),
    ([(10, 20)], 32, 4, 4, 64, 128, ROT(64, 1), 0),                       # values of another size
    ([(3, 300)], 256, 4, 2, 256, 256, ROT(256, 0), 1),                    # a page's rows do not fit in shared memory
    ([(2, 9), (0, 3)], 1, 3, 1, 24, 40, None, 0),                        # pages of one token
    ([(0, 0), (4, 6), (9, 0)], 8, 2, 2, 64, 64, ROT(64, 1), 0),            # portions without tokens
    ([(100000, 3)], 64, 2, 1, 128, 128, ROT(128, 1), 0),                 # a far position
])
def test_append(lens, ps, H, G, d, dv, rot, norm, dtype):
    run_append(lens, ps, H, G, d, dv, dtype, rot, norm, seed=len(lens) + d)


@pytest.mark.gpu
def test_append_reads_columns_anywhere_and_leaves_other_rows():
    run_append([(10, 20), (0, 3)], 16, 4, 2, 64, 64, "bf16", ROT(64, 1), 0, seed=3, gap=3, tail=5)      # (columns that begin at no whole vector; tokens of no portion)
    run_append([(10, 20), (0, 3)], 16, 4, 2, 128, 128, "fp32", ROT(128, 0), 3, seed=4, gap=8, tail=2)


@pytest.mark.gpu
@pytest.mark.parametrize("d,ps", [(128, 64), (80, 16), (30, 5)])
def test_append_moves_the_codes_of_a_page_whose_scale_grows(d, ps):
    grow = lambda T: torch.logspace(-3, 4, T)[:, None]
    lens = [(ps - 2, 1), (3, 1), (ps + 1, ps), (ps // 2, 2)]
    kv, ref = run_append(lens, ps, 4, 2, d, d, "fp32", None, 0, seed=11, scale=grow)
    # and again: what is there already asks for no larger scale, and the same tokens give the same codes
    again, _ = run_append(lens, ps, 4, 2, d, d, "fp32", None, 0, seed=11, scale=grow, times=3)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in ((kv.k, again.k), (kv.v, again.v))) and torch.equal(kv.scales, again.scales)


@pytest.mark.gpu
def test_append_of_nothing_and_of_everything():
    run_append([(0, 4), (6, 3)], 8, 2, 1, 64, 64, "fp32", ROT(64, 1), 0, scale=lambda T: torch.zeros(T, 1))
    run_append([(0, 4), (6, 3)], 8, 2, 1, 64, 64, "fp32", None, 0, scale=lambda T: torch.full((T, 1), 1e-30))
    run_append([(0, 4), (6, 3)], 8, 2, 1, 64, 64, "fp32", None, 0, scale=lambda T: torch.full((T, 1), 1e25))


@pytest.mark.gpu
def test_append_of_infinities_and_nan():
    batch, cache, total = U.batch_of([(0, 3), (0, 3)], 8)
    k, v, s = filled(total, 1, 8, 64, 64, 5)
    proj = torch.randn(6, 192)
    proj[1, 64], proj[1, 70], proj[1, 130] = math.inf, math.nan, -math.inf      # one key row and one value row of the first sequence
    kv = Fp8CacheLayer(*(x.cuda() for x in (k, v, s)))
    fp8_cache_append(proj.cuda(), on(batch), on(cache), kv, 1, 1, 64, 64, (0, 64, 128))
    _, k_ref, v_ref, s_ref, _, _ = U.append(proj, batch, cache, k, v, s, 1, 1, 64, 64, (0, 64, 128))
    assert torch.equal(kv.scales.cpu().double(), s_ref)
    assert torch.equal(kv.k.cpu().double().nan_to_num(1e9), k_ref.nan_to_num(1e9)) and torch.equal(kv.v.cpu().double(), v_ref)


@pytest.mark.gpu
def test_append_leaves_pages_that_are_not_there():
    batch, cache, total = U.batch_of([(4, 10), (0, 3)], 8)
    cache.page_table[0, 1], cache.page_table[1, 0] = total + 5, -1      # the first sequence's second page, the second's first
    k, v, s = filled(total, 2, 8, 64, 64, 6)
    kv = Fp8CacheLayer(*(x.cuda() for x in (k, v, s)))
    fp8_cache_append(torch.randn(13, 6 * 64).cuda(), on(batch), on(cache), kv, 2, 2, 64, 64, (0, 128, 256))
    changed = (kv.k.cpu().view(torch.uint8) != k.view(torch.uint8)).flatten(1).any(1)
    assert changed.nonzero().flatten().tolist() == [int(cache.page_table[0, 0])]


# ------------------------------------------------------------------------------------------------------------------------- attention
def run_attention(lens, ps, H, G, d, dv, dtype, seed=0, tail=0, wide=0, out_stride=0, tensor_cores=True, break_table=None, big=1.0, **o):
    g = torch.Generator().manual_seed(seed)
    batch, cache, total = U.batch_of(lens, ps, seed=seed, tail=tail)
    k, v, s = filled(total, G, ps, d, dv, seed, wide)
    live = torch.zeros((total, ps), dtype=torch.bool)      # rows behind a sequence's last token and pages of nobody: NaN
    for i, (b, n) in enumerate(lens):
        j = torch.arange(b + n)
        live[cache.page_table[i].long()[j // ps], j % ps] = True
    hole = ~live[:, None, :, None]
    k, v = (torch.where(hole, torch.full((), 0x7f, dtype=torch.uint8), x.view(torch.uint8)).view(U.E4M3) for x in (k, v))
    if break_table is not None:
        break_table(cache.page_table, total)
    T, dt = batch.pos.shape[0], DT[dtype]
    q = (big * torch.randn((T, H, d), generator=g)).to(dt)
    scale = d ** -0.5
    for name in ("head_scale", "sink"):
        if o.get(name):
            o[name] = torch.randn(H, generator=g) * (0.3 if name == "head_scale" else 1.0) + (1.0 if name == "head_scale" else 0.0)
    ref = U.attention(q, k, v, s, batch, cache, H, G, d, dv, scale, **o)
    kv = Fp8CacheLayer(*(x.cuda() for x in (k, v, s)))
    wide_out = torch.full((T, H * dv + out_stride), 7.0, dtype=dt, device="cuda")
    out = fp8_cache_attention(q.cuda(), kv, on(batch), on(cache), H, G, d, dv, scale, tensor_cores=tensor_cores, out=wide_out[:, :H * dv], **{n: on(x) for n, x in o.items()}).cpu().double()
    assert (wide_out[:, H * dv:] == 7).all()
    alone = ref.isnan()
    assert (out[alone] == 7).all()      # tokens of no portion
    # scores are sums of d products, off by d x 2^-24 of |q||k| in fp32 and twice that on the tensor cores (which cut what a sum does not hold); a score's error e makes its weight's
    # relative error e, at most 2 e of the weighted mean of values of size V.  Weights rounded to fp16 for the second product: 2^-11 of V
    K = (k.double().nan_to_num(0.0) * s.double()[:, :, None, None, 0]).norm(dim=-1).max()
    V = (v.double().nan_to_num(0.0) * s.double()[:, :, None, None, 1]).abs().max()
    hs = o["head_scale"].abs().max() if o.get("head_scale") is not None else 1.0
    e = float(q.double().norm(dim=-1).max() * K * scale * hs) * (2 * d + 8) * 2.0 ** -24 + 2.0 ** -20
    bound = HALF_STEP[dt] * ref.abs() * 1.02 + float(V) * (2 * e + (2.0 ** -11 if dtype == "bf16" else 0.0)) * abs(o.get("out_scale", 1.0))
    assert ((out - ref).abs() <= bound)[~alone].all(), float(((out - ref).abs() / bound)[~alone].max())


SHAPES = [
    ([(0, 1)], 64, 2, 1, 128, 128),                                   # the first token sees itself alone
    ([(62, 1), (63, 1), (64, 1), (200, 1)], 64, 16, 2, 128, 128),
    ([(1500, 1)], 64, 16, 2, 128, 128),                               # one token over a range that is cut
    ([(333, 1), (5, 1), (90, 1)], 48, 8, 8, 64, 64),                  # pages that are no whole tiles, heads that share nothing
    ([(100, 3), (0, 5), (17, 1)], 16, 12, 4, 96, 96),
    ([(100, 3), (0, 5)], 7, 6, 2, 80, 48),
    ([(70, 2)], 64, 7, 1, 64, 128),
    ([(30, 2)], 32, 32, 1, 64, 64),
    ([(40, 4)], 16, 2, 1, 40, 24),                                    # head sizes that no tensor-core tile takes
    ([(20, 2)], 16, 2, 2, 256, 256),
    ([(0, 70), (33, 40), (500, 1)], 64, 8, 1, 128, 128),              # prompt portions beside a decoded token
    ([(10, 100)], 64, 16, 2, 128, 128),
    ([(3, 0), (9, 20), (0, 0)], 16, 4, 2, 64, 64),                    # portions without tokens
    ([(6, 40)], 5, 4, 2, 128, 64),
    ([(130, 200)], 64, 3, 1, 128, 128),                               # rows that a tile's tokens do not fill
    ([(2000, 20)], 64, 16, 1, 128, 128),                              # a short portion over a range that is cut
    ([(9, 150), (0, 64)], 128, 2, 2, 128, 128),
    ([(500, 1), (3, 1), (129, 1)], 16, 12, 2, 128, 128),
    ([(1400, 1), (900, 1), (0, 1), (300, 1), (511, 1)], 64, 4, 2, 128, 128),
    ([(9000, 1)], 64, 2, 1, 128, 128),
    ([(1400, 1), (901, 1), (0, 1), (300, 1), (511, 1)], 32, 16, 1, 64, 64),
    ([(9001, 1)], 16, 2, 1, 64, 64),
    ([(700, 1), (33, 1)], 80, 12, 1, 64, 64),
    ([(500, 1), (3, 1)], 48, 34, 2, 128, 128),                        # a group that no run of 16 heads divides
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,ps,H,G,d,dv", SHAPES)
def test_attention(lens, ps, H, G, d, dv, dtype):
    run_attention(lens, ps, H, G, d, dv, dtype, seed=d + len(lens))


MASKS = [dict(window=1), dict(window=50), dict(chunk=16), dict(chunk=33, sink=True), dict(window=20, chunk=64, softcap=20.0), dict(head_scale=True, softcap=5.0), dict(sink=True, out_scale=0.25), dict(out_scale=-2.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("options", MASKS, ids=str)
def test_attention_masks_and_scores(options, dtype):
    run_attention([(100, 1), (0, 40), (31, 33), (700, 2)], 32, 8, 2, 128, 128, dtype, seed=5, **options)
    run_attention([(100, 1), (0, 4), (31, 3)], 48, 6, 2, 96, 64, dtype, seed=6, **options)
    run_attention([(150, 40), (0, 140), (600, 3)], 64, 8, 2, 128, 128, dtype, seed=7, **options)
    run_attention([(200, 1), (0, 1), (1300, 1)], 64, 16, 1, 128, 128, dtype, seed=7, **options)
    run_attention([(201, 1), (0, 1), (1300, 1)], 64, 8, 1, 64, 64, dtype, seed=7, **options)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_blocks_of_very_different_scales(dtype):
    run_attention([(400, 1), (90, 5)], 16, 4, 1, 64, 64, dtype, seed=8, wide=5)
    run_attention([(700, 1), (300, 1)], 64, 4, 1, 128, 128, dtype, seed=8, wide=5)
    run_attention([(700, 1), (301, 1)], 64, 4, 1, 64, 64, dtype, seed=8, wide=5)
    run_attention([(300, 40)], 64, 4, 1, 128, 128, dtype, seed=8, wide=5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_writes_its_rows_alone(dtype):
    run_attention([(100, 3), (0, 20)], 16, 4, 2, 64, 64, dtype, seed=9, tail=4, out_stride=24)
    run_attention([(900, 1)], 16, 4, 2, 64, 64, dtype, seed=9, tail=2, out_stride=8)
    run_attention([(90, 2)], 16, 4, 2, 64, 64, dtype, seed=9, out_stride=3)      # rows that begin anywhere
    run_attention([(90, 70)], 64, 4, 2, 128, 128, dtype, seed=9, tail=3, out_stride=3)
    run_attention([(990, 1)], 64, 4, 2, 128, 128, dtype, seed=9, tail=1, out_stride=5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_does_not_see_pages_that_are_not_there(dtype):
    def break_table(t, total):
        t[0, 1], t[1, 0] = total, -3
    run_attention([(100, 2), (0, 3), (60, 40)], 16, 4, 2, 64, 64, dtype, seed=10, break_table=break_table)      # (the second sequence sees nothing at all: zeros)
    run_attention([(1200, 1)], 64, 4, 2, 128, 128, dtype, seed=10, break_table=lambda t, total: t.__setitem__((0, 3), -1))
    run_attention([(1200, 1)], 16, 4, 2, 64, 64, dtype, seed=10, break_table=lambda t, total: t.__setitem__((0, 3), -1))


@pytest.mark.gpu
@pytest.mark.parametrize("d,lens", [(128, [(1500, 1), (300, 1)]), (64, [(1500, 1), (300, 1)]), (128, [(700, 40), (0, 90)])])
def test_attention_cut_and_uncut_agree(d, lens):
    """the caller's parts, the library's own cut, and none"""
    H, G, lib = 8, 2, native.seq_lib()
    batch, cache, total = U.batch_of(lens, 64, seed=2)
    batch, cache, T = on(batch), on(cache), batch.pos.shape[0]
    kv = Fp8CacheLayer(*(x.cuda() for x in filled(total, G, 64, d, d, 2)))
    q, outs = torch.randn((T, H, d), generator=torch.Generator().manual_seed(2)).bfloat16().cuda(), []
    for part in (-1, 0, 128, 384, 1024):
        out = torch.zeros((T, H * d), dtype=torch.bfloat16, device="cuda")
        a = native.Fp8AttnParams(q.data_ptr(), H, G, d, d, d ** -0.5, None, 0.0, 0, 0, None, 1.0, batch.pos.data_ptr(), batch.slot.data_ptr(), batch.seqs.data_ptr(), batch.seqs.stride(0), batch.n_seqs,
                                 cache.page_table.data_ptr(), cache.page_table.shape[0], cache.page_table.shape[1], 64, total, kv.k.data_ptr(), kv.v.data_ptr(), kv.scales.data_ptr(), out.data_ptr(), H * d)
        n = lib.ktb200_fp8_cache_attn_workspace(C.byref(a), T, batch.max_kv, part, native.GGML_BF16, 1)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        native.check_seq(lib.ktb200_fp8_cache_attn(C.byref(a), T, batch.max_kv, part, ws.data_ptr() if n else None, n, native.GGML_BF16, 1, torch.cuda.current_stream().cuda_stream))
        outs.append(out.float())
    # weights and results round to 8 bits on either way (2^-8 of a value each)
    assert all(((o - outs[1]).abs() <= 2.0 ** -7 * outs[1].abs() + 2.0 ** -8 * float(kv.dequantize()[1].abs().max())).all() for o in outs) and outs[1].abs().max() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_over_a_ring_of_pages(dtype):
    """positions far beyond the table's width: logical page p stands in column p % max_pages"""
    batch, cache, total = U.batch_of([(40, 3)], 16)
    lap = cache.max_pages_per_seq * 16
    k, v, s = filled(total, 1, 16, 64, 64, 12)
    q = torch.randn(3, 2, 64).to(DT[dtype])
    kv = Fp8CacheLayer(*(x.cuda() for x in (k, v, s)))
    a = fp8_cache_attention(q.cuda(), kv, on(batch), on(cache), 2, 1, 64, 64, 0.125, window=30)
    batch.pos += 5 * lap
    batch.max_kv += 5 * lap
    b = fp8_cache_attention(q.cuda(), kv, on(batch), on(cache), 2, 1, 64, 64, 0.125, window=30)
    assert torch.allclose(a.float(), b.float(), rtol=0, atol=float(a.float().abs().max()) * (2.0 ** -7 if dtype == "bf16" else 1e-5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d,ps,lens,at", [(128, 64, [(0, 90)], 50), (128, 64, [(0, 20)], 11), (64, 16, [(20, 3)], 21), (96, 48, [(5, 40)], 44), (128, 64, [(200, 300)], 260)])
def test_attention_keeps_nan_to_the_rows_that_see_it(d, ps, lens, at, dtype):
    """a token whose key (or value) is NaN: the tokens ahead of it do not see it, those behind it do"""
    H, G, (b, n) = 4, 2, lens[0]
    batch, cache, total = U.batch_of(lens, ps)
    page, row = int(cache.page_table[0, at // ps]), at % ps
    for what in ("k", "v"):
        kv = Fp8CacheLayer(*(x.cuda() for x in filled(total, G, ps, d, d, 13)))
        q = torch.randn((n, H, d), generator=torch.Generator().manual_seed(1)).to(DT[dtype]).cuda()
        clean = fp8_cache_attention(q, kv, on(batch), on(cache), H, G, d, d, d ** -0.5).view(n, H, d)
        getattr(kv, what).view(torch.uint8)[page, 1, row, 5] = 0x7f if what == "k" else 0xff      # the second key/value head's
        out = fp8_cache_attention(q, kv, on(batch), on(cache), H, G, d, d, d ** -0.5).view(n, H, d)
        first = at - b
        assert torch.equal(out[:, :2], clean[:, :2]) and torch.equal(out[:first, 2:], clean[:first, 2:])
        if what == "k":
            assert out[first:, 2:].isnan().all()
        else:
            assert out[first:, 2:, 5].isnan().all() and not out[first:, 2:, 6:].isnan().any()
            for more in range(at, min(at + 9, b + n), 2):      # whole tokens of them
                kv.v.view(torch.uint8)[int(cache.page_table[0, more // ps]), 1, more % ps] = 0x7f
            out = fp8_cache_attention(q, kv, on(batch), on(cache), H, G, d, d, d ** -0.5).view(n, H, d)
            assert torch.equal(out[:first, 2:], clean[:first, 2:]) and out[first:, 2:].isnan().all()


@pytest.mark.gpu
def test_the_two_calls_as_a_step_uses_them_replayed_on_other_streams():
    """append, then attention over what was appended, decoded token by token behind a prompt: eagerly, and as one captured graph per step"""
    H, G, d, ps, steps = 8, 2, 128, 64, 5
    lens = [(0, 70), (0, 63), (0, 9)]
    full, cache, total = U.batch_of([(0, n + steps) for _, n in lens], ps)
    g = torch.Generator().manual_seed(3)
    rows = [torch.randn((n + steps, (H + 2 * G) * d), generator=g).bfloat16().cuda() for _, n in lens]
    rot, inv = ROT(d, 1), INV(d).cuda()
    cache = on(cache)

    def batch_at(done, n):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        pos = [p for s in range(3) for p in range(done[s], done[s] + n[s])]
        starts = [sum(n[:s]) for s in range(3)]
        return SimpleNamespace(pos=i32(pos), slot=i32([s for s in range(3) for _ in range(n[s])]), seqs=i32([starts, n]), n_seqs=3, max_kv=max(x + y for x, y in zip(done, n)))

    def step(kv, b, proj):
        q = fp8_cache_append(proj, b, cache, kv, H, G, d, d, (0, H * d, (H + G) * d), rot, inv, 1, 1e-6)
        return fp8_cache_attention(q, kv, b, cache, H, G, d, d, d ** -0.5)

    def serve(captured):
        kv = Fp8CacheLayer.empty(total, ps, G, d, d)
        n = [x for _, x in lens]
        outs = [step(kv, batch_at([0, 0, 0], n), torch.cat([r[:m] for r, m in zip(rows, n)]))]
        b, proj, graph, side = batch_at(n, [1, 1, 1]), torch.empty_like(rows[0][:3]), None, torch.cuda.Stream()
        b.max_kv = 64 * ps
        for i in range(steps):
            b.pos.copy_(torch.tensor([x + i for x in n], dtype=torch.int32))
            proj.copy_(torch.stack([r[x + i] for r, x in zip(rows, n)]))
            if not captured:
                outs.append(step(kv, b, proj))
                continue
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    o = step(kv, b, proj)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            torch.cuda.current_stream().wait_stream(side)
            outs.append(o.clone())
        torch.cuda.synchronize()
        return outs, kv

    (eager, a), (replayed, c) = serve(False), serve(True)
    assert all(torch.equal(x, y) for x, y in zip(eager, replayed))
    assert torch.equal(a.k.view(torch.uint8), c.k.view(torch.uint8)) and torch.equal(a.scales, c.scales)
    # the last decoded tokens against attention over all of a sequence's tokens in 64 bits, over what the cache holds
    b = batch_at([n + steps - 1 for _, n in lens], [1, 1, 1])
    proj = torch.stack([r[-1] for r in rows])
    q, *_ = U.append(proj.cpu(), on(b, "cpu"), on(cache, "cpu"), a.k.cpu(), a.v.cpu(), a.scales.cpu(), H, G, d, d, (0, H * d, (H + G) * d), rot, inv.cpu(), 1, 1e-6)
    ref = U.attention(q.bfloat16(), a.k.cpu(), a.v.cpu(), a.scales.cpu(), on(b, "cpu"), on(cache, "cpu"), H, G, d, d, d ** -0.5)
    # queries round as bf16 on both sides (one step apart at most: 2^-7 of a score of size s, s <= 5 here), weights to fp16, results to bf16
    assert ((eager[-1].cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -4 + 2.0 ** -11) * float(a.dequantize()[1].abs().max())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("dim,page,chunk", [(128, 64, 4096), (32, 16, 40)])
def test_an_attention_layer_on_an_8_bit_cache(dim, page, chunk, dtype):
    """KPlusOneAttention through the cache manager, a prompt in portions and decoded tokens, against the 64-bit forms on the same projections"""
    from ktransformers_b200.models.configuration_lipadra import PlusOneAttentionSpec
    from ktransformers_b200.operators.attention import KPlusOneAttention
    H, G, dt = 4, 2, DT[dtype]
    spec = PlusOneAttentionSpec.from_dict({"heads": H, "kv_heads": G, "dim": dim, "vdim": dim, "mask": {"size": chunk}, "rot": {"base": 1000.0, "dims": dim}})
    width, g = H * dim, torch.Generator().manual_seed(4)
    layer = KPlusOneAttention(width, spec, 1e-5, dtype=dt, device="cuda")
    rn = lambda *shape: torch.randn(shape, generator=g)
    layer.w_in.data.copy_(rn(*layer.w_in.shape) / width ** 0.5)
    layer.b_in.data.copy_(0.1 * rn(layer.n_in))
    layer.q_norm.data.copy_(1 + 0.2 * rn(dim))
    layer.k_norm.data.copy_(1 + 0.2 * rn(dim))
    layer.o.data.copy_(torch.eye(width))      # (the layer's result is then the attention's)
    c = PagedStateCache([spec.cache_row_width()], 0, 512, 2, "cuda", dtype=dt, page_size=page, chunks=[chunk], fp8_heads=[(G, dim, dim)])
    held = c.key_cache[0]
    k, v, s = (x.cpu() for x in (held.k, held.v, held.scales))
    offs = (0, H * dim, (H + G) * dim)
    for step in ([("a", 70), ("b", 9)], [("a", 33), ("b", 1)], [("a", 1), ("b", 1)], [("b", 40)], [("a", 1), ("b", 1)]):
        batch = c.build_batch([(name, [0] * n, []) for name, n in step])
        h = rn(batch.n_tokens, width).to(dt).cuda()
        out = layer(h, batch, c, 0).cpu().double()
        c.commit()
        proj = torch.nn.functional.linear(h, layer.w_in, layer.b_in).cpu()
        cpu = SimpleNamespace(pos=batch.pos.cpu(), slot=batch.slot.cpu(), seqs=batch.seqs.cpu(), n_seqs=batch.n_seqs)
        table = SimpleNamespace(page_table=c.page_table.cpu(), max_pages_per_seq=c.max_pages_per_seq, page_size=page)
        inv = layer.inv_freq.cpu()
        q, *_ = U.append(proj, cpu, table, k, v, s, H, G, dim, dim, offs, spec.rot, inv, 3, 1e-5, layer.q_norm.cpu(), layer.k_norm.cpu())
        k, v, s = held.k.cpu(), held.v.cpu(), held.scales.cpu()      # (what the cache holds is tested with the append)
        ref = U.attention(q.to(dt), k, v, s, cpu, table, H, G, dim, dim, spec.scale, chunk=chunk, sink=torch.zeros(H))
        # queries may round to the other side (a step of 2^-7 in bf16, 2^-20 for the fp32 rotation and norm) in scores below 32; weights to fp16; the result and the product with one to the type
        top = float((v.double() * s.double()[:, :, None, None, 1]).nan_to_num(0.0).abs().max())
        off = {"bf16": 2 * (2.0 ** -7 * 6 + 2.0 ** -11), "fp32": 2 * 32 * 2.0 ** -18}[dtype]
        assert ((out - ref).abs() <= 2 * HALF_STEP[dt] * ref.abs() * 1.02 + off * top).all()


@pytest.mark.gpu
def test_a_model_served_from_an_8_bit_cache(tmp_path):
    """the engine's prompt portions, decode steps and captured decode steps on an 8-bit cache: the same tokens whichever way"""
    import lipadra_util as LU
    from ktransformers_b200.models import load_model
    from ktransformers_b200.util.engine import Engine
    cfg = LU.config([(LU.attention(heads=4, kv_heads=2, dim=128, vdim=128, chunk=256, dims=128), LU.moe()), (LU.retention(), None), (LU.attention(heads=4, kv_heads=2, dim=16, vdim=16, chunk=32, dims=16), None)])
    path = LU.save(tmp_path / "m", cfg, LU.weights(cfg, dtype=torch.bfloat16))
    model = load_model(path, "bfloat16")
    prompts = [[(7 * i + j) % 50 for j in range(n)] for i, n in enumerate((90, 3, 41))]
    outs = [Engine(model, max_tokens=1024, page_size=64, max_step_tokens=step, cuda_graphs=graphs, kv_cache="fp8").generate(prompts, 12) for step, graphs in ((2048, False), (2048, True))]
    assert outs[0] == outs[1] and all(len(o) == 12 for o in outs[0])
    eng = Engine(model, max_tokens=1024, page_size=64, kv_cache="fp8")
    assert isinstance(eng.cache.key_cache[0], Fp8CacheLayer) and isinstance(eng.cache.key_cache[2], Fp8CacheLayer)
    logits = eng.step([("x", prompts[0], [89])])
    plain = Engine(model, max_tokens=1024, page_size=64).step([("x", prompts[0], [89])])
    assert logits.shape == plain.shape and torch.isfinite(logits).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d,ps,base,window", [(128, 64, 300, 0), (128, 64, 300, 77), (64, 16, 301, 0), (64, 16, 300, 0), (64, 64, 300, 78), (64, 64, 1300, 77), (96, 16, 300, 77)])
def test_attention_of_one_token_is_free_of_what_it_does_not_see(d, ps, base, window, dtype):
    """NaN in all codes ahead of a window and behind the token, the seen keys' neighbours among them: the same result"""
    H, G = 4, 2
    batch, cache, total = U.batch_of([(base, 1)], ps)
    kv = Fp8CacheLayer(*(x.cuda() for x in filled(total, G, ps, d, d, 14)))
    q = torch.randn((1, H, d), generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
    clean = fp8_cache_attention(q, kv, on(batch), on(cache), H, G, d, d, d ** -0.5, window=window)
    keep = torch.zeros((total, ps), dtype=torch.bool)
    for key in range(max(0, base + 1 - window) if window else 0, base + 1):
        keep[int(cache.page_table[0, key // ps]), key % ps] = True
    for x in (kv.k, kv.v):
        x.view(torch.uint8)[(~keep).cuda()[:, None, :, None].expand(total, G, ps, d)] = 0x7f
    out = fp8_cache_attention(q, kv, on(batch), on(cache), H, G, d, d, d ** -0.5, window=window)
    assert torch.equal(out, clean) and clean.isfinite().all() and float(clean.abs().max()) > 0


RotDims = lambda dims: SimpleNamespace(dims=dims, layout_code=0)


@pytest.mark.gpu
def test_wrappers_refuse_what_does_not_fit():
    H, G, d, ps = 4, 2, 64, 16
    batch, cache, total = U.batch_of([(20, 3)], ps)
    batch, cache = on(batch), on(cache)
    kv = Fp8CacheLayer.empty(total, ps, G, d, d, "cuda")
    proj, q = torch.zeros(3, (H + 2 * G) * d, device="cuda"), torch.zeros(3, H, d, device="cuda")
    n, offsets = H * d, (0, H * d, (H + G) * d)
    append = lambda rows=proj, b=batch, c=cache, layer=kv, at=offsets, kv_heads=G, **o: fp8_cache_append(rows, b, c, layer, H, kv_heads, d, d, at, **o)
    attend = lambda rows=q, b=batch, c=cache, layer=kv, kv_heads=G, dim=d, **o: fp8_cache_attention(rows, layer, b, c, H, kv_heads, dim, d, 1.0, **o)
    assert append().shape == (3, H, d) and attend().shape == (3, n)
    swap = lambda x, **o: SimpleNamespace(**{**{k: getattr(x, k) for k in ("pos", "slot", "seqs", "n_seqs", "max_kv", "page_table", "page_size", "max_pages_per_seq") if hasattr(x, k)}, **o})
    for f in (append, attend):
        for o in (dict(kv_heads=1), dict(layer=Fp8CacheLayer.empty(total, 2 * ps, G, d, d, "cuda")), dict(layer=Fp8CacheLayer.empty(total, ps, G, 32, d, "cuda")),
                  dict(layer=Fp8CacheLayer.empty(total, ps, G, d, d, "cpu")), dict(b=swap(batch, pos=batch.pos.long())), dict(b=swap(batch, pos=batch.pos[:2])), dict(b=swap(batch, slot=batch.slot[:1])),
                  dict(b=swap(batch, seqs=None)), dict(b=swap(batch, seqs=batch.seqs[:1])), dict(b=swap(batch, n_seqs=batch.seqs.shape[1] + 1)), dict(b=swap(batch, pos=batch.pos.cpu())),
                  dict(c=swap(cache, page_table=cache.page_table.long())), dict(c=swap(cache, max_pages_per_seq=cache.max_pages_per_seq + 1))):
            with pytest.raises(ValueError, match="fp8_cache"):
                f(**o)
    freq = torch.ones(4, dtype=torch.float64, device="cuda")
    for o in (dict(at=(0, n, n + 1 + G * d)), dict(at=(-1, n, n + G * d)), dict(rows=proj.half()), dict(rows=proj.t()), dict(rot=RotDims(8)), dict(rot=RotDims(8), inv_freq=freq[:3]),
              dict(rot=RotDims(8), inv_freq=freq.float()), dict(qk_norm=3), dict(qk_norm=3, q_weight=q[0, 0], k_weight=q[0, 0, :5])):
        with pytest.raises(ValueError, match="fp8_cache_append"):
            append(**o)
    row = torch.zeros(H, device="cuda")
    for o in (dict(rows=q[:, :2]), dict(rows=q.transpose(1, 2)), dict(rows=q.half()), dict(head_scale=row[:3]), dict(head_scale=row.double()), dict(sink=row.cpu()),
              dict(out=torch.zeros(3, n - 1, device="cuda")), dict(out=torch.zeros(3, n, device="cuda").half()), dict(out=torch.zeros(n, 3, device="cuda").t())):
        with pytest.raises(ValueError, match="fp8_cache_attention"):
            attend(**o)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp32", 64), ("bf16", 48)])
@pytest.mark.parametrize("before,n", [(20, 100), (0, 65), (63, 300)])
def test_append_of_a_portion_longer_than_the_ring(before, n, dtype, d):
    """its last pages are what stays, each time"""
    H, G, ps, columns = 4, 2, 16, 4
    pool = filled(columns + 1, G, ps, d, d, 3)
    proj = torch.randn((n, (H + 2 * G) * d), generator=torch.Generator().manual_seed(n)).to(DT[dtype]).cuda()
    cache = on(SimpleNamespace(page_table=torch.tensor([[3, 0, 4, 1]], dtype=torch.int32), max_pages_per_seq=columns, page_size=ps))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)

    def append(start):      # the portion's tokens from row `start` on
        m = n - start
        batch = on(SimpleNamespace(pos=torch.arange(before, before + n, dtype=torch.int32), slot=i32([0] * n), seqs=i32([[start], [m], [0], [0]]), n_seqs=1, max_kv=before + n))
        kv = Fp8CacheLayer(*(x.cuda() for x in pool))
        q = fp8_cache_append(proj, batch, cache, kv, H, G, d, d, (0, H * d, (H + G) * d), qk_norm=1)
        return [q] + [x.view(torch.uint8) if x.dtype is U.E4M3 else x for x in (kv.k, kv.v, kv.scales)]
    first = ((before + n - 1) // ps - columns + 1) * ps - before      # the row at which the last pages begin
    assert first > 0
    want = append(first)
    for _ in range(5):
        assert all(torch.equal(x, y) for x, y in zip(append(0), want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,lens", [("bf16", 128, [(900, 1), (70, 1)]), ("bf16", 64, [(900, 1)]), ("bf16", 128, [(300, 90)]), ("bf16", 96, [(300, 5)]), ("fp32", 128, [(300, 5)])])
def test_both_calls_beyond_four_gigabytes(dtype, d, lens):
    """the same blocks at the end of a pool whose offsets pass 32 bits: the same results"""
    H, G, ps = 8, 2, 64
    batch, cache, total = U.batch_of(lens, ps, seed=4)
    far = (1 << 32) // (G * ps * d) + 5
    T = batch.pos.shape[0]
    proj = torch.randn((T, (H + 2 * G) * d), generator=torch.Generator().manual_seed(5)).to(DT[dtype]).cuda()
    near = Fp8CacheLayer(*(x.cuda() for x in filled(total, G, ps, d, d, 15)))
    codes = lambda x: torch.cat([torch.empty((far, G, ps, d), dtype=torch.uint8, device="cuda"), x.view(torch.uint8)]).view(U.E4M3)
    away = Fp8CacheLayer(codes(near.k), codes(near.v), torch.cat([torch.ones((far, G, 2), device="cuda"), near.scales]))
    there = SimpleNamespace(**{**vars(cache), "page_table": cache.page_table + far})
    outs = []
    for kv, c in ((near, cache), (away, there)):
        q = fp8_cache_append(proj, on(batch), on(c), kv, H, G, d, d, (0, H * d, (H + G) * d), qk_norm=1)
        outs.append([q, fp8_cache_attention(q, kv, on(batch), on(c), H, G, d, d, d ** -0.5)] + [x[-total:].view(torch.uint8) for x in (kv.k, kv.v)] + [kv.scales[-total:]])
    assert all(torch.equal(x, y) for x, y in zip(*outs)) and outs[0][1].isfinite().all()
