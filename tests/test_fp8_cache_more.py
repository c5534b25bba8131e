"""The paged e4m3 cache, beside test_fp8_cache.py: waits, single keys with most of the weight, infinite sinks, refusals."""
import math
from types import SimpleNamespace

import pytest
import torch

import fp8_cache_util as U
from ktransformers_b200.models.custom_cache import Fp8CacheLayer
from ktransformers_b200.operators.attention import fp8_cache_append, fp8_cache_attention

on = lambda x, device="cuda": SimpleNamespace(**{k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in vars(x).items()})


def layer(total, G, ps, d, seed, device="cuda"):
    """codes of normal numbers under scales of 2^-7"""
    g = torch.Generator().manual_seed(seed)
    codes = lambda: (torch.randn((total, G, ps, d), generator=g) * 128).clamp(-448, 448).to(U.E4M3).to(device)      # (what is larger would become NaN)
    return Fp8CacheLayer(codes(), codes(), torch.full((total, G, 2), 2.0 ** -7, device=device))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,G", [([(0, 64)], 1, 1), ([(0, 128)], 16, 2), ([(100, 70)], 8, 1), ([(128, 256)], 8, 2), ([(300, 90), (0, 200)], 12, 2), ([(1000, 128)], 16, 1), ([(2000, 130)], 5, 1)])
def test_prompt_attention_never_waits_for_a_phase_that_has_gone(lens, H, G):
    """One to seventeen key tiles, whole and cut: a wait that cannot end gives up after 16 ms at least, 50 calls take less than that; and all give the same bits"""
    d, ps, calls = 128, 64, 50
    batch, cache, total = U.batch_of(lens, ps, seed=1)
    batch, cache, kv = on(batch), on(cache), layer(total, G, ps, d, 1)
    q = torch.randn((batch.pos.shape[0], H, d), generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    first = fp8_cache_attention(q, kv, batch, cache, H, G, d, d, d ** -0.5)
    torch.cuda.synchronize()
    graph, outs = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        for _ in range(calls):
            outs.append(fp8_cache_attention(q, kv, batch, cache, H, G, d, d, d ** -0.5))
    graph.replay()
    for _ in range(4):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        assert begin.elapsed_time(end) < 15.0
        assert all(torch.equal(first, o) for o in outs)


def farthest(out, q, k, v, s, batch, cache, lens, scale, weight, floor, query, wide=1.0):
    """(largest distance of out [T, H, d] from attention in 64 bits, in bounds; the rows' largest weights); all on the CPU.  weight, floor: how far a weight may be off, of itself, and of the
    row's largest; query: how far a query's column, of the row's largest; wide: the largest value scale over the smallest"""
    half, worst, seen, (_, G, ps, d), H = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[q.dtype], 0.0, [], k.shape, q.shape[1]
    for i, (b, n) in enumerate(lens):
        j = torch.arange(b + n)
        page = cache.page_table[i].long()[j // ps]
        for h in range(G):
            K, V = (x[page, h, j % ps].double() * s[page, h, c, None].double() for c, x in ((0, k), (1, v)))
            for t in range(n):
                at_t, rows = b + t + 1, q[int(batch.seqs[0, i]) + t].double().reshape(G, H // G, d)[h]
                w = torch.softmax(rows @ K[:at_t].T * scale, 1)
                ref, spread = w @ V[:at_t], w @ V[:at_t].abs()
                # scores are fp32 sums of d products of queries that are `query` of a row's largest off at most; an error e of them makes weights 2 e off
                e = float(rows.norm(dim=1).max() * K[:at_t].norm(dim=1).max() * scale) * (2 * d + 8) * 2.0 ** -24 + float(rows.abs().max() * K[:at_t].abs().sum(1).max()) * scale * query + 2.0 ** -20
                bound = half * ref.abs() * 1.02 + (weight + 2 * e) * spread * 1.02 + floor * w.amax(1, keepdim=True) * wide * V[:at_t].abs().sum(0)
                got = out[int(batch.seqs[0, i]) + t].reshape(G, H // G, d)[h]
                worst = max(worst, float(((got - ref).abs() / bound).max()))
                seen.append(float(w.amax(1).max()))
    return worst, seen


def run_dominant(lens, ps, H, G, d, dtype, gap, at, equal, wide=0, weight=2.0 ** -8, floor=2.0 ** -35, query=2.0 ** -21, big=1.0, seed=0):
    """One key (gap: None, no such key) with most of every row's weight and a value of zero: what is left is the sum of all the others' small weights, compared with 64 bits relative to that sum.
    at: the key, a share of the first token's range.  gap: by how many nats its score is above the others' mean, about.  equal: the others have one score.  wide: 2^wide is the value
    scale of its page, beside one for the others.  weight, floor, query: as in `farthest`.  big: the size of the queries"""
    g = torch.Generator().manual_seed(seed)
    batch, cache, total = U.batch_of(lens, ps, seed=seed)
    T, dt, scale = batch.pos.shape[0], {"bf16": torch.bfloat16, "fp32": torch.float32}[dtype], d ** -0.5
    q = (big * torch.randn((T, H, d), generator=g)).to(dt)
    for i, (_, n) in enumerate(lens):      # a portion's tokens look the same way
        if n > 1:
            t = int(batch.seqs[0, i])
            q[t + 1:t + n] = q[t] + (0.1 * q[t + 1:t + n].float()).to(dt)
    codes = lambda x: x.clamp(-448, 448).to(U.E4M3)
    k = codes(torch.zeros((total, G, ps, d)) if equal else 16 * torch.randn((total, G, ps, d), generator=g))
    v = codes(16 + 4 * torch.randn((total, G, ps, d), generator=g))
    s = torch.full((total, G, 2), 2.0 ** -4)
    for i, (b, n) in enumerate(lens if gap is not None else []):
        key, rows = int(at * b), q[int(batch.seqs[0, i]):int(batch.seqs[0, i]) + n].double().reshape(n, G, H // G, d)
        page = int(cache.page_table[i, key // ps])
        # along the first token's queries of the group: each head's score is about its own |q|^2 of it
        k[page, :, key % ps] = codes((16 * gap / d ** 0.5 * rows[0].sum(1)).float())
        v[page, :, key % ps] = codes(torch.zeros(G, d))
        s[page, :, 1] *= 2.0 ** wide
    kv = Fp8CacheLayer(k.cuda(), v.cuda(), s.cuda())
    out = fp8_cache_attention(q.cuda(), kv, on(batch), on(cache), H, G, d, d, scale).cpu().double().reshape(T, H, d)
    worst, seen = farthest(out, q, k, v, s, batch, cache, lens, scale, weight, floor, query, 2.0 ** max(0, wide))
    assert gap is None or max(seen) > 0.9      # (the key does have most of the weight)
    assert worst <= 1, worst


DOMINANT = [
    ([(15999, 1)], 64, 16, 2, 128, 12), ([(60000, 1)], 64, 4, 1, 128, 14), ([(15999, 1)], 16, 4, 1, 64, 12), ([(59999, 1)], 64, 4, 1, 64, 14), ([(8000, 1)], 32, 16, 1, 128, 14),
    ([(700, 1), (90, 1), (64, 1)], 64, 8, 1, 128, 8), ([(700, 1), (90, 1), (64, 1)], 16, 8, 1, 64, 8), ([(2000, 1)] * 3, 64, 16, 1, 128, 18),
]


@pytest.mark.gpu
@pytest.mark.parametrize("equal", [False, True])
@pytest.mark.parametrize("at", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("lens,ps,H,G,d,gap", DOMINANT)
def test_single_tokens_keep_the_weights_beside_a_dominant_key(lens, ps, H, G, d, gap, at, equal):
    run_dominant(lens, ps, H, G, d, "bf16", gap, at, equal)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_single_tokens_keep_the_weights_beside_a_dominant_key_of_a_page_of_large_values(d):
    run_dominant([(15999, 1)], 64, 4, 1, d, "bf16", 14, 0.0, True, wide=5)
    run_dominant([(500, 1), (2000, 1)], 64, 4, 1, d, "bf16", 8, 1.0, False, wide=5)


# fp16 weights: a step of 2^-24 beside a largest of 2^7 at least.  Prompt queries are two numbers of one scale, 2^-17 of a row's largest off
SEVERAL = [
    ([(15999, 1)], 64, 8, 2, 96, "bf16", 12), ([(12000, 2)], 20, 4, 1, 80, "bf16", 14), ([(15998, 4)], 64, 8, 2, 128, "bf16", 14), ([(3000, 40)], 32, 4, 1, 128, "bf16", 12), ([(700, 1), (90, 2)], 48, 6, 2, 96, "bf16", 9),
    ([(8000, 40)], 64, 8, 2, 128, "bf16", 13), ([(4000, 130)], 64, 16, 1, 128, "bf16", 14), ([(64, 64), (900, 70)], 64, 8, 1, 128, "bf16", 9), ([(15999, 2)], 64, 4, 1, 128, "fp32", 14), ([(6000, 1)], 20, 4, 1, 80, "fp32", 12),
]


@pytest.mark.gpu
@pytest.mark.parametrize("equal", [False, True])
@pytest.mark.parametrize("at", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("lens,ps,H,G,d,dtype,gap", SEVERAL)
def test_other_calls_keep_the_weights_beside_a_dominant_key(lens, ps, H, G, d, dtype, gap, at, equal):
    run_dominant(lens, ps, H, G, d, dtype, gap, at, equal, weight=2.0 ** -11 if dtype == "bf16" else 2.0 ** -22, floor=2.0 ** -32 if dtype == "bf16" else 0.0, query=2.0 ** -17 if dtype == "bf16" else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,ps,H,G,d", [
    ([(200, 1), (40, 1)], 64, 8, 1, 128), ([(3000, 1), (40, 1)], 64, 16, 1, 128), ([(60000, 1), (40, 1)], 64, 4, 1, 128), ([(900, 1), (40, 1)], 16, 8, 1, 64), ([(100, 3), (40, 2)], 48, 6, 2, 96),
    ([(3000, 1), (40, 1)], 64, 6, 2, 96), ([(100, 40), (10, 40)], 32, 4, 1, 128), ([(700, 90), (10, 90)], 64, 4, 1, 128), ([(5000, 64), (10, 64)], 64, 2, 1, 128), ([(30, 2), (3, 2)], 16, 2, 1, 40),
])
def test_sinks_of_nothing_and_of_everything(lens, ps, H, G, d, dtype):
    """exp(-inf) adds nothing, exp(+inf) leaves nothing of the keys, and the second sequence, none of whose pages is there, is zero beside either"""
    batch, cache, total = U.batch_of(lens, ps, seed=3)
    cache.page_table[1] = -1
    kv, T = layer(total, G, ps, d, 3), batch.pos.shape[0]
    q = torch.randn((T, H, d), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16 if dtype == "bf16" else torch.float32).cuda()
    run = lambda sink: fp8_cache_attention(q, kv, on(batch), on(cache), H, G, d, d, d ** -0.5, sink=sink)
    row, none, first = torch.ones(H, device="cuda"), run(None), lens[0][1]
    assert none.isfinite().all() and (none[:first] != 0).any() and (none[first:] == 0).all()
    for low in (-math.inf, -3.4028234663852886e38):
        assert torch.equal(run(low * row), none)
    assert (run(row)[first:] == 0).all()
    for high in (math.inf, 3.4028234663852886e38):
        assert (run(high * row) == 0).all()


def test_both_calls_refuse_cpu_tensors():
    batch, cache, total = U.batch_of([(5, 1)], 16)
    kv = layer(total, 2, 16, 32, 0, "cpu")
    with pytest.raises(ValueError, match="fp8_cache_append: CUDA tensors only"):
        fp8_cache_append(torch.zeros(1, 256), batch, cache, kv, 4, 2, 32, 32, (0, 128, 192))
    with pytest.raises(ValueError, match="fp8_cache_attention: CUDA tensors only"):
        fp8_cache_attention(torch.zeros(1, 4, 32), kv, batch, cache, 4, 2, 32, 32, 0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_model_on_an_8_bit_cache_is_near_the_one_on_its_own_type(tmp_path, dtype):
    """Logits of prompt portions and of decoded tokens (the last of them replayed from a graph), the same tokens through both caches.
    An e4m3 number is 2^-4 of itself off at most, 2.5 % in the mean square: of values that much, of scores of unit size twice that (weights of 1.1 to 1.3 on normed queries and keys), so of
    an attention's result 7.5 % or less; three of them in a row, of which each passes on what it got, below a quarter.  Another sequence's logits are further off than half."""
    import lipadra_util as LU
    from ktransformers_b200.models import load_model
    from ktransformers_b200.util.engine import Engine
    cfg = LU.config([(LU.attention(heads=4, kv_heads=2, dim=128, vdim=128, chunk=256, dims=128), None), (LU.attention(heads=4, kv_heads=2, dim=64, vdim=64, chunk=4096, dims=64), None),
                     (LU.attention(heads=4, kv_heads=2, dim=16, vdim=16, chunk=64, dims=16), None)], width=96, alpha=1.0)
    model = load_model(LU.save(tmp_path / "m", cfg, LU.weights(cfg, dtype=getattr(torch, dtype))), dtype)
    tokens = {name: torch.randint(0, 50, (n,), generator=torch.Generator().manual_seed(n)).tolist() for name, n in (("a", 330), ("b", 70), ("c", 9))}

    def serve(kind):
        eng, out = Engine(model, max_tokens=2048, page_size=64, kv_cache=kind), []
        for step in ({"a": 200, "b": 33}, {"a": 120, "b": 27, "c": 1}) + ({"a": 1, "b": 1, "c": 1},) * 6:
            entries = []
            for name, n in step.items():
                at = done.get((kind, name), 0)
                done[kind, name] = at + n
                entries.append((name, tokens[name][at:at + n], list(range(n))))
            out.append(eng.step(entries).float().cpu())
        return torch.cat(out)
    done = {}
    held, plain = serve("fp8"), serve(None)
    off = (held - plain).norm(dim=1) / plain.norm(dim=1)
    other = (plain.roll(1, 0) - plain).norm(dim=1) / plain.norm(dim=1)
    assert off.isfinite().all() and float(off.max()) < 0.25 and float(other.median()) > 0.5, (float(off.max()), float(off.median()), float(other.median()))


@pytest.mark.gpu
@pytest.mark.parametrize("big", [4, 16])
@pytest.mark.parametrize("lens,ps,H,G,d,dtype", [
    ([(1500, 1), (64, 1), (0, 1)], 64, 16, 2, 128, "bf16"), ([(700, 1), (129, 1)], 48, 16, 1, 128, "bf16"), ([(1500, 1), (63, 1)], 16, 8, 1, 64, "bf16"), ([(9001, 1)], 64, 2, 1, 128, "bf16"),
    ([(700, 3), (20, 2)], 32, 8, 2, 128, "bf16"), ([(300, 40), (0, 30)], 16, 4, 2, 96, "bf16"), ([(300, 90), (0, 200)], 64, 8, 2, 128, "bf16"), ([(2000, 64)], 64, 2, 1, 128, "bf16"),
    ([(700, 3), (20, 2)], 32, 8, 2, 128, "fp32"), ([(1500, 1), (63, 1)], 20, 4, 1, 80, "fp32"),
])
def test_scores_of_any_size(lens, ps, H, G, d, dtype, big):
    """scores of 4 and 16 times unit size: a few keys have the weight.  The bounds of each kernel's weights, of the row's own weighted mean and not of the cache's largest value"""
    single = dtype == "bf16" and d in (64, 128) and ps % 16 == 0 and all(n == 1 for _, n in lens)
    weight, floor, query = (2.0 ** -22, 0.0, 0.0) if dtype == "fp32" else (2.0 ** -8, 2.0 ** -35, 2.0 ** -21) if single else (2.0 ** -11, 2.0 ** -32, 2.0 ** -17)
    run_dominant(lens, ps, H, G, d, dtype, None, 0.0, False, weight=weight, floor=floor, query=query, big=big)


@pytest.mark.gpu
@pytest.mark.parametrize("d,ps,dtype", [(128, 64, "bf16"), (64, 16, "bf16"), (96, 48, "bf16"), (128, 64, "fp32")])
def test_steps_read_what_they_appended(d, ps, dtype):
    """Prompt portions, steps of portions beside decoded tokens, and decoded tokens: each step's attention against 64 bits over what the cache holds then, of the queries that the append gave"""
    H, G, g, dt = 8, 2, torch.Generator().manual_seed(d), {"bf16": torch.bfloat16, "fp32": torch.float32}[dtype]
    rot, inv, done = SimpleNamespace(dims=d, layout_code=1), 1000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d), [0, 0, 0]
    _, cache, total = U.batch_of([(0, 400)] * 3, ps)
    kv, i32 = Fp8CacheLayer.empty(total, ps, G, d, d), lambda v: torch.tensor(v, dtype=torch.int32)
    for step in ((200, 70, 0), (90, 1, 1), (1, 150, 1), (1, 1, 1), (2, 1, 3), (1, 1, 1)):
        lens = list(zip(done, step))
        starts = [sum(step[:i]) for i in range(3)]
        batch = SimpleNamespace(pos=i32([p for b, n in lens for p in range(b, b + n)]), slot=i32([i for i, n in enumerate(step) for _ in range(n)]), seqs=i32([starts, step]), n_seqs=3,
                                max_kv=max(b + n for b, n in lens))
        proj = (1 + 3 * (torch.rand((H + 2 * G) * d, generator=g) > 0.97)) * torch.randn((sum(step), (H + 2 * G) * d), generator=g)
        q = fp8_cache_append(proj.to(dt).cuda(), on(batch), on(cache), kv, H, G, d, d, (0, H * d, (H + G) * d), rot, inv.cuda(), 1, 1e-6)
        out = fp8_cache_attention(q, kv, on(batch), on(cache), H, G, d, d, 2 * d ** -0.5).cpu().double().reshape(-1, H, d)
        k, v, s = (x.cpu() for x in (kv.k, kv.v, kv.scales))
        spread = float(s[..., 1].max() / s[..., 1].min())
        weight, floor, query = (2.0 ** -22, 0.0, 0.0) if dtype == "fp32" else (2.0 ** -8, 2.0 ** -32, 2.0 ** -17)      # (whichever kernel a step takes)
        worst, _ = farthest(out, q.cpu(), k, v, s, batch, cache, lens, 2 * d ** -0.5, weight, floor, query, spread)
        assert worst <= 1, (step, worst)
        done = [b + n for b, n in lens]
