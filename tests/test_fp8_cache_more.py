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
