"""KDeepseekV2Attention with several tokens a sequence and with scaled rotations: against the plain formulation (DeepseekV3Attention.forward) in 32 bits, over portions, drafts and decoded tokens
in one cache, eagerly and in a graph; and what it refuses."""
import math

import pytest
import torch

from ktransformers_b200.models.modeling_deepseek_v3 import DeepseekV3Attention, DeepseekV3Config, DeepseekV3RotaryEmbedding, DeepseekV3YarnRotaryEmbedding, yarn_get_mscale

gpu = pytest.mark.gpu
YARN = {"type": "yarn", "factor": 40, "original_max_position_embeddings": 4096, "beta_fast": 32, "beta_slow": 1, "mscale": 1.0, "mscale_all_dim": 1.0}


def layer(heads, q_rank, scaling, nope=128, vdim=128, seed=0):
    torch.manual_seed(seed)
    cfg = DeepseekV3Config(hidden_size=512, num_attention_heads=heads, q_lora_rank=q_rank, num_hidden_layers=1, qk_nope_head_dim=nope, v_head_dim=vdim, rope_scaling=scaling)
    plain = DeepseekV3Attention(cfg, layer_idx=0)
    for m in plain.modules():
        if isinstance(m, torch.nn.Linear):
            torch.nn.init.normal_(m.weight, std=m.in_features ** -0.5)
    plain = plain.to(device="cuda", dtype=torch.bfloat16)
    if scaling is None:
        plain.rotary_emb = DeepseekV3RotaryEmbedding(64).to("cuda")
    return cfg, plain


class Exact:
    """the layer over everything so far, its bf16 weights and inputs in 32 bits"""

    def __init__(self, cfg, plain):
        self.layer = DeepseekV3Attention(cfg, layer_idx=0).to("cuda").float()
        self.layer.load_state_dict({k: v.float() for k, v in plain.state_dict().items()})
        self.layer.rotary_emb = plain.rotary_emb
        self.past = None

    def __call__(self, x, position_ids):
        y, self.past = self.layer(x.float(), position_ids, self.past)
        return y


@gpu
@pytest.mark.parametrize("absorb", [False, True])
@pytest.mark.parametrize("bsz,heads,q_rank,scaling,nope,vdim", [(1, 16, 256, None, 128, 128), (2, 5, None, YARN, 128, 128), (3, 8, 128, YARN, 64, 64)])
def test_portions_drafts_and_tokens_against_the_plain_layer(bsz, heads, q_rank, scaling, nope, vdim, absorb):
    from ktransformers_b200.models.custom_cache import StaticCache
    from ktransformers_b200.operators.attention import KDeepseekV2Attention
    from ktransformers_b200.operators.flashinfer_wrapper import MLAWrapper
    cfg, plain = layer(heads, q_rank, scaling, nope, vdim, seed=heads)
    exact = Exact(cfg, plain)
    op = KDeepseekV2Attention("blk.0.self_attn", None, cfg, plain, "cuda", "cuda", absorb_for_prefill=absorb)
    cache = StaticCache(cfg, max_batch_size=bsz + 1, max_cache_len=700, device="cuda")
    op.mla_wrapper = MLAWrapper(bsz, cache.max_pages * bsz)
    at = 0
    for n in (300, 1, 7, 130, 1):      # a prompt portion, a token, drafts, another portion, a token
        x = torch.randn(bsz, n, 512, device="cuda").bfloat16()
        where = torch.arange(at, at + n, device="cuda")
        with torch.no_grad():
            y, _, _ = op(x, position_ids=where[None].expand(bsz, n), past_key_value=cache, cache_position=where)
            want = exact(x, where[None].expand(bsz, n))
        at += n
        assert y.shape == (bsz, n, 512) and cache.get_seq_length(0) == at
        # projections, cache, scores, weights, sums and results are rounded to bf16, some ten roundings of 1.65e-3 (root of mean square) of the values one behind the other: 5.2e-3, three times that
        rel = (y.float() - want).norm() / want.norm()
        assert rel <= 1.6e-2, (n, at, rel.item())
    assert (cache.key_cache[0].view(bsz + 1, -1, 576)[bsz] == 0).all()      # the sequence that was not in the batch


@gpu
def test_scaled_decode_in_a_graph():
    """A decoded token with a scaled rotation, captured once and replayed for the next positions, gives the bits of the eager calls."""
    from ktransformers_b200.models.custom_cache import StaticCache
    from ktransformers_b200.operators.attention import KDeepseekV2Attention
    cfg, plain = layer(16, 128, YARN, seed=3)
    op = KDeepseekV2Attention("blk.0.self_attn", None, cfg, plain, "cuda", "cuda")
    make = lambda: StaticCache(cfg, max_batch_size=2, max_cache_len=300, device="cuda")
    prompt, tokens = torch.randn(2, 100, 512, device="cuda").bfloat16(), torch.randn(5, 2, 1, 512, device="cuda").bfloat16()
    where = lambda a, n: torch.arange(a, a + n, device="cuda")
    with torch.no_grad():
        eager, cache = [], make()
        op(prompt, position_ids=where(0, 100)[None].expand(2, -1), past_key_value=cache, cache_position=where(0, 100))
        for i in range(5):
            eager.append(op(tokens[i], position_ids=where(100 + i, 1)[None].expand(2, -1), past_key_value=cache, cache_position=where(100 + i, 1))[0])
        other = make()
        op(prompt, position_ids=where(0, 100)[None].expand(2, -1), past_key_value=other, cache_position=where(0, 100))
        x, ids, at = tokens[0].clone(), torch.full((2, 1), 100, device="cuda"), torch.full((1,), 100, device="cuda")
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            y = op(x, position_ids=ids, past_key_value=other, cache_position=at)[0]
        for i in range(5):
            x.copy_(tokens[i]); ids.fill_(100 + i); at.fill_(100 + i)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager[i])
    assert torch.equal(cache.key_cache[0], other.key_cache[0])


@gpu
def test_portions_that_are_refused():
    from ktransformers_b200.models.custom_cache import StaticCache
    from ktransformers_b200.operators.attention import KDeepseekV2Attention
    cfg, plain = layer(4, 64, None)
    op = KDeepseekV2Attention("blk.0.self_attn", None, cfg, plain, "cuda", "cuda")
    cache = StaticCache(cfg, max_batch_size=1, max_cache_len=64, device="cuda")
    run = lambda x, n, **kw: op(x, **{**dict(position_ids=torch.arange(n, device="cuda")[None], past_key_value=cache, cache_position=torch.arange(n, device="cuda")), **kw})
    x = torch.randn(1, 8, 512, device="cuda").bfloat16()
    with torch.no_grad():
        run(x, 8)
        for wrong in (dict(cache_position=None), dict(position_ids=None), dict(past_key_value=None)):
            with pytest.raises(NotImplementedError):
                run(x, 8, **wrong)
        with pytest.raises(ValueError):
            run(torch.randn(2, 8, 512, device="cuda").bfloat16(), 8)
        with pytest.raises(ValueError):
            run(torch.randn(1, 65, 512, device="cuda").bfloat16(), 65)
        with pytest.raises(ValueError):
            run(x, 8, cache_position=torch.arange(7, device="cuda"))


def test_yarn_tables():
    """The configuration's scaled rotation: far positions keep their angle (fp64), cosines carry mscale over mscale_all_dim's part, the soft-max scale has that part's square; a cast of the
    model leaves the frequencies alone."""
    cfg = DeepseekV3Config(hidden_size=64, num_attention_heads=2, q_lora_rank=None, num_hidden_layers=1, rope_scaling={**YARN, "mscale": 0.7, "mscale_all_dim": 1.0})
    a = DeepseekV3Attention(cfg).to(torch.bfloat16)
    assert type(a.rotary_emb) is DeepseekV3YarnRotaryEmbedding
    m = yarn_get_mscale(40, 1.0)
    assert math.isclose(a.softmax_scale, 192 ** -0.5 * m * m) and math.isclose(a.rotary_emb.gain, yarn_get_mscale(40, 0.7) / m)
    cos, sin = a.rotary_emb(torch.zeros(1, dtype=torch.float64), torch.tensor([[0, 160000]]))
    assert cos.shape == (1, 2, 64) and torch.allclose(cos[0, 0], torch.full((64,), a.rotary_emb.gain, dtype=torch.float64))
    f = a.rotary_emb.inv_freq_on("cpu")
    assert f.dtype is torch.float64 and torch.allclose(sin[0, 1, :32], torch.sin(160000 * f) * a.rotary_emb.gain, atol=1e-12)
    cfg.rope_scaling = None
    assert type(DeepseekV3Attention(cfg).rotary_emb) is DeepseekV3RotaryEmbedding
