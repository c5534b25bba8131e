"""Latent attention's two operators in 64 bits, token by token and head by head from their definitions, and what their tests draw."""
import math
from types import SimpleNamespace

import torch

RANK, ROT = 512, 64
HALF = 2.0 ** -8            # a rounding to bf16: at most this much of the value


def batch_of(lens, page=64, device="cuda", seed=0, idle=0, spare=1, max_kv=None):
    """lens: (tokens before, new tokens) of every portion; pages in any order, `spare` columns and pages more than needed; `idle`: tokens behind the last portion that belong to none."""
    g = torch.Generator().manual_seed(seed)
    need = [(b + n + page - 1) // page for b, n in lens]
    width, total = max(need + [1]) + spare, sum(need) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    table, at = torch.full((len(lens), width), -7, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    starts = [sum(n for _, n in lens[:i]) for i in range(len(lens))]
    T = sum(n for _, n in lens)
    pos = torch.tensor([p for b, n in lens for p in range(b, b + n)] + [3] * idle, dtype=torch.int32)
    slot = torch.tensor([i for i, (_, n) in enumerate(lens) for _ in range(n)] + [0] * idle, dtype=torch.int32)
    seqs = torch.tensor([starts, [n for _, n in lens]], dtype=torch.int32)
    batch = SimpleNamespace(pos=pos.to(device), slot=slot.to(device), seqs=seqs.to(device), n_seqs=len(lens), n_tokens=T + idle, max_kv=max_kv or max([b + n for b, n in lens] + [1]))
    return batch, SimpleNamespace(page_table=table.to(device), max_pages_per_seq=width, page_size=page), total


def draw(lens, heads=4, nope=128, vdim=128, page=64, seed=0, idle=0, device="cuda", max_kv=None, spread=1.0):
    batch, cache, total = batch_of(lens, page, device, seed, idle, max_kv=max_kv)
    gen = torch.Generator(device=device).manual_seed(seed + 1)
    rand = lambda *s: torch.randn(s, generator=gen, device=device)
    T = batch.n_tokens
    return SimpleNamespace(batch=batch, cache=cache, lens=lens, heads=heads, nope=nope, vdim=vdim, page=page, q=(rand(T, heads * (nope + ROT)) * spread).bfloat16(),
                           q_rot=(rand(T, heads, ROT) * spread).bfloat16(), kv=rand(total, page, RANK + ROT).bfloat16(),
                           w=(rand(heads * (nope + vdim), RANK) / math.sqrt(RANK)).bfloat16(), scale=(nope + ROT) ** -0.5)


def held_rows(d, i, n):
    """the first n cache rows of portion i, 64 bits"""
    at = torch.arange(n, device=d.kv.device)
    return d.kv[d.cache.page_table[i].long()[at // d.page], at % d.page].double()


def attention(d):
    """(out, bound) [tokens of all portions, heads * vdim]: the definition in 64 bits, and how far a result may be off that rounds the expanded keys and values, or the absorbed queries and sums,
    the weights and the result to bf16, a rounding being at most HALF of the value:
        scores      |ds_j| <= HALF scale (sum_d |q_d| |k_jd| or sum_r |q'_r| |c_jr|) =: D_j (the larger)        softmax moves a weight by at most 2 max D of itself
        weights, values (or sums) and result, HALF each; what 32-bit sums and exponentials lose stays below another HALF"""
    outs, bounds, at = [], [], 0
    w = d.w.view(d.heads, d.nope + d.vdim, RANK).double()
    for i, (b, n) in enumerate(d.lens):
        rows = held_rows(d, i, b + n)
        lat, rot = rows[:, :RANK], rows[:, RANK:]
        q = d.q.view(-1, d.heads, d.nope + ROT)[at:at + n, :, :d.nope].double()
        see = torch.arange(b + n, device=rows.device)[None, :] <= torch.arange(b, b + n, device=rows.device)[:, None]
        o, e = [], []
        for h in range(d.heads):
            wk, wv = w[h, :d.nope], w[h, d.nope:]
            s = (q[:, h] @ wk @ lat.t() + d.q_rot[at:at + n, h].double() @ rot.t()) * d.scale
            p = torch.softmax(s.masked_fill(~see, -math.inf), 1)
            k, v = lat @ wk.t(), lat @ wv.t()
            off = torch.maximum(q[:, h].abs() @ k.abs().t(), (q[:, h] @ wk).abs() @ lat.abs().t()).masked_fill(~see, 0.0).amax(1) * (HALF * d.scale)
            mass = torch.maximum(p @ v.abs(), (p @ lat).abs() @ wv.abs().t() + (p @ lat.abs()) @ wv.abs().t() * HALF)
            o.append(p @ v)
            e.append(mass * (torch.expm1(2 * off)[:, None] * (1 + 4 * HALF) + 4 * HALF) + o[-1].abs() * HALF)
        outs.append(torch.stack(o, 1).flatten(1))
        bounds.append(torch.stack(e, 1).flatten(1))
        at += n
    return torch.cat(outs), torch.cat(bounds)


def near(got, want, bound, rel=8e-3):
    """Every value within its bound, and all of them together within `rel` in the 2-norm: a rounding to bf16 is 1.65e-3 of a value (root of mean square); four of them and the scores', whose
    spread is about one, are 3.7e-3, and twice that is allowed."""
    got = got.double()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / bound.clamp_min(1e-300)).max().item() if got.numel() else 0.0
    norm = ((got - want).norm() / want.norm().clamp_min(1e-300)).item() if got.numel() else 0.0
    assert worst <= 1.0 and norm <= rel, (worst, norm)
    return norm


def turned(x, pos, rot, freq):
    """x [T, heads, width] in 64 bits: the pairs of the first rot.dims columns as complex numbers"""
    x, half = x.double(), rot.dims // 2
    i = torch.arange(half, device=x.device)
    a, b = (i, i + half) if rot.layout_code else (2 * i, 2 * i + 1)
    z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.full_like(freq, rot.gain), pos.double()[:, None, None] * freq)
    out = x.clone()
    a, b = (i, i + half) if rot.layout_code or rot.split else (2 * i, 2 * i + 1)
    out[..., a], out[..., b] = z.real, z.imag
    return out
