"""Plain forms of the 8-bit cache's append and attention (64-bit, sequence by sequence, on the CPU) and the batches that their tests run."""
import math
from types import SimpleNamespace

import torch

E4M3 = torch.float8_e4m3fn


def batch_of(lens, page_size, device="cpu", spare=1, seed=0, tail=0):
    """lens: (tokens before, tokens of the step) of each sequence; pages in any order, `spare` of them nobody's; `tail` rows behind the last sequence's"""
    g = torch.Generator().manual_seed(seed)
    need = [-(-(b + n) // page_size) for b, n in lens]
    width, total = max(need + [1]) + 1, sum(need) + spare
    order, table, at = torch.randperm(total, generator=g).to(torch.int32), torch.zeros((max(1, len(lens)), width), dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    starts = [sum(n for _, n in lens[:i]) for i in range(len(lens))]
    pos = i32([p for b, n in lens for p in range(b, b + n)] + [0] * tail)
    slot = i32([i for i, (_, n) in enumerate(lens) for _ in range(n)] + [0] * tail)
    seqs = torch.zeros((4, max(1, len(lens))), dtype=torch.int32)
    seqs[0, :len(lens)], seqs[1, :len(lens)] = i32(starts), i32([n for _, n in lens])
    batch = SimpleNamespace(pos=pos.to(device), slot=slot.to(device), seqs=seqs.to(device), n_seqs=len(lens), max_kv=max([b + n for b, n in lens] + [1]))
    cache = SimpleNamespace(page_table=table.to(device), max_pages_per_seq=width, page_size=page_size)
    return batch, cache, total


def exponent(top):
    """the smallest e in [-64, 64] with 448 * 2^e >= top"""
    if not top > 0:
        return -64
    if math.isinf(top):
        return 64
    e = math.ceil(math.log2(top / 448.0))
    e += 448.0 * 2.0 ** e < top
    e -= 448.0 * 2.0 ** (e - 1) >= top
    return min(64, max(-64, e))


def to_codes(x):
    """e4m3 of 64-bit numbers, nearest even, saturating, as the 64-bit numbers they stand for"""
    return x.clamp(-448, 448).to(E4M3).double()


def turned(x, pos, inv_freq, layout_code):
    """x [T, heads, d] (64 bits), its first 2 len(inv_freq) columns turned"""
    n = inv_freq.numel()
    y = x.clone()
    if n:
        a = pos.double()[:, None] * inv_freq
        c, s = a.cos()[:, None], a.sin()[:, None]
        i = torch.arange(n)
        i, j = (i, i + n) if layout_code else (2 * i, 2 * i + 1)
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


def append(proj, batch, cache, k, v, scales, heads, kv_heads, dim, vdim, offsets, rot=None, inv_freq=None, qk_norm=0, eps=0.0, q_weight=None, k_weight=None):
    """(q, k, v, scales, k before rounding, v before rounding) after the append, 64 bits: k, v the codes' own values; what no token reached is as it was in both"""
    p, T = proj.double(), proj.shape[0]
    cols = lambda off, h, d: p[:, off:off + h * d].reshape(T, h, d)
    inv = inv_freq.double() if rot is not None and rot.dims else torch.zeros(0, dtype=torch.float64)

    def ready(x, w):
        if qk_norm:
            x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
            if qk_norm == 3:
                x = x * w.double()
        return turned(x, batch.pos[:T], inv, rot.layout_code if rot is not None else 0)

    q, new = ready(cols(offsets[0], heads, dim), q_weight), (ready(cols(offsets[1], kv_heads, dim), k_weight), cols(offsets[2], kv_heads, vdim))
    held, scales, ps = (k.double(), v.double()), scales.double().clone(), cache.page_size
    ahead = (held[0].clone(), held[1].clone())
    for s in range(batch.n_seqs):
        t, end = int(batch.seqs[0, s]), int(batch.seqs[0, s]) + int(batch.seqs[1, s])
        while t < end:
            at = int(batch.pos[t])
            m = min(end - t, ps - at % ps)
            page = int(cache.page_table[int(batch.slot[t]), (at // ps) % cache.max_pages_per_seq])
            for i in (0, 1):
                for g in range(kv_heads):
                    rows, here = new[i][t:t + m, g], held[i][page, g]
                    e = exponent(float(rows.nan_to_num(0.0, posinf=math.inf, neginf=-math.inf).abs().max()))
                    if at % ps:
                        was = round(math.log2(float(scales[page, g, i])))
                        e = max(e, was)
                        here[:at % ps] = to_codes(here[:at % ps] * 2.0 ** (was - e))
                        ahead[i][page, g, :at % ps] = here[:at % ps]
                    here[at % ps:at % ps + m] = to_codes(rows * 2.0 ** -e)
                    ahead[i][page, g, at % ps:at % ps + m] = rows * 2.0 ** -e
                    scales[page, g, i] = 2.0 ** e
            t += m
    return q, held[0], held[1], scales, ahead[0], ahead[1]


def attention(q, k, v, scales, batch, cache, heads, kv_heads, dim, vdim, scale, head_scale=None, softcap=None, window=None, chunk=None, sink=None, out_scale=1.0):
    """o [T, heads * vdim] in 64 bits; rows of tokens in no portion are NaN"""
    out, ps = torch.full((q.shape[0], heads * vdim), math.nan, dtype=torch.float64), cache.page_size
    keys, values = k.double() * scales.double()[:, :, None, None, 0], v.double() * scales.double()[:, :, None, None, 1]
    n_pages = k.shape[0]
    for s in range(batch.n_seqs):
        t0, n = int(batch.seqs[0, s]), int(batch.seqs[1, s])
        if n == 0:
            continue
        b, slot = int(batch.pos[t0]), int(batch.slot[t0])
        j = torch.arange(b + n)
        page = cache.page_table[slot].long()[(j // ps) % cache.max_pages_per_seq]
        there = (page >= 0) & (page < n_pages)
        page = page.clamp(0, n_pages - 1)
        K, V = keys[page, :, j % ps], values[page, :, j % ps]      # [L, G, d]
        for i in range(n):
            at = b + i
            see = there & (j <= at)
            if window:
                see &= at - j < window
            if chunk:
                see &= j // chunk == at // chunk
            idx = see.nonzero()[:, 0]
            for h in range(heads):
                g = h // (heads // kv_heads)
                z = K[idx, g] @ q[t0 + i].double().reshape(heads, dim)[h] * scale
                if head_scale is not None:
                    z = z * float(head_scale[h])
                if softcap:
                    z = softcap * torch.tanh(z / softcap)
                if sink is not None:
                    z = torch.cat((z, sink[h:h + 1].double()))
                if len(z) == 0:
                    o = torch.zeros(vdim, dtype=torch.float64)
                else:
                    o = torch.softmax(z, 0)[:len(idx)] @ V[idx, g]
                out[t0 + i, h * vdim:(h + 1) * vdim] = o * out_scale
    return out
