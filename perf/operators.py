"""Cases of the 8-bit serving operators: the linear with 8-bit integers (a scale per token and output channel), the append of rotated keys and of values
to a paged e4m3 cache (a scale per page and key/value head), and the attention that reads that cache.

Sizes of the linears are DeepSeek-V3's (models/modeling_deepseek_v3.DeepseekV3Config: width 7168, feed-forward 18432, query latent 1536 -> 128 heads of 192,
query and key/value latents 1536 + 576), head layouts those of util/model_bench's "v3-layer" (64 over 8 heads of 128) and "2k-wide" (16 over 2).  `run` is
plain torch in 32 bits, or the framework's calls where `own` is set; `exact` is the definition in 64 bits.  What is 8 bits wide by definition (the
tokens' integers, the cache's codes and scales) is made there as the formats define it."""
import math
from types import SimpleNamespace

import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
DEV = "cuda"
E4M3_MAX, E_MIN, E_MAX = 448.0, -64, 64


# ------------------------------------------------------------------------------------------------------------------------- cases
def _linear(tokens, n_in, n_out, dtype="bf16", bias=False):
    return {"kind": "linear", "tokens": tokens, "n_in": n_in, "n_out": n_out, "dtype": dtype, "bias": bias}


def _append(seqs, tokens, before, heads=64, kv_heads=8, dim=128, rot=128, layout="halves", norm=0, page=64, dtype="bf16"):
    return {"kind": "append", "seqs": seqs, "tokens": tokens, "before": before, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot, "layout": layout, "norm": norm, "page": page,
            "dtype": dtype}


def _attention(seqs, tokens, before, heads=64, kv_heads=8, dim=128, page=64, window=0, chunk=0, cap=0.0, sink=False, dtype="bf16"):
    return {"kind": "attention", "seqs": seqs, "tokens": tokens, "before": before, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "chunk": chunk,
            "cap": cap, "sink": sink, "dtype": dtype}


def listed():
    return [
        # one decoded token through the widest feed-forward matrix: the weights' bytes are all there is
        dict(_linear(1, 7168, 18432), name="linear_decode_1"),
        # a decode batch of an odd number of users through the query projection, with a bias, in half precision
        dict(_linear(33, 1536, 24576, "fp16", True), name="linear_batch_33"),
        # a short prompt portion through the two latent projections at once, whose rows are not whole tiles, fp32 activations
        dict(_linear(270, 7168, 2112, "fp32"), name="linear_portion_270"),
        # a prompt portion through the down projection
        dict(_linear(4000, 18432, 7168), name="linear_prompt_4000"),
        # one user's decoded token: the smallest call of a serving loop
        dict(_append(1, 1, 5000, heads=16, kv_heads=2), name="append_decode_1"),
        # a decode batch with normed queries and keys, half the columns turned, fp32 activations
        dict(_append(100, 1, 9000, dim=64, rot=32, layout="interleaved", norm=3, dtype="fp32"), name="append_decode_100"),
        # a prompt portion that starts inside a page
        dict(_append(1, 2000, 1061), name="append_prompt_2000"),
        # many users' prompt portions of different lengths in one step
        dict(_append(12, 1900, 300, norm=1), name="append_prompts_12"),
        # one user's decoded token over a short context
        dict(_attention(1, 1, 1500, heads=16, kv_heads=2), name="attention_decode_1"),
        # a decode batch over contexts of different lengths
        dict(_attention(64, 1, 8190), name="attention_decode_64"),
        # one user's decoded token over a very long context
        dict(_attention(1, 1, 131000, sink=True), name="attention_long_1"),
        # a prompt portion behind an earlier one
        dict(_attention(1, 2048, 2001), name="attention_prompt_2048"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("linear", "append", "attention"))
    if kind == "linear":
        while True:
            c = _linear(_log(rng, 1, 4000), 16 * _log(rng, 32, 1152), _log(rng, 500, 24576), rng.choice(("bf16", "fp16", "fp32")), rng.random() < 0.5)
            if c["tokens"] * c["n_in"] * c["n_out"] <= 4000 * 18432 * 7168:
                return c
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 7, 8, 16))
    dim = rng.choice((64, 64, 80, 96, 128, 128, 128, 128))
    page, dtype = rng.choice((16, 32, 48, 64, 64, 64)), rng.choice(("bf16", "bf16", "bf16", "fp32"))
    if kind == "append":
        while True:
            seqs, tokens = _log(rng, 1, 200), _log(rng, 1, 4000)
            if seqs * tokens * (heads + 2 * kv_heads) * dim <= 12 * 1900 * 80 * 128:
                break
        return _append(seqs, tokens, rng.randrange(9000), heads, kv_heads, dim, rng.choice((dim, dim // 2)), rng.choice(("halves", "interleaved")), rng.choice((0, 1, 3)), page, dtype)
    window, chunk = rng.choice(((0, 0), (0, 0), (0, 0), (_log(rng, 1, 4096), 0), (0, _log(rng, 16, 4096))))
    cap, sink = rng.choice((0.0, 0.0, 30.0)), rng.random() < 0.3
    while True:
        seqs, tokens, before = _log(rng, 1, 100), rng.choice((1, 1, 1, _log(rng, 2, 2048))), _log(rng, 8, 131000)
        # what the plain form holds at once (scores and copies of the keys), and the pairs
        if seqs * (before + tokens) <= 300000 and seqs * tokens * heads * (before + tokens) <= 64 * 2048 * 4049:
            return _attention(seqs, tokens, before, heads, kv_heads, dim, page, window, chunk, cap, sink, dtype)


def _lens(c):
    """(tokens before this call, tokens of this call) of every sequence: the case's largest and, behind the first sequence, others down to half of it"""
    n, b = c["tokens"], c["before"]
    return [(b - (7919 * i) % (b // 2 + 1), n - (37 * i) % (n // 2 + 1)) for i in range(c["seqs"])]


# ------------------------------------------------------------------------------------------------------------------------- state
def _pages(c, g):
    """The page table of a cache whose pages lie in any order, one more page than the sequences need, and the batch's index rows."""
    ps, lens = c["page"], _lens(c)
    need = [(b + n + ps - 1) // ps for b, n in lens]
    width, total = max(need) + 1, sum(need) + 1
    order = torch.randperm(total, generator=g, dtype=torch.int64).to(torch.int32)
    table, at = torch.zeros((len(lens), width), dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    starts = [sum(n for _, n in lens[:i]) for i in range(len(lens))]
    zeros = [0] * len(lens)
    pos = torch.cat([torch.arange(b, b + n, dtype=torch.int32) for b, n in lens]).to(DEV)
    slot = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, (_, n) in enumerate(lens)]).to(DEV)
    batch = SimpleNamespace(pos=pos, slot=slot, seqs=ints([starts, [n for _, n in lens], zeros, zeros]), n_seqs=len(lens), n_tokens=int(pos.numel()), max_kv=max(b + n for b, n in lens))
    cache = SimpleNamespace(page_table=table.to(DEV), max_pages_per_seq=width, page_size=ps)
    return batch, cache, total


def _exponent(top):
    """The smallest e with 448 * 2^e >= top, within the format's range (all of them where there is nothing but zeros: the smallest)."""
    m, x = torch.frexp(top)
    e = torch.where(m <= E4M3_MAX / 512, x - 9, x - 8)
    return torch.where(top > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _power(e):
    return torch.ldexp(torch.ones(e.shape, device=e.device), e)


def _random_cache(total, c, gen):
    """Pages that hold keys and values of unit size (some channels larger, as keys have them), quantised page by page and head by head."""
    G, ps, d = c["kv_heads"], c["page"], c["dim"]
    out = []
    for which in range(2):
        x = torch.randn((total, G, ps, d), generator=gen, device=DEV)
        if which == 0:
            x *= 1 + 3 * (torch.rand((1, G, 1, d), generator=gen, device=DEV) > 0.97)
        s = _power(_exponent(x.abs().amax((2, 3))))
        out += [(x / s[:, :, None, None]).to(torch.float8_e4m3fn), s]
        del x
    return out[0], out[2], torch.stack((out[1], out[3]), -1).contiguous()


def prepare(case, seed):
    c = case
    g, gen = torch.Generator().manual_seed(seed), torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    rand = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
    if c["kind"] == "linear":
        T, K, N = c["tokens"], c["n_in"], c["n_out"]
        # activations whose tokens differ in size; weights quantised row by row
        x = (rand(T, K) * torch.exp(rand(T, 1))).to(dt)
        w = rand(N, K)
        top = w.abs().amax(1)
        codes = (w * (127 / top)[:, None]).round_().to(torch.int8)
        return {"kind": "linear", "x": x, "w": codes, "w_scale": top / 127 / math.sqrt(K), "bias": rand(N) if c["bias"] else None}
    batch, cache, total = _pages(c, g)
    H, G, d, T = c["heads"], c["kv_heads"], c["dim"], batch.n_tokens
    k, v, scales = _random_cache(total, c, gen)
    state = {"kind": c["kind"], "batch": batch, "cache": cache, "k": k, "v": v, "scales": scales, "heads": H, "kv_heads": G, "dim": d}
    if c["kind"] == "append":
        lens = _lens(c)
        rot = SimpleNamespace(dims=c["rot"], layout_code=1 if c["layout"] == "halves" else 0)
        inv = 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=DEV) / c["rot"])
        # sequences that go on inside a page
        state |= {"proj": rand(T, (H + 2 * G) * d).to(dt), "rot": rot, "inv_freq": inv, "norm": c["norm"], "eps": 1e-6,
                  "q_w": (1 + 0.2 * rand(d)).to(dt) if c["norm"] == 3 else None, "k_w": (1 + 0.2 * rand(d)).to(dt) if c["norm"] == 3 else None,
                  "begun": torch.tensor([b % c["page"] for b, _ in lens], device=DEV)}
        return state
    n = c["tokens"]
    starts = batch.seqs[0].long()
    place = torch.arange(n, device=DEV)[None, :]
    seq = torch.repeat_interleave(torch.arange(batch.n_seqs, device=DEV), batch.seqs[1].long())
    return state | {"q": rand(T, H, d).to(dt), "scale": d ** -0.5, "window": c["window"], "chunk": c["chunk"], "cap": c["cap"], "sink": rand(H) if c["sink"] else None,
                    # where the plain form finds a sequence's tokens as rows of one length, and the tokens in those rows
                    "rows": starts[:, None] + torch.minimum(place, batch.seqs[1].long()[:, None] - 1), "back": seq * n + torch.arange(T, device=DEV) - starts[seq]}


# ------------------------------------------------------------------------------------------------------------------------- the operators, plainly
def _plain_linear(x, w, w_scale, bias):
    s = x.float().abs().amax(1) / 127
    codes = torch.where(s[:, None] > 0, torch.round(x.float() / s[:, None]), torch.zeros((), device=x.device)).clamp(-127, 127)
    y = (codes @ w.float().T) * (s[:, None] * w_scale)
    return (y if bias is None else y + bias).to(x.dtype)


def _turned(x, angle, dims, layout):
    """x [T, heads, d], its first `dims` columns turned by angle [T, dims / 2]"""
    cos, sin = angle.cos().to(x.dtype)[:, None], angle.sin().to(x.dtype)[:, None]
    r = x[..., :dims]
    a, b = (r[..., :dims // 2], r[..., dims // 2:]) if layout else (r[..., 0::2], r[..., 1::2])
    u, w = a * cos - b * sin, b * cos + a * sin
    return torch.cat((torch.cat((u, w), -1) if layout else torch.stack((u, w), -1).flatten(-2), x[..., dims:]), -1)


def _normed(x, norm, weight, eps, first):
    if norm == 0 or (norm == 3) != first:
        return x
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    return y if weight is None else y * weight.to(x.dtype)


def _plain_append(s):
    batch, cache, H, G, d, norm = s["batch"], s["cache"], s["heads"], s["kv_heads"], s["dim"], s["norm"]
    p, T, ps = s["proj"].float(), batch.n_tokens, cache.page_size
    angle = batch.pos.double()[:, None] * s["inv_freq"]
    ready = lambda x, w: _normed(_turned(_normed(x, norm, w, s["eps"], True), angle, s["rot"].dims, s["rot"].layout_code), norm, None, s["eps"], False)
    q = ready(p[:, :H * d].view(T, H, d), s["q_w"])
    new = {0: ready(p[:, H * d:(H + G) * d].view(T, G, d), s["k_w"]), 1: p[:, (H + G) * d:].view(T, G, d)}
    pos = batch.pos.long()
    page, row = cache.page_table[batch.slot.long(), pos // ps].long(), pos % ps
    # the pages that tokens go on in keep what they hold
    first = batch.seqs[0].long()
    goes_on = (s["begun"] > 0)[:, None]
    held_page, held_rows = page[first], torch.arange(ps, device=pos.device)[None, :] < s["begun"][:, None]
    for i, codes in ((0, s["k"]), (1, s["v"])):
        scale = s["scales"][:, :, i]
        old = scale[held_page]
        top = torch.zeros_like(scale).scatter_reduce_(0, page[:, None].expand(T, G), new[i].abs().amax(-1), "amax")
        made = _power(_exponent(top))
        now = torch.where(goes_on, torch.maximum(made[held_page], old), made[held_page])
        made[held_page] = now
        kept = codes[held_page]
        moved = (kept.float() * (old / now)[:, :, None, None]).to(codes.dtype)
        codes[held_page] = torch.where(held_rows[:, None, :, None], moved.view(torch.int8), kept.view(torch.int8)).view(codes.dtype)
        scale[page] = made[page]
        codes[page, :, row] = (new[i] / made[page][:, :, None]).to(codes.dtype)
    return q.to(s["proj"].dtype), s["k"], s["v"], s["scales"]


def _plain_attention(s):
    batch, cache, H, G, d = s["batch"], s["cache"], s["heads"], s["kv_heads"], s["dim"]
    B, ps, R = batch.n_seqs, cache.page_size, H // G
    pages = cache.page_table[:, :(batch.max_kv + ps - 1) // ps].long()
    L = pages.shape[1] * ps
    read = lambda codes, i: (codes[pages].float() * s["scales"][pages][..., i, None, None]).transpose(1, 2).reshape(B, G, L, d)
    n = s["rows"].shape[1]
    q = s["q"][s["rows"]].float().view(B, n, G, R, d).permute(0, 2, 1, 3, 4).reshape(B, G, n * R, d)
    z = (q @ read(s["k"], 0).transpose(-1, -2)).view(B, G, n, R, L) * s["scale"]
    if s["cap"]:
        z = s["cap"] * torch.tanh(z / s["cap"])
    at, key = batch.pos[s["rows"]][:, :, None], torch.arange(L, device=z.device)
    seen = key <= at
    if s["window"]:
        seen = seen & (at - key < s["window"])
    if s["chunk"]:
        seen = seen & (key // s["chunk"] == at // s["chunk"])
    z = z.masked_fill(~seen[:, None, :, None, :], -math.inf)
    top = z.amax(-1, keepdim=True)
    sink = s["sink"].view(1, G, 1, R, 1) if s["sink"] is not None else None
    if sink is not None:
        top = torch.maximum(top, sink)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    # (rows behind a sequence's last token are never written: their values must not be either)
    v = read(s["v"], 1).masked_fill(~(key[None, :] < batch.pos[s["rows"][:, -1]][:, None] + 1)[:, None, :, None], 0.0)
    o = (e.view(B, G, n * R, L) @ v).view(B, G, n, R, d) / total
    return o.permute(0, 2, 1, 3, 4).reshape(B * n, H * d)[s["back"]].to(s["q"].dtype)


def run(state):
    s = state
    if s["kind"] == "linear":
        if own:
            from ktransformers_b200.operators.linear import int8_linear
            return int8_linear(s["x"], s["w"], s["w_scale"], s["bias"])
        return _plain_linear(s["x"], s["w"], s["w_scale"], s["bias"])
    if own:
        from ktransformers_b200.models.custom_cache import Fp8CacheLayer
        from ktransformers_b200.operators.attention import fp8_cache_append, fp8_cache_attention
        H, G, d = s["heads"], s["kv_heads"], s["dim"]
        kv = Fp8CacheLayer(s["k"], s["v"], s["scales"])
        if s["kind"] == "append":
            q = fp8_cache_append(s["proj"], s["batch"], s["cache"], kv, H, G, d, d, (0, H * d, (H + G) * d), rot=s["rot"], inv_freq=s["inv_freq"], qk_norm=s["norm"], eps=s["eps"],
                                 q_weight=s["q_w"], k_weight=s["k_w"])
            return q, s["k"], s["v"], s["scales"]
        return fp8_cache_attention(s["q"], kv, s["batch"], s["cache"], H, G, d, d, s["scale"], softcap=s["cap"] or None, window=s["window"] or None, chunk=s["chunk"] or None, sink=s["sink"])
    return _plain_append(s) if s["kind"] == "append" else _plain_attention(s)


# ------------------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    e = BYTES[c["dtype"]]
    if c["kind"] == "linear":
        T, K, N = c["tokens"], c["n_in"], c["n_out"]
        return {"bytes": T * K * e + N * K + 4 * N * (2 if c["bias"] else 1) + T * N * e, "flops": 2 * T * K * N}
    H, G, d, lens, ps = c["heads"], c["kv_heads"], c["dim"], _lens(c), c["page"]
    T = sum(n for _, n in lens)
    if c["kind"] == "append":
        blocks = sum((b + n - 1) // ps - b // ps + 1 for b, n in lens) * G
        return {"bytes": T * (H + 2 * G) * d * e + T * H * d * e + T * 2 * G * d + 8 * blocks, "flops": T * (H + G) * (4 * c["rot"] + (4 * d if c["norm"] else 0)) + T * 4 * G * d}
    pairs, keys = 0, 0
    for b, n in lens:
        lo = lambda p: max(p - c["window"] + 1 if c["window"] else 0, p - p % c["chunk"] if c["chunk"] else 0, 0)
        pairs += sum(p + 1 - lo(p) for p in range(b, b + n))
        keys += b + n - lo(b)
    return {"bytes": 2 * T * H * d * e + keys * G * 2 * d + 8 * G * (keys // ps), "flops": 4 * H * d * pairs}


# ------------------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_turn(row, position, freq, dims, halves):
    """one head's columns [.., d] in 64 bits; the pair i turns as a complex number"""
    out = row.clone()
    first = torch.arange(dims // 2, device=row.device) if halves else 2 * torch.arange(dims // 2, device=row.device)
    second = first + (dims // 2 if halves else 1)
    z = torch.complex(row[..., first], row[..., second]) * torch.polar(torch.ones_like(freq), position[:, None, None] * freq)
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "linear":
        x = s["x"].double()
        step = (x.abs().max(1).values / 127).float().double()      # the token's scale is a number of 32 bits, and so is the quotient that is rounded
        codes = torch.round((x / step.clamp_min(1e-300)[:, None]).float().double())
        y = torch.matmul(codes, s["w"].double().t()) * step[:, None] * s["w_scale"].double()[None, :]
        return y + s["bias"].double() if s["bias"] is not None else y
    batch, cache, H, G, d, ps = s["batch"], s["cache"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    lens, table = _lens(c), cache.page_table.long()
    if c["kind"] == "append":
        x = s["proj"].double()
        position = batch.pos.double()
        heads = x.view(x.shape[0], H + 2 * G, d)
        qk = heads[:, :H + G]
        if c["norm"]:
            qk = qk * torch.rsqrt(qk.pow(2).sum(-1, keepdim=True) / d + s["eps"])
            if c["norm"] == 3:
                qk = torch.cat((qk[:, :H] * s["q_w"].double(), qk[:, H:] * s["k_w"].double()), 1)
        qk = _exact_turn(qk, position, s["inv_freq"], c["rot"], c["layout"] == "halves")
        k, v, scales = s["k"].double(), s["v"].double(), s["scales"].double()
        at = 0
        for i, (b, n) in enumerate(lens):
            p = b
            while p < b + n:      # page by page
                m = min(ps - p % ps, b + n - p)
                page = int(table[i, p // ps])
                for j, (codes, rows) in enumerate(((k, qk[at:at + m, H:]), (v, heads[at:at + m, H + G:]))):
                    e = _exponent(rows.abs().amax((0, 2)))
                    if p % ps:
                        e = torch.maximum(e, torch.log2(scales[page, :, j]).round().to(e.dtype))
                        was = codes[page, :, :p % ps] * scales[page, :, j][:, None, None]
                        codes[page, :, :p % ps] = (was * torch.exp2(-e.double())[:, None, None]).float().to(torch.float8_e4m3fn).double()
                    scales[page, :, j] = torch.exp2(e.double())
                    codes[page, :, p % ps:p % ps + m] = (rows * torch.exp2(-e.double())[:, None]).float().to(torch.float8_e4m3fn).double().transpose(0, 1)
                at, p = at + m, p + m
        return qk[:, :H], k, v, scales
    if sum(n * (b + n) for b, n in lens) * H * d > 1 << 40:
        return None
    out, at = [], 0
    for i, (b, n) in enumerate(lens):
        pages = table[i, :(b + n + ps - 1) // ps]
        wide = lambda codes, j: (codes[pages].double() * s["scales"][pages][:, :, j, None, None].double()).permute(1, 0, 2, 3).flatten(1, 2)[:, :b + n]
        keys, values = wide(s["k"], 0), wide(s["v"], 1)
        i_at, j_at = torch.arange(b, b + n, device=DEV)[:, None], torch.arange(b + n, device=DEV)[None, :]
        hidden = j_at > i_at
        if c["window"]:
            hidden |= j_at <= i_at - c["window"]
        if c["chunk"]:
            hidden |= torch.div(j_at, c["chunk"], rounding_mode="floor") != torch.div(i_at, c["chunk"], rounding_mode="floor")
        rows = []
        for h in range(H):
            z = s["q"][at:at + n, h].double() @ keys[h // (H // G)].t() / math.sqrt(d)
            if c["cap"]:
                z = torch.tanh(z / c["cap"]) * c["cap"]
            z = torch.where(hidden, torch.full_like(z, -math.inf), z)
            if c["sink"]:
                z = torch.cat((z, s["sink"][h].double().expand(n, 1)), 1)
            w = torch.softmax(z, 1)[:, :b + n]
            rows.append(w @ values[h // (H // G)])
        out.append(torch.stack(rows, 1).flatten(1))
        at += n
    return torch.cat(out)
