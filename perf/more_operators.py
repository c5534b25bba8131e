"""Cases of latent attention beyond one decoded token with plain rotary positions: the append to the paged latent cache (rotation of the queries' and the key's rotated parts, also
scaled for long contexts; norm of the latent; both written to their page), and the attention of new tokens over that cache, from one token a sequence to long prompt portions.

Sizes are DeepSeek-V3's (models/modeling_deepseek_v3.DeepseekV3Config: 128 heads of 128 + 64 over latents of 512 + 64, values of 128), and those with 16 heads and halves of them.  `run` is
plain torch in 32 bits, or the framework's calls where `own` is set; `exact` is the definition in 64 bits."""
import math
from types import SimpleNamespace

import torch

own = False
DEV, BF16 = "cuda", torch.bfloat16
RANK, ROT = 512, 64
ORIGINAL = 4096            # positions that a scaled rotation was trained on


# ------------------------------------------------------------------------------------------------------------------------- cases
def _append(seqs, tokens, before, heads=128, nope=128, page=64, layout="split", factor=1.0, dims=ROT):
    return {"kind": "append", "seqs": seqs, "tokens": tokens, "before": before, "heads": heads, "nope": nope, "page": page, "layout": layout, "factor": factor, "dims": dims}


def _attention(seqs, tokens, before, heads=128, nope=128, vdim=128, page=64, factor=1.0):
    return {"kind": "attention", "seqs": seqs, "tokens": tokens, "before": before, "heads": heads, "nope": nope, "vdim": vdim, "page": page, "factor": factor}


def listed():
    return [
        # one user's decoded token in a context of 40 times the trained length: the smallest call of a serving loop
        dict(_append(1, 1, 100000, factor=40.0), name="append_decode_1"),
        # a decode batch of an odd number of users, the plain rotation
        dict(_append(67, 1, 9000), name="append_decode_67"),
        # a prompt portion that starts inside a page
        dict(_append(1, 2000, 1061, factor=40.0), name="append_prompt_2000"),
        # many users' prompt portions of different lengths in one step, columns in halves, half of them turned, short pages
        dict(_append(12, 1900, 300, heads=16, page=16, layout="halves", dims=32), name="append_prompts_12"),
        # one user's decoded token over a short context
        dict(_attention(1, 1, 1500, heads=16), name="attention_decode_1"),
        # a decode batch over contexts of different lengths
        dict(_attention(32, 1, 8190), name="attention_decode_32"),
        # a few drafted tokens a user, to be verified in one step
        dict(_attention(16, 5, 3000, factor=40.0), name="attention_drafts_16"),
        # a short question behind a long document
        dict(_attention(1, 45, 30000), name="attention_question_45"),
        # a first prompt portion
        dict(_attention(1, 1000, 0), name="attention_prompt_1000"),
        # a prompt portion behind an earlier one
        dict(_attention(1, 2048, 2001, factor=40.0), name="attention_prompt_2048"),
        # several users' portions of odd lengths, fewer and smaller heads, short pages
        dict(_attention(6, 1201, 700, heads=16, nope=64, vdim=64, page=16), name="attention_prompts_6"),
        # the last portion of a long prompt
        dict(_attention(1, 1000, 31000), name="attention_long_1000"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, nope, page, factor = rng.choice((5, 16, 16, 64, 128, 128)), rng.choice((64, 128, 128, 128)), rng.choice((16, 32, 48, 64, 64)), rng.choice((1.0, 1.0, 40.0))
    if rng.choice((False, False, True)):
        while True:
            seqs, tokens = _log(rng, 1, 200), _log(rng, 1, 4000)
            if seqs * tokens * (heads + 9) <= 2000 * 137:
                return _append(seqs, tokens, rng.randrange(100000 // seqs + 1), heads, nope, page, rng.choice(("split", "split", "halves", "interleaved")), factor, rng.choice((ROT, ROT, ROT // 2)))
    while True:
        seqs, tokens, before = _log(rng, 1, 64), rng.choice((1, _log(rng, 2, 64), _log(rng, 40, 2500), _log(rng, 40, 2500))), rng.choice((0, _log(rng, 1, 31000), _log(rng, 100, 31000)))
        keys = before + tokens
        # what the plain form multiplies, and what it holds at once (keys and values of 16 heads)
        if seqs * tokens * keys * heads <= 1000 * 32000 * 128 and seqs * keys <= 262080 and (tokens < 64 or seqs * keys <= 33000):
            return _attention(seqs, tokens, before, heads, nope, rng.choice((64, 128, 128, 128)), page, factor)


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
    pos = torch.cat([torch.arange(b, b + n, dtype=torch.int32) for b, n in lens]).to(DEV)
    slot = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, (_, n) in enumerate(lens)]).to(DEV)
    batch = SimpleNamespace(pos=pos, slot=slot, seqs=ints([starts, [n for _, n in lens]]), n_seqs=len(lens), n_tokens=int(pos.numel()), max_kv=max(b + n for b, n in lens))
    cache = SimpleNamespace(page_table=table.to(DEV), max_pages_per_seq=width, page_size=ps)
    return batch, cache, total


def _rotation(c):
    """What a model keeps of its rotation: the frequencies in 64 bits, those of a scaled one stretched where they turn less than once in the trained length, kept where they turn more
    than 32 times, and in between in a straight line (over the column); the factor that its cosines and sines get."""
    dims, factor = c["dims"], c["factor"]
    i = torch.arange(dims // 2, dtype=torch.float64)
    freq = 10000.0 ** (-2.0 * i / dims)
    if factor > 1:
        column = lambda turns: dims * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
        lo, hi = max(math.floor(column(32)), 0), min(math.ceil(column(1)), dims - 1)
        share = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        freq = freq * (1 - share) + freq / factor * share
    # DeepSeek-V3 has the factor of long contexts in its soft-max; models without have it here
    gain = 0.1 * math.log(factor) + 1 if c["layout"] != "split" else 1.0
    return SimpleNamespace(dims=dims, layout_code=1 if c["layout"] == "halves" else 0, split=c["layout"] == "split", gain=gain), freq.to(DEV)


def prepare(case, seed):
    c = case
    g, gen = torch.Generator().manual_seed(seed), torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
    batch, cache, total = _pages(c, g)
    T, H, N = batch.n_tokens, c["heads"], c["nope"]
    kv = rand(total, c["page"], RANK + ROT).to(BF16)        # normed latents and turned keys
    state = {"kind": c["kind"], "batch": batch, "cache": cache, "kv": kv, "heads": H, "nope": N, "q": rand(T, H * (N + ROT)).to(BF16)}
    if c["kind"] == "append":
        rot, freq = _rotation(c)
        # the projection's row holds the latent, whose tokens differ in size, and the key's rotated part
        return state | {"kva": torch.cat((rand(T, RANK) * torch.exp(rand(T, 1)), rand(T, ROT)), 1).to(BF16), "weight": (1 + 0.2 * rand(RANK)).to(BF16), "eps": 1e-6, "rot": rot, "freq": freq}
    V, n = c["vdim"], c["tokens"]
    starts, count = batch.seqs[0].long(), batch.seqs[1].long()
    seq = torch.repeat_interleave(torch.arange(batch.n_seqs, device=DEV), count)
    scale = (N + ROT) ** -0.5 * (0.1 * math.log(c["factor"]) + 1) ** 2
    return state | {"q_rot": rand(T, H, ROT).to(BF16), "w": (rand(H * (N + V), RANK) / math.sqrt(RANK)).to(BF16), "vdim": V, "scale": scale,
                    # where the plain form finds a sequence's tokens as rows of one length, and the tokens in those rows
                    "rows": starts[:, None] + torch.minimum(torch.arange(n, device=DEV)[None, :], count[:, None] - 1), "back": seq * n + torch.arange(T, device=DEV) - starts[seq]}


# ------------------------------------------------------------------------------------------------------------------------- the operators, plainly
def _turned(x, angle, rot):
    """x [T, heads, ROT], the pairs of its first rot.dims columns turned by angle [T, dims / 2]"""
    half = rot.dims // 2
    cos, sin = (angle.cos() * rot.gain).to(x.dtype)[:, None], (angle.sin() * rot.gain).to(x.dtype)[:, None]
    r = x[..., :rot.dims]
    a, b = (r[..., :half], r[..., half:]) if rot.layout_code else (r[..., 0::2], r[..., 1::2])
    u, w = a * cos - b * sin, b * cos + a * sin
    return torch.cat((torch.cat((u, w), -1) if rot.layout_code or rot.split else torch.stack((u, w), -1).flatten(-2), x[..., rot.dims:]), -1)


def _plain_append(s):
    batch, cache, H, N, rot = s["batch"], s["cache"], s["heads"], s["nope"], s["rot"]
    T, ps = batch.n_tokens, cache.page_size
    pos = batch.pos.long()
    angle = pos.double()[:, None] * s["freq"]
    q = _turned(s["q"].view(T, H, N + ROT)[..., N:].float(), angle, rot)
    x = s["kva"][:, :RANK].float()
    latent = x / torch.sqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    key = _turned(s["kva"][:, None, RANK:].float(), angle, rot)[:, 0]
    s["kv"][cache.page_table[batch.slot.long(), pos // ps].long(), pos % ps] = torch.cat((latent, key), -1).to(BF16)
    return q.to(BF16), s["kv"]


def _plain_attention(s):
    batch, cache, H, N, V = s["batch"], s["cache"], s["heads"], s["nope"], s["vdim"]
    ps, n, B = cache.page_size, s["rows"].shape[1], batch.n_seqs
    pages = cache.page_table[:, :(batch.max_kv + ps - 1) // ps].long()
    L = pages.shape[1] * ps
    pos = batch.pos[s["rows"]].long()
    key = torch.arange(L, device=pos.device)
    seen = key[None, None, :] <= pos[:, :, None]
    held = s["kv"][pages].view(B, L, RANK + ROT).float()
    held = held.masked_fill((key[None, :] > pos[:, -1:])[:, :, None], 0.0)      # (rows behind a sequence's last token hold anything)
    w = s["w"].view(H, N + V, RANK).float()
    q = s["q"].view(-1, H, N + ROT)[..., :N][s["rows"]].float()
    q_rot = s["q_rot"][s["rows"]].float()
    out = torch.empty((B, n, H, V), device=pos.device)
    # few tokens: the query goes to the latents, and the sum of latents to the values; many: keys and values are made of the latents.  As many heads at once as fit
    step = max(1, min(H, (1 << 29) // (B * n * L), (1 << 30) // (B * L * (N + V)) if n >= 64 else H))
    for h in range(0, H, step):
        at = slice(h, min(h + step, H))
        z = torch.einsum("bnhr,blr->bhnl", q_rot[:, :, at], held[..., RANK:])
        if n < 64:
            z += torch.einsum("bnhr,blr->bhnl", torch.einsum("bnhd,hdr->bnhr", q[:, :, at], w[at, :N]), held[..., :RANK])
        else:
            z += torch.einsum("bnhd,bhld->bhnl", q[:, :, at], torch.einsum("blr,hdr->bhld", held[..., :RANK], w[at, :N]))
        z = (z * s["scale"]).masked_fill(~seen[:, None], -math.inf)
        e = torch.exp(z - z.amax(-1, keepdim=True))
        total = e.sum(-1)
        if n < 64:
            o = torch.einsum("bhnr,hdr->bhnd", torch.einsum("bhnl,blr->bhnr", e, held[..., :RANK]), w[at, N:])
        else:
            o = torch.einsum("bhnl,bhld->bhnd", e, torch.einsum("blr,hdr->bhld", held[..., :RANK], w[at, N:]))
        out[:, :, at] = (o / total[..., None]).transpose(1, 2)
    return out.view(B * n, H * V)[s["back"]].to(BF16)


def run(state):
    s = state
    if own:
        from ktransformers_b200.operators.latent_attention import latent_append, latent_attention
        if s["kind"] == "append":
            return latent_append(s["q"], s["kva"], s["weight"], s["eps"], s["batch"], s["cache"], s["kv"], s["heads"], s["nope"], rot=s["rot"], inv_freq=s["freq"]), s["kv"]
        return latent_attention(s["q"], s["q_rot"], s["kv"], s["w"], s["batch"], s["cache"], s["heads"], s["nope"], s["vdim"], s["scale"])
    return _plain_append(s) if s["kind"] == "append" else _plain_attention(s)


# ------------------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    H, N, lens = c["heads"], c["nope"], _lens(c)
    T = sum(n for _, n in lens)
    if c["kind"] == "append":
        return {"bytes": 4 * T * (H * ROT + RANK + ROT) + 2 * RANK, "flops": T * ((H + 1) * 3 * c["dims"] + 4 * RANK)}
    V, flops = c["vdim"], 0
    for b, n in lens:      # the cheaper form of each sequence
        pairs = n * b + n * (n + 1) // 2
        flops += min(2 * n * RANK * H * (N + V) + 2 * pairs * H * (2 * RANK + ROT), 2 * (b + n) * RANK * H * (N + V) + 2 * pairs * H * (N + ROT + V))
    return {"bytes": 2 * (T * H * (N + ROT + V) + H * (N + V) * RANK + sum(b + n for b, n in lens) * (RANK + ROT)), "flops": flops}


# ------------------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_turn(x, position, freq, rot):
    """x [T, heads, ROT] in 64 bits; the pair i turns as a complex number"""
    out, half = x.clone(), rot.dims // 2
    i = torch.arange(half, device=x.device)
    first, second = (i, i + half) if rot.layout_code else (2 * i, 2 * i + 1)
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.full_like(freq, rot.gain), position[:, None, None] * freq)
    first, second = (i, i + half) if rot.layout_code or rot.split else (2 * i, 2 * i + 1)
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    batch, cache, H, N = s["batch"], s["cache"], c["heads"], c["nope"]
    lens, table, ps = _lens(c), cache.page_table.long(), c["page"]
    if c["kind"] == "append":
        x = s["kva"].double()
        latent = x[:, :RANK] * torch.rsqrt(x[:, :RANK].pow(2).sum(-1, keepdim=True) / RANK + s["eps"]) * s["weight"].double()
        position = batch.pos.double()
        row = torch.cat((latent, _exact_turn(x[:, None, RANK:], position, s["freq"], s["rot"])[:, 0]), 1)
        held, at = s["kv"].double(), 0
        for i, (b, n) in enumerate(lens):
            p = b
            while p < b + n:      # page by page
                m = min(ps - p % ps, b + n - p)
                held[table[i, p // ps], p % ps:p % ps + m] = row[at:at + m]
                at, p = at + m, p + m
        return _exact_turn(s["q"].view(-1, H, N + ROT)[..., N:].double(), position, s["freq"], s["rot"]), held
    V = c["vdim"]
    if sum(n * (b + n) for b, n in lens) * H * (N + V + ROT) > 3 << 40:
        return None
    w, q, q_rot = s["w"].view(H, N + V, RANK).double(), s["q"].view(-1, H, N + ROT).double(), s["q_rot"].double()
    out, at = torch.empty((batch.n_tokens, H, V), dtype=torch.float64, device=DEV), 0
    for i, (b, n) in enumerate(lens):
        held = s["kv"][table[i, :(b + n + ps - 1) // ps]].flatten(0, 1)[:b + n].double()
        hidden = torch.arange(b + n, device=DEV)[None, :] > torch.arange(b, b + n, device=DEV)[:, None]
        for h in range(H):
            latents = held[:, :RANK]
            if n >= 64:
                z = q[at:at + n, h, :N] @ (latents @ w[h, :N].t()).t()
            else:
                z = (q[at:at + n, h, :N] @ w[h, :N]) @ latents.t()
            z = (z + q_rot[at:at + n, h] @ held[:, RANK:].t()) * s["scale"]
            p = torch.softmax(torch.where(hidden, torch.full_like(z, -math.inf), z), 1)
            out[at:at + n, h] = p @ (latents @ w[h, N:].t()) if n >= 64 else (p @ latents) @ w[h, N:].t()
        at += n
    return out.flatten(1)
