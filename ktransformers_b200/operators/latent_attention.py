"""Latent attention beyond one decoded token with plain rotary positions (bf16): what KDeepseekV2Attention runs for prompts, drafted tokens and scaled rotations.

    latent_append       rotation of the queries' and the key's rotated columns (part of them, either layout, scaled), norm of the latent, the row of the token's page; one launch
    latent_attention    soft-max attention of any number of new tokens a sequence over the paged latents, in one of two forms of the same sum (csrc/latent_attn.cu):
                        "expanded": keys and values are made of the latents, W_h c, and attended to; "absorbed": the query goes to the latents, and the sum of latents to the values

The reference has both in its attention operator (archive/ktransformers/operators/attention.py:140-344 for prompts, :349-478) and the scaled rotation in operators/RoPE.py:222-326."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from .. import native
from ..models.modeling_deepseek_v3 import yarn_inv_freq  # noqa: F401  (the frequencies of a scaled LatentRotation)
from .base_operator import device_of, stream_of

FORMS = {None: 0, "absorbed": 1, "expanded": 2}
LATENT, LATENT_ROT = 512, 64


class LatentRotation:
    """A rotation of the first `dims` columns: pairs (2 i, 2 i + 1) ("interleaved") or (i, i + dims / 2) ("halves") turn by position * inv_freq[i]; with `split` interleaved pairs come out
    in halves, as DeepSeek's caches hold them.  Cosines and sines are multiplied by `gain`.  `inv_freq`: float64, on the device of the call."""

    __slots__ = ("dims", "layout_code", "split", "gain", "inv_freq")

    def __init__(self, inv_freq: torch.Tensor, layout: str = "interleaved", split: bool = True, gain: float = 1.0):
        self.dims, self.layout_code = 2 * int(inv_freq.numel()), {"interleaved": 0, "halves": 1}[layout]
        self.split, self.gain, self.inv_freq = bool(split), float(gain), inv_freq.to(torch.float64).contiguous()


def _latent_batch(what: str, T: int, dev, kv: torch.Tensor, width: int, batch, cache):
    """Checks what both calls share; their arguments from `pos` to the number of pages"""
    pos, slot, seqs, table, ps, n_seqs = batch.pos, batch.slot, batch.seqs, cache.page_table, cache.page_size, batch.n_seqs
    if kv.dtype is not torch.bfloat16 or dev.type != "cuda":
        raise ValueError(f"{what}: CUDA tensors and a bfloat16 cache only; got {kv.dtype} on {dev}")
    if not kv.is_contiguous() or kv.dim() not in (3, 4) or kv.shape[1] != ps or kv.shape[-1] != width or kv.numel() != kv.shape[0] * ps * width:
        raise ValueError(f"{what}: the cache layer has to be contiguous [pages, {ps}, {width}], got {tuple(kv.shape)}")
    if seqs is None or not (seqs.dtype is pos.dtype is slot.dtype is table.dtype is torch.int32):
        raise ValueError(f"{what}: needs int32 pos, slot, seqs and page table")
    if pos.shape[0] < T or slot.shape[0] < T or seqs.shape[0] < 2 or n_seqs > seqs.shape[1]:
        raise ValueError(f"{what}: {T} tokens, but {pos.shape[0]} positions, {slot.shape[0]} slots; {n_seqs} portions of {tuple(seqs.shape)}")
    if pos.stride(0) != 1 or slot.stride(0) != 1 or seqs.stride(1) != 1 or table.dim() != 2 or not table.is_contiguous() or table.shape[1] != cache.max_pages_per_seq:
        raise ValueError(f"{what}: index rows and page table rows have to be contiguous, max_pages_per_seq = {cache.max_pages_per_seq} of them")
    if not (kv.device == pos.device == slot.device == seqs.device == table.device == dev):
        raise ValueError(f"{what}: all tensors have to be on one device")
    return pos.data_ptr(), slot.data_ptr(), seqs.data_ptr(), seqs.stride(0), n_seqs, table.data_ptr(), table.shape[0], table.shape[1], ps, kv.shape[0]


def _rows(what: str, name: str, t: torch.Tensor, T: Optional[int], width: int, dev):
    """rows of bf16 with their columns side by side: (pointer, stride)"""
    if t.dim() != 2 or t.dtype is not torch.bfloat16 or t.device != dev or (T is not None and t.shape[0] != T) or t.shape[1] < width or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{what}: {name} has to be rows of {width} bfloat16 values side by side on {dev}, got {tuple(t.shape)} of {t.dtype} on {t.device}")
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def latent_append(q: torch.Tensor, kva: torch.Tensor, weight: torch.Tensor, eps: float, batch, cache, kv: torch.Tensor, heads: int, nope: int, rot=None, inv_freq: Optional[torch.Tensor] = None,
                  positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    """From the projections' rows to the turned queries [T, heads, rot_dim] and the tokens' rows of cache layer `kv` [pages, page_size, rank + rot_dim], one `ktb200_latent_append` launch.
    q [T, heads * (nope + rot_dim)]; kva [T, rank + rot_dim or more]: latent, key part; weight [rank]: the latent's norm.  rot: `LatentRotation` or anything with its dims, layout_code, split and
    gain (None: no rotation), with float64 frequencies in inv_freq (or rot.inv_freq).  batch: pos, slot [T], seqs [2, portions], n_seqs; `positions` [T] int32: the angles' where they are not
    batch.pos.  Rows of tokens in none of the batch's portions are left as they were (in the new tensor: as they came)."""
    what = "latent_append"
    T, dev, rank = q.shape[0], q.device, weight.numel()
    width = kv.shape[-1]
    rot_dim = width - rank
    if heads <= 0 or nope < 0 or rank <= 0 or rot_dim < 0:
        raise ValueError(f"{what}: {heads} heads of {nope} + {rot_dim}, cache rows of {width} for latents of {rank}")
    index = _latent_batch(what, T, dev, kv, width, batch, cache)
    q_ptr, q_stride = _rows(what, "q", q, T, heads * (nope + rot_dim), dev)
    kva_ptr, kva_stride = _rows(what, "kva", kva, T, width, dev)
    if weight.dtype is not torch.bfloat16 or weight.device != dev or not weight.is_contiguous():
        raise ValueError(f"{what}: weight has to be contiguous bfloat16 on {dev}")
    dims = layout = split = 0
    gain, freq, at = 1.0, None, None
    if rot is not None and rot.dims:
        f = rot.inv_freq if inv_freq is None and hasattr(rot, "inv_freq") else inv_freq
        if f is None or torch.is_tensor(f) is False or f.numel() != rot.dims // 2 or f.dtype is not torch.float64 or f.device != dev or not f.is_contiguous():
            raise ValueError(f"{what}: a rotation needs {rot.dims // 2} contiguous float64 frequencies on {dev}")
        dims, layout, split, gain, freq = rot.dims, rot.layout_code, int(getattr(rot, "split", False)), float(getattr(rot, "gain", 1.0)), f.data_ptr()
    if positions is not None:
        if positions.dtype is not torch.int32 or positions.device != dev or positions.shape[0] < T or positions.stride(0) != 1:
            raise ValueError(f"{what}: positions have to be {T} contiguous int32 values on {dev}")
        at = positions.data_ptr()
    out = q.new_empty((T, heads, rot_dim))
    a = native.LatentAppendParams(q_ptr, q_stride, heads, nope, kva_ptr, kva_stride, rank, rot_dim, weight.data_ptr(), eps, dims, layout, split, gain, freq, at, *index, kv.data_ptr(), out.data_ptr())
    with device_of(dev):
        native.check(native.lib().ktb200_latent_append(C.byref(a), T, stream_of(dev)))
    return out


def latent_attention(q: torch.Tensor, q_rot: torch.Tensor, kv: torch.Tensor, w: torch.Tensor, batch, cache, heads: int, nope: int, vdim: int, scale: float, form: Optional[str] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """o [T, heads * vdim] = soft-max attention of the queries [q_nope | q_rot] over the latents of cache layer `kv` [pages, page_size, 512 + 64] up to each token's position, `ktb200_latent_attn`:
    keys [W_K,h c | k_rot], values W_V,h c with w [heads * (nope + vdim), 512] (kv_b_proj's weight: every head's W_K above its W_V); q [T, heads * (nope + 64)] of any row stride, of which the
    first `nope` columns of a head are read; q_rot [T, heads, 64] as `latent_append` gives them.  nope, vdim: 64 or 128.  form: "expanded", "absorbed" (module docstring) or None, by
    the tokens a sequence has on average.  batch.max_kv: no position is max_kv or more.  To `out` (a view of any row stride) or a new tensor; rows of tokens in none of the batch's portions are
    left as they were (in a new tensor: as they came)."""
    what = "latent_attention"
    T, dev = q.shape[0], q.device
    index = _latent_batch(what, T, dev, kv, LATENT + LATENT_ROT, batch, cache)
    q_ptr, q_stride = _rows(what, "q", q, T, heads * (nope + LATENT_ROT), dev)
    if q_rot.numel() != T * heads * LATENT_ROT or not q_rot.is_contiguous() or q_rot.dtype is not torch.bfloat16 or q_rot.device != dev:
        raise ValueError(f"{what}: q_rot has to be contiguous [{T}, {heads}, {LATENT_ROT}] of bfloat16 on {dev}, got {tuple(q_rot.shape)} of {q_rot.dtype} on {q_rot.device}")
    if tuple(w.shape) != (heads * (nope + vdim), LATENT) or not w.is_contiguous() or w.dtype is not torch.bfloat16 or w.device != dev:
        raise ValueError(f"{what}: w has to be contiguous [{heads * (nope + vdim)}, {LATENT}] of bfloat16 on {dev}, got {tuple(w.shape)} of {w.dtype} on {w.device}")
    if form not in FORMS:
        raise ValueError(f"{what}: form {form!r}: one of {', '.join(map(repr, FORMS))}")
    if out is None:
        out = q.new_empty((T, heads * vdim))
    elif out.shape[0] != T or out.dim() != 2 or out.shape[1] != heads * vdim:
        raise ValueError(f"{what}: out has to be [{T}, {heads * vdim}], got {tuple(out.shape)}")
    out_ptr, out_stride = _rows(what, "out", out, T, heads * vdim, dev)
    a = native.LatentAttnParams(q_ptr, q_stride, q_rot.data_ptr(), heads, nope, vdim, w.data_ptr(), scale, FORMS[form], *index, kv.data_ptr(), out_ptr, out_stride)
    lib, ref, keys = native.lib(), C.byref(a), batch.max_kv
    with device_of(dev):
        nbytes = lib.ktb200_latent_attn_workspace(ref, T, keys)
        ws = q.new_empty(nbytes + 512, dtype=torch.uint8) if nbytes else None      # (the allocator's blocks begin at multiples of 512 bytes)
        native.check(lib.ktb200_latent_attn(ref, T, keys, (ws.data_ptr() + 1023) // 1024 * 1024 if nbytes else None, nbytes, stream_of(dev)))
    return out
