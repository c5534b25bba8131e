"""Latent attention beyond one decoded token with plain rotary positions (bf16): what KDeepseekV2Attention runs for prompts, drafted tokens and scaled rotations.

    latent_append       rotation of the queries' and the key's rotated columns (part of them, either layout, scaled), norm of the latent, the row of the token's page; one launch
    latent_attention    soft-max attention of any number of new tokens a sequence over the paged latents, in one of two forms of the same sum (csrc/latent_attn.cu):
                        "expanded": keys and values are made of the latents, W_h c, and attended to; "absorbed": the query goes to the latents, and the sum of latents to the values

The reference has both in its attention operator (archive/ktransformers/operators/attention.py:140-344 for prompts, :349-478) and the scaled rotation in operators/RoPE.py:222-326."""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional

import torch

from .. import native
from ..models.modeling_deepseek_v3 import yarn_inv_freq  # noqa: F401  (the frequencies of a scaled LatentRotation)

FORMS = {None: 0, "absorbed": 1, "expanded": 2}
LATENT, LATENT_ROT = 512, 64
_HERE, _stream = contextlib.nullcontext(), getattr(torch._C, "_cuda_getCurrentRawStream", None)      # (the current stream of a device as the C-ABI takes it)


class LatentRotation:
    """A rotation of the first `dims` columns: pairs (2 i, 2 i + 1) ("interleaved") or (i, i + dims / 2) ("halves") turn by position * inv_freq[i]; with `split` interleaved pairs come out
    in halves, as DeepSeek's caches hold them.  Cosines and sines are multiplied by `gain`.  `inv_freq`: float64, on the device of the call."""

    __slots__ = ("dims", "layout_code", "split", "gain", "inv_freq")

    def __init__(self, inv_freq: torch.Tensor, layout: str = "interleaved", split: bool = True, gain: float = 1.0):
        self.dims, self.layout_code = 2 * int(inv_freq.numel()), {"interleaved": 0, "halves": 1}[layout]
        self.split, self.gain, self.inv_freq = bool(split), float(gain), inv_freq.to(torch.float64).contiguous()


_BF16, _I32, _F64 = torch.bfloat16, torch.int32, torch.float64


def _latent_batch(what: str, T: int, dev: int, kv: torch.Tensor, width: int, batch, cache):
    """Checks what both calls share; their arguments from `pos` to the number of pages.  (A decode step's calls are bound by their host work: each tensor is asked for its sizes once.)"""
    pos, slot, seqs, table, ps, n_seqs, columns = batch.pos, batch.slot, batch.seqs, cache.page_table, cache.page_size, batch.n_seqs, cache.max_pages_per_seq
    shape = kv.shape
    if kv.dtype is not _BF16 or dev < 0:
        raise ValueError(f"{what}: CUDA tensors and a bfloat16 cache only; got {kv.dtype} on {kv.device}")
    if len(shape) not in (3, 4) or shape[1] != ps or shape[-1] != width or (len(shape) == 4 and shape[2] != 1) or not kv.is_contiguous():
        raise ValueError(f"{what}: the cache layer has to be contiguous [pages, {ps}, {width}], got {tuple(shape)}")
    if seqs is None or not (seqs.dtype is pos.dtype is slot.dtype is table.dtype is _I32):
        raise ValueError(f"{what}: needs int32 pos, slot, seqs and page table")
    (rows, portions), (seqs_stride, step), slots = seqs.shape, seqs.stride(), table.shape
    if pos.numel() < T or slot.numel() < T or rows < 2 or n_seqs > portions:
        raise ValueError(f"{what}: {T} tokens, but {pos.numel()} positions, {slot.numel()} slots; {n_seqs} portions of {tuple(seqs.shape)}")
    if not (pos.is_contiguous() and slot.is_contiguous() and table.is_contiguous()) or (step != 1 and portions > 1) or len(slots) != 2 or slots[1] != columns:
        raise ValueError(f"{what}: index rows and page table rows have to be contiguous, max_pages_per_seq = {columns} of them")
    if not (kv.get_device() == pos.get_device() == slot.get_device() == seqs.get_device() == table.get_device() == dev):
        raise ValueError(f"{what}: all tensors have to be on one device")
    return pos.data_ptr(), slot.data_ptr(), seqs.data_ptr(), seqs_stride, n_seqs, table.data_ptr(), slots[0], columns, ps, shape[0]


def _rows(what: str, name: str, t: torch.Tensor, T: int, width: int, dev: int):
    """rows of bf16 with their columns side by side: (pointer, stride)"""
    shape = t.shape
    if t.dtype is not _BF16 or len(shape) != 2 or shape[0] != T or shape[1] < width or t.get_device() != dev:
        raise ValueError(f"{what}: {name} has to be {T} rows of {width} bfloat16 values or more, got {tuple(shape)} of {t.dtype} on {t.device}")
    stride, step = t.stride()
    if step != 1 and shape[1] > 1:
        raise ValueError(f"{what}: {name} has to have its columns side by side")
    return t.data_ptr(), stride if T > 1 else width      # (one row has no other)


def _on(dev: int):
    """`dev` as the current device: kernels are launched on the current one, whatever their stream's"""
    return _HERE if dev == torch.cuda.current_device() else torch.cuda.device(dev)


def latent_append(q: torch.Tensor, kva: torch.Tensor, weight: torch.Tensor, eps: float, batch, cache, kv: torch.Tensor, heads: int, nope: int, rot=None, inv_freq: Optional[torch.Tensor] = None,
                  positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    """From the projections' rows to the turned queries [T, heads, rot_dim] and the tokens' rows of cache layer `kv` [pages, page_size, rank + rot_dim], one `ktb200_latent_append` launch.
    q [T, heads * (nope + rot_dim)]; kva [T, rank + rot_dim or more]: latent, key part; weight [rank]: the latent's norm.  rot: `LatentRotation` or anything with its dims, layout_code, split and
    gain (None: no rotation), with float64 frequencies in inv_freq (or rot.inv_freq).  batch: pos, slot [T], seqs [2, portions], n_seqs; `positions` [T] int32: the angles' where they are not
    batch.pos.  Tokens at positions behind the page table's last column are turned and written nowhere.  Rows of tokens in none of the batch's portions are left as they were (in the new
    tensor: as they came)."""
    what = "latent_append"
    T, dev, rank, width = q.shape[0], q.get_device(), weight.numel(), kv.shape[-1]
    rot_dim = width - rank
    if heads <= 0 or nope < 0 or rank <= 0 or rot_dim < 0:
        raise ValueError(f"{what}: {heads} heads of {nope} + {rot_dim}, cache rows of {width} for latents of {rank}")
    index = _latent_batch(what, T, dev, kv, width, batch, cache)
    q_ptr, q_stride = _rows(what, "q", q, T, heads * (nope + rot_dim), dev)
    kva_ptr, kva_stride = _rows(what, "kva", kva, T, width, dev)
    if weight.dtype is not _BF16 or weight.get_device() != dev or not weight.is_contiguous():
        raise ValueError(f"{what}: weight has to be contiguous bfloat16 on the queries' device, got {weight.dtype} on {weight.device}")
    dims = layout = split = 0
    gain, freq, at = 1.0, None, None
    if rot is not None and rot.dims:
        f, dims = getattr(rot, "inv_freq", None) if inv_freq is None else inv_freq, rot.dims
        if not isinstance(f, torch.Tensor) or f.numel() != dims // 2 or f.dtype is not _F64 or f.get_device() != dev or not f.is_contiguous():
            raise ValueError(f"{what}: a rotation needs {dims // 2} contiguous float64 frequencies on the queries' device")
        layout, split, gain, freq = rot.layout_code, int(getattr(rot, "split", False)), getattr(rot, "gain", 1.0), f.data_ptr()
    if positions is not None:
        if positions.dtype is not _I32 or positions.get_device() != dev or positions.numel() < T or not positions.is_contiguous():
            raise ValueError(f"{what}: positions have to be {T} contiguous int32 values on the queries' device")
        at = positions.data_ptr()
    out = q.new_empty((T, heads, rot_dim))
    a = native.LatentAppendParams(q_ptr, q_stride, heads, nope, kva_ptr, kva_stride, rank, rot_dim, weight.data_ptr(), eps, dims, layout, split, gain, freq, at, *index, kv.data_ptr(), out.data_ptr())
    with _on(dev):
        native.check(native.lib().ktb200_latent_append(C.byref(a), T, _stream(dev)))
    return out


def latent_attention(q: torch.Tensor, q_rot: torch.Tensor, kv: torch.Tensor, w: torch.Tensor, batch, cache, heads: int, nope: int, vdim: int, scale: float, form: Optional[str] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """o [T, heads * vdim] = soft-max attention of the queries [q_nope | q_rot] over the latents of cache layer `kv` [pages, page_size, 512 + 64] up to each token's position, `ktb200_latent_attn`:
    keys [W_K,h c | k_rot], values W_V,h c with w [heads * (nope + vdim), 512] (kv_b_proj's weight: every head's W_K above its W_V); q [T, heads * (nope + 64)], rows at multiples of 16 bytes, of which
    the first `nope` columns of a head are read; q_rot [T, heads, 64] as `latent_append` gives them.  nope, vdim: 64 or 128.  form: "expanded", "absorbed" (module docstring) or None, by the tokens a
    sequence has on average and batch.max_kv: one form for all portions, so that long ones and decoded tokens are better given in two calls.  batch.max_kv: no position is max_kv or more; the workspace
    of the expanded form, and of pages that are no whole 32 rows, follows max_kv times the portions.  Keys behind the page table's last column and in pages outside the pool are not seen (tokens at
    such positions see the others; a row that sees no key becomes zero).  To `out` (a view of any row stride) or a new tensor; rows of tokens in none of the batch's portions are left as they were (in
    a new tensor: as they came)."""
    what = "latent_attention"
    T, dev = q.shape[0], q.get_device()
    index = _latent_batch(what, T, dev, kv, LATENT + LATENT_ROT, batch, cache)
    q_ptr, q_stride = _rows(what, "q", q, T, heads * (nope + LATENT_ROT), dev)
    if q_rot.numel() != T * heads * LATENT_ROT or not q_rot.is_contiguous() or q_rot.dtype is not _BF16 or q_rot.get_device() != dev:
        raise ValueError(f"{what}: q_rot has to be contiguous [{T}, {heads}, {LATENT_ROT}] of bfloat16 on the queries' device, got {tuple(q_rot.shape)} of {q_rot.dtype} on {q_rot.device}")
    if w.shape != (heads * (nope + vdim), LATENT) or not w.is_contiguous() or w.dtype is not _BF16 or w.get_device() != dev:
        raise ValueError(f"{what}: w has to be contiguous [{heads * (nope + vdim)}, {LATENT}] of bfloat16 on the queries' device, got {tuple(w.shape)} of {w.dtype} on {w.device}")
    if form not in FORMS:
        raise ValueError(f"{what}: form {form!r}: one of {', '.join(map(repr, FORMS))}")
    if out is None:
        out = q.new_empty((T, heads * vdim))
    elif out.shape != (T, heads * vdim):
        raise ValueError(f"{what}: out has to be [{T}, {heads * vdim}], got {tuple(out.shape)}")
    out_ptr, out_stride = _rows(what, "out", out, T, heads * vdim, dev)
    a = native.LatentAttnParams(q_ptr, q_stride, q_rot.data_ptr(), heads, nope, vdim, w.data_ptr(), scale, FORMS[form], *index, kv.data_ptr(), out_ptr, out_stride)
    lib, ref, keys = native.lib(), C.byref(a), batch.max_kv
    with _on(dev):
        nbytes = lib.ktb200_latent_attn_workspace(ref, T, keys)
        ws = q.new_empty(nbytes + 512, dtype=torch.uint8) if nbytes else None      # (the allocator's blocks begin at multiples of 512 bytes)
        native.check(lib.ktb200_latent_attn(ref, T, keys, (ws.data_ptr() + 1023) // 1024 * 1024 if nbytes else None, nbytes, _stream(dev)))
    return out
