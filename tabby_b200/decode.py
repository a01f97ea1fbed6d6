"""Decode steps that carry several hypotheses a sequence: beam search and drafted trees.

The calls of include/tabby_decode.h on torch tensors. All of them are asynchronous on the
current stream of the tensors' device, take and give device tensors, allocate through
PyTorch (so they can be captured in a CUDA graph) and keep nothing between calls.

Beam search, one step:

    step = beam_step(logits.view(batch, beams, vocab), scores, finished=finished, eos_id=eos)
    reorder_states(caches, step.parents, lengths)        # the beams' caches follow them
    reorder_states([history], step.parents)              # and their tokens

Drafted trees, one step (slot 0 of a tree is the sequence's last token):

    o = tree_attention(q, k_cache, v_cache, lengths, parents)      # in every layer
    sampler.sample_rows_async(logits, params, uniforms, out)       # a row for every slot
    sampled = out.view(torch.int32).view(batch, nodes, 12)[..., 0] # the outcomes' ids
    step = tree_accept(sampled, tokens, parents, lengths, caches)
    lengths = step.lengths                                # next root: step.next_tokens
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import _lib
from ._lib import StateLayout, TreeAttentionArgs, check_decode, decode_lib

_DTYPES = {torch.float32: _lib.TABBY_F32, torch.bfloat16: _lib.TABBY_BF16,
           torch.float16: _lib.TABBY_F16}


class BeamStep(NamedTuple):
    """beam_step's outputs: [batch, n_out] each, status [batch]."""

    scores: torch.Tensor    # float32 log-probabilities, falling
    parents: torch.Tensor   # int32 beam each continues, -1: no candidate
    tokens: torch.Tensor    # int32, -1: no candidate
    finished: torch.Tensor  # bool
    status: torch.Tensor    # int32 tabby_status of each prompt


class TreeAccept(NamedTuple):
    """tree_accept's outputs, int32."""

    path: torch.Tensor         # [batch, nodes] accepted slots, then -1
    counts: torch.Tensor       # [batch]
    next_tokens: torch.Tensor  # [batch]
    lengths: torch.Tensor      # [batch] the caches' new lengths


def _need(x, name: str, dtypes, shape, device) -> None:
    """Type, shape (None: any size) and device of an argument."""
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(map(str, dtypes))}, got {x.dtype}")
    if x.dim() != len(shape) or any(w is not None and w != g for w, g in zip(shape, x.shape)):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} must live on {device}, got {x.device}")


def _cuda(x, name: str) -> torch.device:
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return x.device


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


_I32 = (torch.int32,)


@lru_cache(maxsize=256)
def _beam_workspace(batch: int, beams: int, vocab: int, n_out: int) -> int:
    n = ctypes.c_size_t()
    check_decode(decode_lib().tabby_beam_workspace_bytes(batch, beams, vocab, n_out,
                                                         ctypes.byref(n)))
    return n.value


def beam_step(logits: torch.Tensor, scores: torch.Tensor, n_out: Optional[int] = None, *,
              finished: Optional[torch.Tensor] = None, eos_id: int = -1) -> BeamStep:
    """Beam search's selection: of all continuations (beam, token) of a prompt the ``n_out``
    (default: one a beam) with the largest log-probability
    ``scores[beam] + log_softmax(logits[beam])[token]``, ties to the lower beam, then token.

    logits [batch, beams, vocab] float32, bfloat16 or float16 (rows may be strided or shared),
    scores [batch, beams] float32. -inf logits are banned tokens, -inf scores dead beams; a
    ``finished`` beam [batch, beams] goes on with ``eos_id`` at its score. Missing
    continuations have parent and token -1 and score -inf. A prompt whose live beams hold NaN
    or +inf has status TABBY_EINPUT and no continuations.
    """
    device = _cuda(logits, "logits")
    if logits.dim() != 3:
        raise ValueError("logits must be [batch, beams, vocab]")
    if logits.dtype not in _DTYPES:
        raise TypeError("logits must be float32, bfloat16 or float16")
    batch, beams, vocab = logits.shape
    if vocab > 1 and logits.stride(2) != 1:
        logits = logits.contiguous()
    _need(scores, "scores", (torch.float32,), (batch, beams), device)
    scores = scores.contiguous()
    if finished is not None:
        _need(finished, "finished", (torch.bool, torch.uint8), (batch, beams), device)
        finished = finished.contiguous()
    n_out = beams if n_out is None else int(n_out)
    need = _beam_workspace(batch, beams, vocab, n_out)
    new = torch.empty
    r = BeamStep(new((batch, n_out), dtype=torch.float32, device=device),
                 new((batch, n_out), dtype=torch.int32, device=device),
                 new((batch, n_out), dtype=torch.int32, device=device),
                 new((batch, n_out), dtype=torch.bool, device=device),
                 new((batch,), dtype=torch.int32, device=device))
    work = new((need,), dtype=torch.uint8, device=device)
    check_decode(decode_lib().tabby_beam_step_async(
        device.index, logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0),
        logits.stride(1), batch, beams, vocab, scores.data_ptr(),
        None if finished is None else finished.data_ptr(), eos_id, n_out, r.scores.data_ptr(),
        r.parents.data_ptr(), r.tokens.data_ptr(), r.finished.data_ptr(), r.status.data_ptr(),
        work.data_ptr(), need, _stream(device)))
    return r


@lru_cache(maxsize=256)
def _layout(shape: tuple, stride: tuple, size: int, with_entries: bool) -> StateLayout:
    """The layout of rows [rows, ...] of `size`-byte elements. With entries the shape is
    [rows, heads, entries, dim]; else the axes behind the first are merged where memory
    allows, and three may remain."""
    axes = [(n, s) for n, s in zip(shape[1:], stride[1:])]
    if with_entries:
        if len(axes) != 3:
            raise ValueError("states with lengths must be [rows, heads, entries, dim]")
    else:
        merged: list = []
        for n, s in axes:
            if n == 1:
                continue
            if merged and merged[-1][1] == n * s:
                merged[-1] = (merged[-1][0] * n, s)
            else:
                merged.append((n, s))
        if not merged or merged[-1][1] != 1:
            merged.append((1, 1))
        if len(merged) > 3:
            raise ValueError("a state's rows may have at most two strides beside the innermost")
        axes = [(1, 0)] * (3 - len(merged)) + merged
    (segments, seg), (entries, ent), (dim, inner) = axes
    if dim > 1 and inner != 1:
        raise ValueError("a state's innermost axis must be contiguous")
    return StateLayout(stride[0] * size if shape[0] > 1 else 0, seg * size, ent * size,
                       dim * size, segments, entries)


def _states(states: Union[torch.Tensor, Sequence[torch.Tensor]], rows: int, with_entries: bool,
            device, name: str):
    """(layout, pointers) groups of states with one layout each."""
    if isinstance(states, torch.Tensor):
        if states.dim() < 2:
            raise ValueError(f"stacked {name} must be [states, rows, ...]")
        if states.device != device:
            raise ValueError(f"{name} must live on {device}, got {states.device}")
        if states.shape[1] != rows:
            raise ValueError(f"{name} must have {rows} rows, got {states.shape[1]}")
        if states.numel() == 0:
            return []
        n, step, size = states.shape[0], states.stride(0), states.element_size()
        if n > 1 and step == 0:
            raise ValueError(f"{name} overlap")
        p = states.data_ptr()
        return [(_layout(states.shape[1:], states.stride()[1:], size, with_entries),
                 [p + i * step * size for i in range(n)])]
    groups: dict = {}
    for x in states:
        if x.device != device:
            raise ValueError(f"{name} must live on {device}, got {x.device}")
        if x.dim() < 1 or x.shape[0] != rows:
            raise ValueError(f"{name} must have {rows} rows, got shape {tuple(x.shape)}")
        if x.numel():
            groups.setdefault((x.shape, x.stride(), x.element_size()), []).append(x.data_ptr())
    return [(_layout(shape, stride, size, with_entries), p)
            for (shape, stride, size), p in groups.items()]


def reorder_states(states: Union[torch.Tensor, Sequence[torch.Tensor]], parents: torch.Tensor,
                   lengths: Optional[torch.Tensor] = None) -> None:
    """Moves the beams' states in place so that row b * beams + i holds what row
    b * beams + parents[b, i] held (parents [batch, beams] int32, as beam_step gives them; a
    row whose parent is outside [0, beams) stays).

    states: tensors [batch * beams, ...] of any type, or one tensor that stacks them along
    its first axis. With ``lengths`` ([batch] int32) they are caches [batch * beams, heads,
    entries, dim] (any strides, dim contiguous) and only the first lengths[b] entries move.
    """
    device = _cuda(parents, "parents")
    _need(parents, "parents", _I32, (None, None), device)
    batch, beams = parents.shape
    parents = parents.contiguous()
    if lengths is not None:
        _need(lengths, "lengths", _I32, (batch,), device)
        lengths = lengths.contiguous()
    for layout, p in _states(states, batch * beams, lengths is not None, device, "states"):
        check_decode(decode_lib().tabby_states_reorder_async(
            device.index, (ctypes.c_void_p * len(p))(*p), len(p), layout, batch, beams,
            parents.data_ptr(), None if lengths is None else lengths.data_ptr(),
            _stream(device)))


@lru_cache(maxsize=256)
def _tree_workspace(batch: int, nodes: int, heads: int, kv_heads: int, dim: int) -> int:
    n = ctypes.c_size_t()
    check_decode(decode_lib().tabby_tree_workspace_bytes(batch, nodes, heads, kv_heads, dim,
                                                         ctypes.byref(n)))
    return n.value


def _strides(x: torch.Tensor):
    """Strides of the outer axes, 0 for an axis of one."""
    return [s if n > 1 else 0 for n, s in zip(x.shape[:-1], x.stride()[:-1])]


def _fits(x: torch.Tensor) -> bool:
    """Rows of the last axis contiguous, 16-byte aligned."""
    return (x.stride(-1) == 1 and x.data_ptr() % 16 == 0
            and all(s % 8 == 0 for s in _strides(x)))


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   lengths: torch.Tensor, parents: torch.Tensor,
                   scale: Optional[float] = None) -> torch.Tensor:
    """Attention of drafted trees over a cache: slot j of sequence b attends to the
    lengths[b] entries of its context, to itself and to its ancestors in the tree, whose keys
    and values lie at entries lengths[b] + slot. Returns [batch, nodes, heads, dim] in q's
    type; slots that are not in use give 0.

    q [batch, nodes, heads, dim] bfloat16 or float16; k_cache and v_cache [batch, kv_heads,
    entries, dim] in any strides with dim contiguous (16-byte aligned rows); lengths [batch]
    int32; parents [batch, nodes] or [nodes] int32, -1 for a root, lower for unused slots.
    nodes <= 64, dim a multiple of 8 up to 128, heads a multiple of kv_heads. scale defaults
    to dim ** -0.5. One slot (parents -1) is the ordinary decode step.
    """
    device = _cuda(q, "q")
    if q.dim() != 4:
        raise ValueError("q must be [batch, nodes, heads, dim]")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("q must be bfloat16 or float16")
    batch, nodes, heads, dim = q.shape
    _need(k_cache, "k_cache", (q.dtype,), (batch, None, None, dim), device)
    _need(v_cache, "v_cache", (q.dtype,), k_cache.shape, device)
    _need(lengths, "lengths", _I32, (batch,), device)
    if parents.dim() == 1:
        parents = parents.expand(batch, nodes) if parents.shape[0] == nodes else parents
    _need(parents, "parents", _I32, (batch, nodes), device)
    if nodes > 1 and parents.stride(1) != 1:
        parents = parents.contiguous()
    kv_heads, entries = k_cache.shape[1], k_cache.shape[2]
    need = _tree_workspace(batch, nodes, heads, kv_heads, dim)
    if not _fits(q):
        q = q.contiguous()
    if not _fits(k_cache) or not _fits(v_cache):
        raise ValueError("the caches' rows must be contiguous and 16-byte aligned")
    lengths = lengths.contiguous()
    out = torch.empty((batch, nodes, heads, dim), dtype=q.dtype, device=device)
    if batch == 0:
        return out
    work = torch.empty((need,), dtype=torch.uint8, device=device)
    args = TreeAttentionArgs(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), *_strides(q),
        *_strides(k_cache), *_strides(v_cache), *_strides(out), lengths.data_ptr(),
        parents.data_ptr(), parents.stride(0) if batch > 1 else 0, _DTYPES[q.dtype], batch,
        nodes, heads, kv_heads, dim, entries, dim ** -0.5 if scale is None else float(scale),
        work.data_ptr(), need)
    check_decode(decode_lib().tabby_tree_attention_async(device.index, args, _stream(device)))
    return out


def tree_accept(sampled: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor,
                lengths: torch.Tensor,
                caches: Union[torch.Tensor, Sequence[torch.Tensor]] = ()) -> TreeAccept:
    """Walks every tree from its root (slot 0) along the drafted tokens that the sampled ones
    agree with and, in place, moves the accepted slots' cache entries up to lengths[b].

    sampled [batch, nodes] int32 in any strides: the token chosen after each slot; tokens
    [batch, nodes] int32: the drafted ones; parents [batch, nodes] or [nodes] as in
    tree_attention; caches: [batch, heads, entries, dim] each, or one tensor that stacks
    them. ``lengths`` itself is not changed: the new ones are returned.
    """
    device = _cuda(tokens, "tokens")
    _need(tokens, "tokens", _I32, (None, None), device)
    batch, nodes = tokens.shape
    _need(sampled, "sampled", _I32, (batch, nodes), device)
    if parents.dim() == 1:
        parents = parents.expand(batch, nodes) if parents.shape[0] == nodes else parents
    _need(parents, "parents", _I32, (batch, nodes), device)
    _need(lengths, "lengths", _I32, (batch,), device)
    tokens, lengths = tokens.contiguous(), lengths.contiguous()
    if nodes > 1 and parents.stride(1) != 1:
        parents = parents.contiguous()
    groups = _states(caches, batch, True, device, "caches")
    if len(groups) > 1:
        raise ValueError("the caches must share one layout")
    layout, p = groups[0] if groups else (None, [])
    new = torch.empty
    r = TreeAccept(new((batch, nodes), dtype=torch.int32, device=device),
                   new((batch,), dtype=torch.int32, device=device),
                   new((batch,), dtype=torch.int32, device=device),
                   new((batch,), dtype=torch.int32, device=device))
    check_decode(decode_lib().tabby_tree_accept_async(
        device.index, sampled.data_ptr(), sampled.stride(0), sampled.stride(1),
        tokens.data_ptr(), parents.data_ptr(), parents.stride(0) if batch > 1 else 0, batch,
        nodes, lengths.data_ptr(), r.path.data_ptr(), r.counts.data_ptr(),
        r.next_tokens.data_ptr(), r.lengths.data_ptr(), (ctypes.c_void_p * len(p))(*p), len(p),
        layout, _stream(device)))
    return r


__all__ = ["BeamStep", "TreeAccept", "beam_step", "reorder_states", "tree_accept",
           "tree_attention"]
