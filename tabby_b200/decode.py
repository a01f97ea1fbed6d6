"""Decode steps that carry several hypotheses a sequence: beam search and drafted trees.

The calls of include/tabby_decode.h on torch tensors. All of them are asynchronous on the
current stream of the tensors' device, take and give device tensors, allocate through
PyTorch (so they can be captured in a CUDA graph) and keep nothing between calls. They take no
part in autograd; the calls that work in place do not count the tensors' versions up, so autograd
does not notice that a tensor it has saved was moved.

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

import importlib.machinery
import importlib.util
import os
from typing import NamedTuple, Optional, Sequence, Union

import torch

from ._lib import DECODE_TORCH_PATH, StateLayout

_extension = None


def extension():
    """The compiled half of this module (csrc/decode_torch.cpp); raises if it is missing."""
    global _extension
    if _extension is None:
        if not os.path.exists(DECODE_TORCH_PATH):
            raise RuntimeError(
                f"{DECODE_TORCH_PATH} is missing; build it with `python -m tabby_b200.build`")
        loader = importlib.machinery.ExtensionFileLoader("tabby_decode_torch", DECODE_TORCH_PATH)
        spec = importlib.util.spec_from_loader("tabby_decode_torch", loader)
        _extension = importlib.util.module_from_spec(spec)
        loader.exec_module(_extension)
    return _extension


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


def beam_step(logits: torch.Tensor, scores: torch.Tensor, n_out: Optional[int] = None, *,
              finished: Optional[torch.Tensor] = None, eos_id: int = -1) -> BeamStep:
    """Beam search's selection: of all continuations (beam, token) of a prompt the ``n_out``
    (default: one a beam) with the largest log-probability
    ``scores[beam] + log_softmax(logits[beam])[token]``, ties to the lower beam, then token.

    logits [batch, beams, vocab] float32, bfloat16 or float16 (rows may be strided or shared),
    scores [batch, beams] float32. -inf logits are banned tokens, -inf scores dead beams; a
    ``finished`` beam [batch, beams] goes on with ``eos_id`` at its score. Missing
    continuations have parent and token -1 and score -inf. Keys of different beams closer than
    about 1e-12 may change places unless the beams are alike. A prompt whose live beams hold NaN
    or +inf has status TABBY_EINPUT and no continuations.
    """
    return BeamStep(*extension().beam_step(logits, scores, n_out, finished, eos_id))


def _layout(shape: Sequence[int], stride: Sequence[int], size: int,
            with_entries: bool) -> StateLayout:
    """The layout that rows [rows, ...] of `size`-byte elements have for the library."""
    return StateLayout(*extension().layout(shape, stride, size, with_entries))


def reorder_states(states: Union[torch.Tensor, Sequence[torch.Tensor]], parents: torch.Tensor,
                   lengths: Optional[torch.Tensor] = None) -> None:
    """Moves the beams' states in place so that row b * beams + i holds what row
    b * beams + parents[b, i] held (parents [batch, beams] int32, as beam_step gives them; a
    row whose parent is outside [0, beams) stays).

    states: tensors [batch * beams, ...] of any type, or one tensor that stacks them along
    its first axis. With ``lengths`` ([batch] int32) they are caches [batch * beams, heads,
    entries, dim] (any strides, dim contiguous) and only the first lengths[b] entries move.
    No state may overlap another. All are checked before the first is moved.
    """
    extension().reorder_states(states, parents, lengths)


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
    to dim ** -0.5. One slot (parents -1) is the ordinary decode step. The softmax is in float32;
    its weights are rounded to the caches' type where they meet the values, the output once.
    """
    return extension().tree_attention(q, k_cache, v_cache, lengths, parents, scale)


def tree_accept(sampled: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor,
                lengths: torch.Tensor,
                caches: Union[torch.Tensor, Sequence[torch.Tensor]] = ()) -> TreeAccept:
    """Walks every tree from its root (slot 0) along the drafted tokens that the sampled ones
    agree with and, in place, moves the accepted slots' cache entries up to lengths[b].

    sampled [batch, nodes] int32 in any strides: the token chosen after each slot; tokens
    [batch, nodes] int32: the drafted ones; parents [batch, nodes] or [nodes] as in
    tree_attention; caches: [batch, heads, entries, dim] each, or one tensor that stacks
    them, all of one shape, type and strides. ``lengths`` itself is not changed: the new ones are returned.
    """
    return TreeAccept(*extension().tree_accept(sampled, tokens, parents, lengths, caches))


__all__ = ["BeamStep", "TreeAccept", "beam_step", "reorder_states", "tree_accept",
           "tree_attention"]
