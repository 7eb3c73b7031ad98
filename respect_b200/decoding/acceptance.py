"""Greedy token choice, token log probabilities and the acceptance walk over a verified trie.

Mirror of ``respect.decoding.acceptance`` (respect/decoding/acceptance.py:11-46).
`greedy_token` runs on the device (rb_greedy_token): the action-vocabulary range
is skipped inside the argmax instead of materialising a masked fp32 clone of
the [q, vocab] logits. `token_logprobs` (rb_token_logprobs) says how likely given
tokens were under the same exclusion, with the entropy and the best alternatives.
"""
from __future__ import annotations

import functools
from typing import Callable, NamedTuple

import torch

from respect_b200 import _lib
from respect_b200.candidates.trie import Trie


def mask_action_vocab(logits: torch.Tensor, offset: int, size: int) -> torch.Tensor:
    """fp32 copy of the logits with the trajectory-token range set to -inf."""
    masked = logits.float().clone()
    masked[:, offset:offset + size] = float("-inf")
    return masked


def greedy_token(logits: torch.Tensor, offset: int, size: int) -> torch.Tensor:
    """Row-wise argmax with [offset, offset + size) excluded; int64 [rows] on the logits' device."""
    x = logits if logits.stride(-1) == 1 else logits.contiguous()
    x2 = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    M, V = x2.shape
    out = torch.empty(M, dtype=torch.int64, device=x.device)
    _lib.call("rb_greedy_token", x2.data_ptr(), _lib.dtype_code(x2.dtype), x2.stride(0), M, V,
              int(offset), int(size), out.data_ptr(), _lib.stream_of(x2))
    return out.reshape(x.shape[:-1])


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                 # fp32 [rows]: log softmax at the given token
    entropy: torch.Tensor                 # fp32 [rows], in nats
    top_logprobs: torch.Tensor | None     # fp32 [rows, top], descending
    top_ids: torch.Tensor | None          # int64 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, offset: int = 0,
                   size: int = 0) -> TokenLogprobs:
    """Log probability of ``tokens`` (int64, one per row of ``logits`` [..., vocab], fp32 or bf16),
    the rows' entropy and their ``top`` (at most 32) best entries, ties to the lowest index, with
    [offset, offset + size) excluded as in greedy_token (-inf for an excluded token; excluded
    entries follow the others among the alternatives). A row holding NaN or +inf, or nothing but
    -inf, gives NaN, and so does a token outside the vocabulary."""
    shape, dtype = logits.shape, logits.dtype
    if not shape or (dtype is not torch.float32 and dtype is not torch.bfloat16):
        raise TypeError("token_logprobs takes fp32 or bf16 logits [..., vocab]")
    V, lead = shape[-1], shape[:-1]
    if tokens.dtype is not torch.int64 or tokens.shape != lead or tokens.get_device() != logits.get_device():
        raise ValueError(f"tokens must be int64 {tuple(lead)} on {logits.device}")
    if not 0 <= top <= min(_lib.LOGPROBS_MAX_TOP, V):
        raise ValueError(f"top must be between 0 and {min(_lib.LOGPROBS_MAX_TOP, V)}")
    if offset < 0 or size < 0 or V == 0:
        raise ValueError("token_logprobs: bad excluded range or empty vocabulary")
    x = logits if V == 1 or logits.stride(-1) == 1 else logits.contiguous()
    if len(lead) != 1:
        x, tokens = x.reshape(-1, V), tokens.reshape(-1)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    M, dev = x.shape[0], x.device
    if M > 1 and x.stride(0) < V:
        x = x.contiguous()                   # rows that overlap, as of an expanded tensor
    if top:
        lp, ent, tlp = torch.empty((2 + top) * M, dtype=torch.float32, device=dev).split_with_sizes((M, M, top * M))
        tlp, ids = tlp.view(*lead, top), torch.empty((*lead, top), dtype=torch.int64, device=dev)
        tlp_at, ids_at = tlp.data_ptr(), ids.data_ptr()
    else:
        lp, ent = torch.empty(2 * M, dtype=torch.float32, device=dev).split_with_sizes((M, M))
        tlp = ids = tlp_at = ids_at = None
    nbytes = _scratch_bytes(M, V, top)
    ws = _lib.scratch(x, nbytes)
    _lib.launch("rb_token_logprobs", x, x.data_ptr(), _lib.dtype_code(dtype), x.stride(0) if M > 1 else V, M, V,
                tokens.data_ptr(), min(offset, V), min(size, V), top, lp.data_ptr(), ent.data_ptr(), tlp_at, ids_at,
                None if ws is None else ws.data_ptr(), nbytes)
    if len(lead) != 1:
        lp, ent = lp.view(lead), ent.view(lead)
    return TokenLogprobs(lp, ent, tlp, ids)


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(M: int, V: int, top: int) -> int:
    return _lib.lib().rb_token_logprobs_workspace(M, V, top)


def walk(tree: Trie, first: int, cap: int, eos: int,
         pick: Callable[[list, int], int]) -> tuple[list, list, int]:
    """Follow the trie from the root holding `first` while each node's token
    matches the target's choice after its parent.

    `pick(accepted, node)` is the target's token after `node`. Stops at EOS, at
    a mismatch, at a leaf, or after `cap` tokens. Returns (node path, accepted
    tokens, correction token): the correction is the target's last choice (or
    `first` when nothing was accepted).
    """
    path: list = []
    accepted: list = []
    correction = first
    node = tree.roots.get(first)
    while node is not None and len(accepted) < cap:
        nd = tree.nodes[node]
        path.append(node)
        accepted.append(nd.token)
        if nd.token == eos:
            break
        correction = pick(accepted, node)
        node = nd.children.get(correction)
    return path, accepted, correction
