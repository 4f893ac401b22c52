"""Speculative decoding over a paged 16-bit cache: trees of drafted tokens, and which of them stay.

The reference decodes one token at a time (fade/cache.py:347-379); here a step takes a row's
last known token and drafted ones behind it, a chain or a tree, through ``paged_append`` and
``paged_attention`` (mask ``"tree"``) at once.  ``draft_tree`` gives what that needs from the
tokens' parents, ``verify_drafts`` which tokens the target's probabilities keep, and
``TokenPagePool.accept`` the cache with those alone.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from .. import _lib


@dataclass
class DraftTree:
    """What ``draft_tree`` writes (int32, on the GPU).

    ``bits`` [tokens, words]: for each token the row's tokens that it sees, its ancestors and itself,
    number j as bit j % 32 of word j / 32 (``paged_attention``'s ``tree``).  ``depth`` [tokens]: its
    ancestors' number.  ``positions`` [tokens]: its rotary position, the row's tokens ahead of
    the drafted ones plus the depth.  Zeros past the last row's tokens.  ``status`` [B]: 0, or
    what was wrong with the row (``check()``)."""

    bits: Tensor
    depth: Tensor
    positions: Tensor
    status: Tensor

    def check(self) -> "DraftTree":
        """Raise RuntimeError where a row's tokens are no tree or too many (a host synchronization)."""
        for b, word in enumerate(self.status.tolist()):
            if word:
                what = ", ".join(t for bit, t in _lib.DRAFT_STATUS.items() if word & bit)
                raise RuntimeError(f"draft_tree: row {b}: {what}")
        return self


def draft_tree(parents: Tensor, lens: Tensor, starts: Tensor, max_nodes: int) -> DraftTree:
    """Masks, depths and positions of each row's drafted tokens, in one launch.

    ``parents`` int32 [tokens]: the number in its row of the token that each token follows, below its
    own, or -1 for the first (several may follow none).  ``lens`` [B]: the rows' tokens, the
    drafted ones included; ``starts`` [B + 1]: the first of each row's tokens (both as
    ``page_slots`` gives them).  ``max_nodes``: the most tokens of a row, up to 1024; a row's
    tokens past ``32 * ceil(max_nodes / 32)`` see none and are seen by none, a parent that is no
    earlier token counts as -1, and ``status`` says so."""
    op = "draft_tree"
    _lib.require_gpu(parents, lens, starts, op=op)
    words = -(-int(max_nodes) // 32)
    if max_nodes < 1 or max_nodes > _lib.DRAFT_MAX_NODES:
        raise ValueError(f"{op}: max_nodes must be 1 to {_lib.DRAFT_MAX_NODES}, got {max_nodes}")
    T, B = parents.numel(), lens.numel()
    for name, t, size in (("parents", parents, T), ("lens", lens, B), ("starts", starts, B + 1)):
        if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != size or not t.is_contiguous():
            raise ValueError(f"{op}: {name} must be a contiguous int32 tensor of {size} elements, got {t.dtype} {list(t.shape)}")
    sizes = (T * words, T, T, B)
    buf = parents.new_empty(sum(sizes))  # (one allocation)
    bits, depth, positions, status = buf.split_with_sizes(sizes)
    at = buf.data_ptr()
    a = _lib.DraftTreeArgs(B, T, words, parents.data_ptr(), lens.data_ptr(), starts.data_ptr(), at, at + 4 * T * words,
                           at + 4 * T * (words + 1), at + 4 * T * (words + 2))
    _lib.launch("fade_draft_tree", a, parents.device)
    return DraftTree(bits.view(T, words), depth, positions, status)


@dataclass
class VerifiedDrafts:
    """What ``verify_drafts`` writes (on the GPU).

    ``path`` int32 [B, max_path]: the numbers in their row of the tokens that stay, from the first
    one on, -1 past them; ``counts`` int32 [B]: how many (``paged_compact``, ``TokenPagePool.accept``).
    ``tokens`` [B, max_path]: what the row goes on by, ``counts[b]`` tokens: the path's behind its
    first, then the new one; -1 past them.  ``next`` [B]: the new one, the first token of the
    row's next step.  A row without tokens: no path, and -1."""

    path: Tensor
    counts: Tensor
    tokens: Tensor
    next: Tensor


def verify_drafts(
    target: Tensor,
    tokens: Tensor,
    parents: Tensor,
    starts: Tensor,
    uniforms: Tensor,
    final: Tensor,
    max_path: int,
    draft: Tensor | None = None,
) -> VerifiedDrafts:
    """Which drafted tokens stay, and the token after them: distributed as the target's own tokens.

    Row b's tokens are ``starts[b]`` .. ``starts[b + 1] - 1`` of all, the first of them the row's
    last known token, the others drafted, each behind an earlier one (``parents``, as in ``draft_tree``).
    ``target`` [tokens, V] (fp32, fp16 or bf16, V contiguous): the target's probabilities of the token
    after each token.  From the first token on, the tokens that follow it are tried in the order of
    their numbers, and the walk goes on at the first that is accepted:

    - with ``draft`` (like ``target``: the probabilities that the tokens after each token were drawn
      from, one by one), a token x with uniform number u is accepted where
      ``u * draft[x] < target[x]``, else what is left of the target, ``max(target - draft, 0)`` over its sum,
      takes the target's place for the next one;
    - without (tokens chosen without chance: the likeliest ones, or found in the text so far), where
      ``u < target[x]``, else what is left is the target without x, over its sum.

    Where none is accepted, ``next`` is drawn from what is left: the first token at which the running
    sum passes ``final[b]`` of the sum.  ``uniforms`` [tokens] and ``final`` [B]: fp32 in [0, 1).
    ``tokens`` int64 or int32 [tokens]; one outside the vocabulary, e.g. the -1 that fills up a tree
    of a fixed number of tokens, is not tried, and what is left stays as it is.  ``max_path``: the most
    tokens that a path may have, up to 1024, the first included; behind so many no token is tried, nor any past
    a row's first 1024.  Sums are held in 64 bits.  Probabilities that are NaN or not above zero count as zero, infinite ones give an
    unspecified token; where the target has none above zero, ``next`` is -1."""
    op = "verify_drafts"
    _lib.require_gpu(target, tokens, parents, starts, uniforms, final, draft, op=op)
    _lib.no_gradient(op, target, draft, uniforms, final)
    if target.dim() != 2 or target.dtype not in _lib.DTYPE_CODES or target.shape[1] < 1:
        raise ValueError(f"{op}: target must be [tokens, V] of float32, float16 or bfloat16, got {target.dtype} {tuple(target.shape)}")
    if draft is not None and (draft.shape != target.shape or draft.dtype != target.dtype):
        raise ValueError(f"{op}: draft must be like target, {target.dtype} {tuple(target.shape)}, got {draft.dtype} {tuple(draft.shape)}")
    T, V = target.shape
    for name, t in (("target", target), ("draft", draft)):
        if t is not None and ((t.stride(1) != 1 and V > 1) or t.is_neg()):
            raise ValueError(f"{op}: {name} needs a contiguous vocabulary axis (make a copy)")
    B, M, i32 = final.numel(), int(max_path), torch.int32
    if tokens.dtype not in (torch.int64, i32):
        raise ValueError(f"{op}: tokens must be int64 or int32, got {tokens.dtype}")
    for name, t, size, dtype in (("tokens", tokens, T, tokens.dtype), ("parents", parents, T, i32), ("starts", starts, B + 1, i32),
                                 ("uniforms", uniforms, T, torch.float32), ("final", final, B, torch.float32)):
        if t.dtype is not dtype or t.dim() != 1 or t.shape[0] != size or not t.is_contiguous() or t.is_neg():
            raise ValueError(f"{op}: {name} must be a contiguous {dtype} [{size}], got {t.dtype} {list(t.shape)}")
    if not 1 <= M <= _lib.DRAFT_MAX_NODES:
        raise ValueError(f"{op}: max_path must be 1 to {_lib.DRAFT_MAX_NODES}, got {max_path}")
    r = VerifiedDrafts(starts.new_empty((B, M)), starts.new_empty(B), tokens.new_empty((B, M)), tokens.new_empty(B))
    a = _lib.VerifyArgs(B, T, V, M, target.data_ptr(), target.stride(0), _lib.ptr(draft), 0 if draft is None else draft.stride(0),
                        tokens.data_ptr(), parents.data_ptr(), starts.data_ptr(), uniforms.data_ptr(), final.data_ptr(),
                        r.path.data_ptr(), r.counts.data_ptr(), r.tokens.data_ptr(), r.next.data_ptr(), _lib.DTYPE_CODES[target.dtype],
                        int(tokens.dtype is torch.int64))
    _lib.launch_with_workspace("fade_verify_drafts", a, target.device)
    return r


__all__ = ["DraftTree", "VerifiedDrafts", "draft_tree", "verify_drafts"]
