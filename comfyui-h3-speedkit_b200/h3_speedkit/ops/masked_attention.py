"""BF16 / FP16 attention under masks (B200).

Stands beside ``ops.dense`` (the unmasked INT8 attention of one geometry): documents
packed into one sequence, padded batches, causal and prefix masks, scores capped by a
tanh, a bias by distance, grouped heads, any lengths from zero, through
``h3_masked_attention_run`` of libh3sk_b200.so (tcgen05):

    score = scale * q . k
    score = softcap * tanh(score / softcap)            with softcap > 0
    score = score - slopes[head] * |pos - j|           with slopes
    out = softmax(score) v,   lse = ln sum exp(score)  over the visible keys j

``pos`` is the query's place among its sequence's keys: its number plus the keys less
the queries of the sequence (the last query stands at the last key).  Statistics in
FP32, probabilities rounded to the inputs' type for the second product, the result
rounded once.  ``MaskedAttentionProvider`` puts it, with the rotary positions, behind
``Backend.block(attention=...)`` and ``patch_model(attention=...)``.  Inference only.
"""
from __future__ import annotations

import torch

from .. import _lib
from .rope import rope_axes


def masked_attention(q, k, v, *, scale=None, softcap=0.0, slopes=None, causal=False, prefix=None, q_offsets=None,
                     k_offsets=None, q_lengths=None, k_lengths=None, out=None, lse=None, return_lse=False):
    """Attention of q [B, Sq, Hq, D] over k and v [B, Sk, Hk, D]; 3-D operands
    [S, H, D] are one sequence.  D is 64 or 128, Hq a multiple of Hk, lengths from 0.

    Documents (one sequence only): q_offsets, k_offsets INT32 [N + 1], ascending;
    document n's queries see its keys.  Padded batch: q_lengths, k_lengths INT32 [B],
    the valid tokens of each sequence.  causal: keys up to the query's place, and,
    with prefix (INT32 [N] or [B]), all below the sequence's prefix.

    A row that sees no key gives zeros and an lse of -inf.  Rows that belong to no
    sequence stay as they were in a given ``out`` and ``lse``, and are zero in new
    ones.  Masked values, NaN and infinities among them, reach no result.  Strides are
    multiples of 8 values, operands 16-byte aligned; expanded heads of k and v and
    expanded batches are taken as they are.  The sum of weights times v is FP32 and is
    divided at the end: |v| times a row's keys, times 2^8, has to stay below 3.4e38.

    Returns out (q's shape and type), or (out, lse) with ``return_lse`` or a given
    ``lse``: FP32 [B, Hq, Sq] ([Hq, Sq] for 3-D operands)."""
    return _lib.binding().masked_attention(q, k, v, scale, softcap, slopes, causal, prefix, q_offsets, k_offsets, q_lengths,
                                           k_lengths, out, lse, return_lse)


class MaskedAttentionProvider:
    """The ``attention`` of ``Backend.block`` / ``patch_model`` in BF16: the slices of a
    plain QKV projection, Q and K normalised per head and turned to their positions,
    then ``masked_attention``.

    heads: query (and key) heads of the projection's slices.  positions [M, A] and
    sections as ``rope_axes`` takes them (None: no rotation).  masks: any of
    ``masked_attention``'s keyword arguments (scale, softcap, slopes, causal, prefix,
    q_offsets, k_offsets, q_lengths, k_lengths).  The per-head norm weights are the
    block's ``attn.q_norm`` / ``attn.k_norm``; called directly, without a block, Q and
    K are not normalised."""

    MASKS = ('scale', 'softcap', 'slopes', 'causal', 'prefix', 'q_offsets', 'k_offsets', 'q_lengths', 'k_lengths')

    def __init__(self, heads, *, positions=None, sections=None, theta=10000.0, interleaved=False, **masks):
        if (positions is None) != (sections is None):
            raise ValueError('positions and sections are given together')
        if not set(masks) <= set(self.MASKS):
            raise ValueError(f'masks are any of {", ".join(self.MASKS)}')
        self.heads, self.positions, self.masks = heads, positions, masks
        self.rope = dict(sections=sections, theta=theta, interleaved=interleaved)

    def for_block(self, block):
        """The callable of one block, with its norm weights (none where it has none)."""
        attn = block.attn
        if not hasattr(attn, 'q_norm'):
            return self
        return lambda q, k, v: self(q, k, v, attn.q_norm.weight, attn.k_norm.weight, float(attn.q_norm.eps))

    def __call__(self, q, k, v, q_weight=None, k_weight=None, eps=1e-6):
        m, width = q.shape
        if width % self.heads:
            raise ValueError('The projection does not divide into the heads')
        q, k, v = (t.view(m, self.heads, width // self.heads) for t in (q, k, v))
        if self.positions is not None:
            # both as they are stored, in FP32 if either is (or is of another type)
            own = all(t is None or t.dtype == q.dtype for t in (q_weight, k_weight))
            w = [None if t is None else t.detach().to(device=q.device, dtype=q.dtype if own else torch.float32).contiguous()
                 for t in (q_weight, k_weight)]
            q, k = rope_axes(q, k, self.positions, q_weight=w[0], k_weight=w[1], eps=eps, **self.rope)
        elif q_weight is not None:
            raise ValueError('A block with per-head norms needs positions')
        return masked_attention(q, k, v, **self.masks).view(m, width)
