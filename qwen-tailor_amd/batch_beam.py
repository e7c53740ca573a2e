"""Beam search on the slot pools of the batched decode step: the selection over beams and vocabulary, and the reordering of the beams' states.

A sequence g has W beams, each a slot of the pools (slots int32 [G, W]).  A step decodes all G*W rows (batch.deltanet_b, attn_layer_b, ..); select picks
the continuations from the logits, reorder lets the states follow.  A drafted tree (batch_tree) is grown the same way, a level at a time.

Both run on the device of their tensors, on that device's current stream."""
from __future__ import annotations

from . import _lib as L


def select(logits, scores, n):
    """The n best continuations of each sequence's beams.  logits [G, W, V] bf16, fp16 or float32 (the vocabulary contiguous, any strides of the other
    two), scores float32 [G, W]: the beams' log-probabilities, -inf for a beam that is none.  Candidate (w, t) scores scores[w] + log_softmax(logits[w])[t].
    Returns scores float32, parents int32 (w) and tokens int32 (t), each [G, n], in falling order, equal scores by the lower w V + t (the log-sum of a
    beam is known to 1e-6: candidates of two beams that lie closer may change places).  A
    candidate whose score is -inf (as float32) or NaN is none; places left over get -inf, -1, -1.  W and n up to 64, G W up to 65535."""
    return L.host.beam_select(logits, scores, n)


def reorder(P, slots, parents, start, pos):
    """The state of beam w of sequence g becomes that of its beam parents[g, w], for all beams at once and in place, in every layer of the pools P
    (batch.Pools, or any object with its lists conv, ssm, K and V): the recurrent state, the conv buffer pos[g] & 1 (the one that a step at pos
    reads) and the K / V rows start[g] .. pos[g] - 1.  slots, parents int32 [G, W], start, pos int32 [G]; rows before start are common to a
    sequence's beams and stay.  A beam whose parent is itself or none (-1) stays as it is.  The slots are different from each other, but for those of
    beams that stay.  W up to 32."""
    L.host.beam_reorder(P.conv, P.ssm, P.K, P.V, slots, parents, start, pos)
