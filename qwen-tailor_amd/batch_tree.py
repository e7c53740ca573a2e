"""Verification of a tree of drafted tokens for each of B sequences, on the pools of the batched decode step (batch.Pools).

batch_spec verifies chains: M tokens a sequence, a state snapshot after each.  Here a sequence's M <= 64 tokens form a tree, given by parents int32 [B, M]
on the device: the index of a token's parent among the M, smaller than its own, or -1 for a child of the last committed token (anything else counts
as -1).  A sequence that drafts fewer tokens pads its rows with -1: no other token sees them.  Row b*M + j is token j of sequence b.  The slots of a call
are different from each other, but for those of sequences that pad the batch: they may all point at the trash slot, and their outputs mean nothing.

A round: the layers run deltanet_bt / attn_layer_bt on the tree, which leave the recurrent state and the conv window as they are and the K / V
rows of the tree behind the cache; the program picks a path (path int32 [B, D], count int32 [B]); commit takes it into the pools of all layers.

Every operator runs on the device of its tensors, on that device's current stream."""
from __future__ import annotations

from . import _lib as L


def deltanet_bt(proj, conv_pool, conv_w, A_log, dt_bias, ssm_pool, slots, pos, parents):
    """The GatedDeltaNet step of the tokens of B trees: every token continues from the state and conv window of its parent.  proj [B*M, 8224] bf16; pools,
    slots and pos int32 [B] as for batch.deltanet_b.  Returns y [B*M, 2048] bf16; nothing is written to the pools (a chain gives the outputs of
    batch_spec.deltanet_bm up to the order of sums).  The rows of a sequence whose slot is out of range are zero.  A token whose conv outputs or gates
    are not finite (or |v| >= 2^100) makes its own row and its descendants' NaN and no other."""
    return L.host.deltanet_bt(proj, conv_pool, conv_w, A_log, dt_bias, ssm_pool, slots, pos, parents)


def attn_bt(q, k, v, Kp, Vp, slots, pos, parents):
    """Attention of the tokens of B trees: token j sees the pool keys below pos[b], the new keys of its ancestors and its own.  q [B*M, 8, 256], k / v
    [B*M, 2, 256] bf16 (normed and roped), pools [S+1, 2, Lmax, 256].  Returns o [B*M, 8, 256] bf16 and appends new row j at pos[b] + j (in place);
    a sequence whose slot or rows do not fit is skipped: its outputs are zero.  B up to 1024."""
    return L.host.attn_bt(q, k, v, Kp, Vp, slots, pos, parents)


def attn_layer_bt(qkv, q_norm, k_norm, Kp, Vp, slots, pos, parents, eps=1e-6):
    """The attention half of a full-attention layer for the tokens of B trees (batch.attn_layer_b for chains): q / k RMSNorm, rotary embedding at position
    pos[b] + the token's depth, attn_bt, and o * sigmoid(gate).  qkv [B*M, 5120] bf16.  Returns [B*M, 2048] bf16."""
    return L.host.attn_layer_bt(qkv, q_norm, k_norm, Kp, Vp, slots, pos, parents, eps)


def commit(P, projs, conv_ws, A_logs, dt_biases, slots, pos, path, count, M=None):
    """The accepted path of each tree becomes part of its sequence, in every layer of the pools P (batch.Pools, or any object with its lists conv, ssm, K and
    V).  projs: the projection rows [B*M, 8224] that deltanet_bt was given, one tensor for each recurrent layer; conv_ws, A_logs, dt_biases the
    layers' parameters.  path int32 [B, D]: indices among the M tokens from the root down, count int32 [B] how many (0: the sequence stays as it is; more than D
    or M count as the smaller of the two).
    In place: states advance with the bits of as many batch.deltanet_b steps, the conv window goes to buffer (pos + count) & 1, K / V rows pos + path[j]
    move to pos + j.  The caller then counts pos + count tokens.  M: tokens a tree, needed only where there is no recurrent layer."""
    L.host.tree_commit(P.conv, P.ssm, P.K, P.V, projs, conv_ws, A_logs, dt_biases, slots, pos, path, count, M)
