"""Decoding along several branches, as measurable cases: the operators of a drafted tree and of a beam search.

Five kinds of pass, all on the slot pools of the batched decode step (ssm [S+1,16,128,128] float32, conv [(S+1)*2,3,6144] bf16, K / V
[S+1,2,Lmax,256] bf16):
  select   the best n continuations of a sequence's beams: log-softmax of every beam's logits over the vocabulary, the beam's score added,
           the n largest of beams x vocabulary
  reorder  the beams' states follow the selection: the slot of beam w takes over the state of its parent's slot, in place
  attn     attention of the M drafted tokens of each sequence over its cache and over their own ancestors in the tree; `layer`: with
           the q / k norm, rotary embedding and output gate of a full-attention layer around it
  gdn      the GatedDeltaNet step of those M tokens: every token continues from the state of its parent
  commit   the accepted path: the recurrent states advance along it, its K / V rows move up behind the cache

A tree is given by parents [B,M]: the index of a token's parent among the M, smaller than its own, or -1 for a child of the sequence's
last committed token.  The plain forms below are the definitions.  The layer core has bf16 rounding points of its own (conv, SiLU, norms,
gates, as in a decode step); they are part of the definition, and everything between them is taken in 32 bits, sums of squares and
transcendental functions in 64."""
from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HV, DK, DV, KD, CD, PW, QKV = 16, 128, 128, 2048, 6144, 8224, 5120
VOCAB = 248320                     # of the package's model configuration
MOST_LOGITS = 16 * 4 * VOCAB * 2   # bytes


def listed():
    return [
        # one user, the first level of a draft: eight children of the root
        {"name": "select_1x1", "kind": "select", "G": 1, "W": 1, "V": VOCAB, "n": 8, "dtype": "bf16"},
        # sixteen users with four beams each
        {"name": "select_16x4", "kind": "select", "G": 16, "W": 4, "V": VOCAB, "n": 4, "dtype": "bf16"},
        # one user's four beams, a short answer behind a prompt that all beams share
        {"name": "reorder_1x4", "kind": "reorder", "G": 1, "W": 4, "layers": 24, "Lmax": 512, "start": 250, "pos": 300},
        # eight users with four beams, long answers
        {"name": "reorder_8x4", "kind": "reorder", "G": 8, "W": 4, "layers": 24, "Lmax": 2048, "start": 700, "pos": 1900},
        # one user, a small tree on a short context: latency
        {"name": "attn_b1_m7", "kind": "attn", "layer": False, "B": 1, "M": 7, "lo": 300, "hi": 301},
        # an ordinary batch, the attention half of a layer
        {"name": "attn_layer_b16_m16", "kind": "attn", "layer": True, "B": 16, "M": 16, "lo": 1024, "hi": 8192},
        # wide trees on long contexts
        {"name": "attn_b8_m64_long", "kind": "attn", "layer": False, "B": 8, "M": 64, "lo": 8192, "hi": 32768},
        # the recurrent layers of the same three
        {"name": "gdn_b1_m7", "kind": "gdn", "B": 1, "M": 7},
        {"name": "gdn_b16_m16", "kind": "gdn", "B": 16, "M": 16},
        {"name": "gdn_b16_m64", "kind": "gdn", "B": 16, "M": 64},
        # what one user and a batch accept of their trees, all layers of the stack
        {"name": "commit_b1_m7", "kind": "commit", "B": 1, "M": 7, "D": 4, "layers": 24, "Lmax": 512},
        {"name": "commit_b16_m64", "kind": "commit", "B": 16, "M": 64, "D": 8, "layers": 24, "Lmax": 2048},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["select", "reorder", "attn", "attn", "gdn", "gdn", "commit"])
    if kind == "select":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        V = _log(rng, 1000, 262144)
        most = max(1, MOST_LOGITS // (V * (4 if dtype == "fp32" else 2)))
        W = _log(rng, 1, min(16, most))
        return {"kind": kind, "G": _log(rng, 1, max(1, min(32, most // W))), "W": W, "V": V, "n": rng.choice([1, 2, 3, 4, 5, 8, 10, 16, 32]), "dtype": dtype}
    if kind == "reorder":
        W = rng.choice([2, 3, 4, 5, 6, 8, 12, 16])
        pos = _log(rng, 20, 2000)
        return {"kind": kind, "G": _log(rng, 1, 32 // W), "W": W, "layers": rng.choice([8, 24]), "Lmax": pos + rng.randint(0, 100), "start": int(pos * rng.uniform(0, 0.95)),
                "pos": pos}
    if kind == "attn":
        M = _log(rng, 1, 64)
        B = _log(rng, 1, 32)
        hi = _log(rng, 64, min(32768, 8 * 20480 // B * min(4, 64 // M)))
        return {"kind": kind, "layer": rng.random() < 0.5, "B": B, "M": M, "lo": max(1, int(hi * rng.uniform(0.02, 0.7))), "hi": hi}
    if kind == "gdn":
        M = _log(rng, 1, 64)
        return {"kind": kind, "B": _log(rng, 1, min(64, 16 * 64 // M)), "M": M}
    M = _log(rng, 1, 64)
    return {"kind": kind, "B": _log(rng, 1, 16), "M": M, "D": rng.randint(1, min(M, 8)), "layers": rng.choice([8, 24]), "Lmax": 64 + _log(rng, 64, 1900)}


# ---- what a program has in hand ---------------------------------------------------------------------------------------

def _randn(gen, shape, scale=1.0, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=gen)


def _near_one(gen, n):
    return (1.0 + _randn(gen, (n,), 0.1, F32)).to(BF16)


def _on_gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _params(gen):
    return SimpleNamespace(cw=_randn(gen, (CD, 4, 1), 0.5), A_log=torch.empty(HV, device="cuda").uniform_(0.0, 2.7, generator=gen), dtb=_randn(gen, (HV,), 0.1, F32))


def _kinds(layers):
    """recurrent and full-attention layers of a stack (every fourth layer is one of the latter)"""
    return layers - layers // 4, layers // 4


def _trees(rng, B, M):
    """a drafted tree for each sequence: token 0 is the one that the last round ended with, every other token hangs on an earlier one, most of
    them near the root; one sequence in three drafts less than M, its last rows are padding"""
    p = np.full((B, M), -1, np.int32)
    for b in range(B):
        used = M if rng.random() < 0.67 else int(rng.integers(max(1, M // 2), M + 1))
        for j in range(1, used):
            p[b, j] = int(j * rng.random() ** 1.5)
    return p


def _paths(rng, parents, D):
    """from each tree the root path of one of its tokens, cut to D: the indices, and how many there are"""
    B, M = parents.shape
    path, count = np.zeros((B, D), np.int32), np.zeros(B, np.int32)
    for b in range(B):
        way, j = [], int(rng.integers(0, M))
        while j >= 0:
            way.append(j)
            j = parents[b, j]
        way = way[::-1][:D]
        path[b, :len(way)], count[b] = way, len(way)
    return path, count


def _positions(rng, B, lo, hi):
    return rng.permutation(np.linspace(lo, max(hi - 1, lo), B).round().astype(np.int32))


def prepare(case, seed):
    rng, gen = np.random.default_rng(seed), torch.Generator("cuda").manual_seed(seed)
    return {"select": _prepare_select, "reorder": _prepare_reorder, "attn": _prepare_attn, "gdn": _prepare_gdn, "commit": _prepare_commit}[case["kind"]](case, rng, gen)


def _prepare_select(case, rng, gen):
    G, W, V = case["G"], case["W"], case["V"]
    logits = _randn(gen, (G, W, V), 2.5, DTYPES[case["dtype"]])
    scores = torch.empty((G, W), device="cuda").uniform_(-12.0, -2.0, generator=gen)
    return SimpleNamespace(kind="select", logits=logits, scores=scores, n=case["n"])


def _pools(gen, layers, slots, Lmax):
    lin, att = _kinds(layers)
    return SimpleNamespace(conv=[_randn(gen, ((slots + 1) * 2, 3, CD)) for _ in range(lin)], ssm=[_randn(gen, (slots + 1, HV, DV, DK), 0.02, F32) for _ in range(lin)],
                           K=[_randn(gen, (slots + 1, 2, Lmax, 256)) for _ in range(att)], V=[_randn(gen, (slots + 1, 2, Lmax, 256)) for _ in range(att)])


def _prepare_reorder(case, rng, gen):
    G, W = case["G"], case["W"]
    return SimpleNamespace(kind="reorder", P=_pools(gen, case["layers"], G * W, case["Lmax"]), slots=_on_gpu(rng.permutation(G * W).reshape(G, W)),
                           parents=_on_gpu(rng.integers(0, W, (G, W))), start=_on_gpu(np.full(G, case["start"])), pos=_on_gpu(np.full(G, case["pos"])))


def _prepare_attn(case, rng, gen):
    B, M, Lmax = case["B"], case["M"], case["hi"] + case["M"]
    s = SimpleNamespace(kind="attn", layer=case["layer"], M=M, Kp=_randn(gen, (B + 1, 2, Lmax, 256)), Vp=_randn(gen, (B + 1, 2, Lmax, 256)), slots=_on_gpu(rng.permutation(B)),
                        pos=_on_gpu(_positions(rng, B, case["lo"], case["hi"])), parents=_on_gpu(_trees(rng, B, M)))
    if case["layer"]:
        s.qkv, s.q_norm, s.k_norm = _randn(gen, (B * M, QKV)), _near_one(gen, 256), _near_one(gen, 256)
    else:
        s.q, s.k, s.v = _randn(gen, (B * M, 8, 256)), _randn(gen, (B * M, 2, 256)), _randn(gen, (B * M, 2, 256))
    return s


def _prepare_gdn(case, rng, gen):
    B, M = case["B"], case["M"]
    return SimpleNamespace(kind="gdn", p=_params(gen), proj=_randn(gen, (B * M, PW)), conv=_randn(gen, ((B + 1) * 2, 3, CD)), ssm=_randn(gen, (B + 1, HV, DV, DK), 0.02, F32),
                           slots=_on_gpu(rng.permutation(B)), pos=_on_gpu(rng.integers(1, 30000, B)), parents=_on_gpu(_trees(rng, B, M)))


def _prepare_commit(case, rng, gen):
    B, M, layers, Lmax = case["B"], case["M"], case["layers"], case["Lmax"]
    lin = _kinds(layers)[0]
    path, count = _paths(rng, _trees(rng, B, M), case["D"])
    return SimpleNamespace(kind="commit", P=_pools(gen, layers, B, Lmax), projs=[_randn(gen, (B * M, PW)) for _ in range(lin)], p=[_params(gen) for _ in range(lin)],
                           slots=_on_gpu(rng.permutation(B)), pos=_on_gpu(rng.integers(1, Lmax - M + 1, B)), path=_on_gpu(path), count=_on_gpu(count))


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"select": _select, "reorder": _reorder, "attn": _attn, "gdn": _gdn, "commit": _commit}[s.kind](s)


def _run_own(s):
    import qwen_tailor_amd as qt
    if s.kind == "select":
        return qt.batch_beam.select(s.logits, s.scores, s.n)
    if s.kind == "reorder":
        qt.batch_beam.reorder(s.P, s.slots, s.parents, s.start, s.pos)
        return s.P.conv, s.P.ssm, s.P.K, s.P.V
    if s.kind == "attn":
        if s.layer:
            o = qt.batch_tree.attn_layer_bt(s.qkv, s.q_norm, s.k_norm, s.Kp, s.Vp, s.slots, s.pos, s.parents)
        else:
            o = qt.batch_tree.attn_bt(s.q, s.k, s.v, s.Kp, s.Vp, s.slots, s.pos, s.parents)
        return o, s.Kp, s.Vp
    if s.kind == "gdn":
        return qt.batch_tree.deltanet_bt(s.proj, s.conv, s.p.cw, s.p.A_log, s.p.dtb, s.ssm, s.slots, s.pos, s.parents)
    qt.batch_tree.commit(s.P, s.projs, [p.cw for p in s.p], [p.A_log for p in s.p], [p.dtb for p in s.p], s.slots, s.pos, s.path, s.count)
    return s.P.conv, s.P.ssm, s.P.K, s.P.V


# -- beams

def _select(s):
    G, W, V = s.logits.shape
    x = s.logits.to(F64)                                          # (candidates of two beams may lie closer than 32 bits tell apart)
    top = x.amax(-1, keepdim=True)
    x = s.scores.to(F64)[..., None] + (x - (top + (x - top).exp().sum(-1, keepdim=True).log()))
    best, at = x.reshape(G, W * V).sort(dim=-1, descending=True, stable=True)      # (stable: equal scores in the order of their indices)
    at = at[:, :s.n]
    return best[:, :s.n].to(F32), (at // V).to(I32), (at % V).to(I32)


def _reorder(s):
    slots = s.slots.long()
    src, dst = slots.gather(1, s.parents.long()).flatten(), slots.flatten()
    W = slots.shape[1]
    live = (s.pos.long() & 1).repeat_interleave(W)                # the conv buffer that a step at pos reads
    for pool in s.P.ssm:
        pool[dst] = pool[src]
    for pool in s.P.conv:
        pool[dst * 2 + live] = pool[src * 2 + live]
    for pool in s.P.K + s.P.V:
        at = torch.arange(pool.shape[2], device=pool.device)
        moved = ((at >= s.start[:, None]) & (at < s.pos[:, None])).repeat_interleave(W, 0)[:, None, :, None]
        pool[dst] = torch.where(moved, pool[src], pool[dst])
    return s.P.conv, s.P.ssm, s.P.K, s.P.V


# -- rounding points of the layer core

def _bf(x):
    return x.to(F32).to(BF16).to(F32)


def _sigmoid(x):                                                  # of bf16 values
    y = _bf(1.0 / _bf(1.0 + _bf(x.abs().to(F64).exp())))
    return torch.where(x < 0, y, _bf(1.0 - y))


def _softplus(x):
    e = _bf((-x.abs()).to(F64).exp())
    up = 1.0 + e
    log1p = torch.where(up == 1.0, e, e * (up.to(F64).log().to(F32) / (up - 1.0)))
    return _bf(x.clamp(min=0) + _bf(log1p))


def _norm128(u, scale):
    ss = u.to(F64).square().sum(-1, keepdim=True).to(F32)
    eps = np.float32(np.float32(1e-6) * np.float32(128 ** -0.5)) * np.float32(128 ** -0.5)
    r = ((ss / 128.0 + float(eps)).to(F64).sqrt().reciprocal()).to(F32)
    return _bf(_bf(u * r) * float(_bf(torch.tensor(scale))))


def _layer_core(rows, p, gates):
    """rows [..., 4, 6144]: a token's input row and the three before it (oldest first); gates [..., 32] = b | a.  -> q, k, v, g, beta"""
    w, x = p.cw.reshape(CD, 4).float(), rows.float()
    t = x[..., 0, :] * w[:, 0]
    for i in range(1, 4):
        t = t + x[..., i, :] * w[:, i]
    t = _bf(t)
    u = _bf(t * _sigmoid(t)).unflatten(-1, (3, HV, 128))
    b, a = gates.float().unflatten(-1, (2, HV)).unbind(-2)
    g = (-(p.A_log.to(F64).exp() * _softplus(_bf(a + p.dtb)))).exp().to(F32)
    inv = np.float32(128 ** -0.5)
    return _norm128(u[..., 0, :, :], inv * inv), _norm128(u[..., 1, :, :], inv), u[..., 2, :, :], g, _sigmoid(b)


def _delta(S, k, v, g, beta):
    """one token of the gated delta rule: the state that it leaves.  S [..., dv, dk]"""
    S = S * g[..., None, None]
    return S + ((v - (S * k[..., None, :]).sum(-1)) * beta[..., None])[..., None] * k[..., None, :]


# -- trees

def _gdn(s):
    B, M = s.parents.shape
    slots, parents = s.slots.long(), s.parents.long()
    window = s.conv[slots * 2 + (s.pos.long() & 1)]
    proj = s.proj.reshape(B, M, PW)
    rows = torch.cat([window, proj[..., :CD]], 1)                 # the window's rows 0 .. 2, then the tokens' own
    up = torch.cat([torch.tensor([0, 0, 1], device=parents.device).expand(B, 3), parents + 3], 1)     # the row before each row
    at = [torch.arange(3, M + 3, device=parents.device).expand(B, M)]
    for _ in range(3):
        at.insert(0, up.gather(1, at[0]))
    batch = torch.arange(B, device=parents.device)
    q, k, v, g, beta = _layer_core(rows[batch[:, None, None], torch.stack(at, -1)], s.p, proj[..., CD + KD:])
    states = torch.empty((B, M + 1, HV, DV, DK), device=proj.device)
    states[:, 0] = s.ssm[slots]
    for j in range(M):                                            # every token from its parent's state
        states[:, j + 1] = _delta(states[batch, parents[:, j] + 1], k[:, j], v[:, j], g[:, j], beta[:, j])
    y = torch.empty((B, M, HV, DV), device=proj.device)
    for j in range(M):
        y[:, j] = (states[:, j + 1] * q[:, j, :, None, :]).sum(-1)
    return y.reshape(B * M, KD).to(BF16)


def _commit(s):
    B, D = s.path.shape
    slots, pos, path, count = s.slots.long(), s.pos.long(), s.path.long(), s.count.long()
    batch = torch.arange(B, device=path.device)
    for conv, ssm, proj, p in zip(s.P.conv, s.P.ssm, s.projs, s.p):
        new = proj.reshape(B, -1, PW)[batch[:, None], path]
        rows = torch.cat([conv[slots * 2 + (pos & 1)], new[..., :CD]], 1)
        _, k, v, g, beta = _layer_core(rows.unfold(1, 4, 1).transpose(2, 3), p, new[..., CD + KD:])
        S = ssm[slots]
        for j in range(D):
            S = torch.where((j < count)[:, None, None, None], _delta(S, k[:, j], v[:, j], g[:, j], beta[:, j]), S)
        ssm[slots] = S
        conv[slots * 2 + ((pos + count) & 1)] = rows[batch[:, None], count[:, None] + torch.arange(3, device=path.device)]
    to = pos[:, None] + torch.arange(D, device=path.device)
    keep = (torch.arange(D, device=path.device) < count[:, None])[:, None, :, None]
    for pool in s.P.K + s.P.V:
        moved, there = pool[slots[:, None], :, pos[:, None] + path].transpose(1, 2), pool[slots[:, None], :, to].transpose(1, 2)
        pool[slots[:, None], :, to] = torch.where(keep, moved, there).transpose(1, 2)
    return s.P.conv, s.P.ssm, s.P.K, s.P.V


def _reach(parents):
    """[B,M,M]: token j is token i or one of its ancestors"""
    B, M = parents.shape
    eye = torch.eye(M, device=parents.device)
    r = eye + (parents[..., None] == torch.arange(M, device=parents.device)).float()
    for _ in range(6):
        r = ((r @ r) > 0).float()
    return r > 0


def _rope(x, pos):
    """rotary embedding of the first 64 of 256 features, half-split pairs, theta 1e7; x [..., heads, 256], pos [...]"""
    freq = (1e7 ** (-torch.arange(32, device=x.device, dtype=F64) / 32)).to(F32)
    th = (pos.float()[..., None] * freq).to(F64)[..., None, :]
    c, s = th.cos().to(F32), th.sin().to(F32)
    a, b = x[..., :32], x[..., 32:64]
    return torch.cat([_bf(a * c - b * s), _bf(a * s + b * c), x[..., 64:]], -1)


def _rms(x, w):
    inv = ((x.to(F64).square().sum(-1, keepdim=True).to(F32) / 256.0 + 1e-6).to(F64).sqrt().reciprocal()).to(F32)
    return _bf(w.float() * _bf(x * inv))


def _attn(s):
    B, M = s.parents.shape
    slots, pos = s.slots.long(), s.pos.long()
    reach = _reach(s.parents)
    if s.layer:
        heads = s.qkv[:, :4096].float().reshape(B, M, 8, 512)
        at = pos[:, None] + reach.sum(-1) - 1                     # a token's position: behind the cache by its depth
        q = _rope(_rms(heads[..., :256], s.q_norm), at)
        k = _rope(_rms(s.qkv[:, 4096:4608].float().reshape(B, M, 2, 256), s.k_norm), at)
        v = s.qkv[:, 4608:].float().reshape(B, M, 2, 256)
    else:
        q, k, v = s.q.float().reshape(B, M, 8, 256), s.k.float().reshape(B, M, 2, 256), s.v.float().reshape(B, M, 2, 256)
    to = pos[:, None] + torch.arange(M, device=pos.device)
    s.Kp[slots[:, None], :, to], s.Vp[slots[:, None], :, to] = k.to(BF16), v.to(BF16)
    L = s.Kp.shape[2]
    K, V = s.Kp[slots].float(), s.Vp[slots].float()
    key = torch.arange(L, device=pos.device)
    seen = torch.zeros((B, M, L), dtype=torch.bool, device=pos.device)
    seen[torch.arange(B, device=pos.device)[:, None, None], torch.arange(M, device=pos.device)[:, None], to[:, None]] = reach
    seen |= (key < pos[:, None])[:, None]
    rows = q.reshape(B, M, 2, 4, 256).transpose(1, 2).reshape(B, 2, M * 4, 256)
    x = (rows @ K.transpose(2, 3)).reshape(B, 2, M, 4, L) / 16.0
    x = torch.where(seen[:, None, :, None], x, float("-inf"))
    x = (x - x.amax(-1, keepdim=True)).exp()
    x = (x / x.sum(-1, keepdim=True)).reshape(B, 2, M * 4, L)
    o = (x @ V).reshape(B, 2, M, 4, 256).transpose(1, 2).reshape(B * M, 8, 256)
    if s.layer:
        o = (_bf(o) * _sigmoid(heads[..., 256:].reshape(B * M, 8, 256))).reshape(B * M, KD)
    return o.to(BF16), s.Kp, s.Vp


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "select":
        n = case["G"] * case["W"] * case["V"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + case["G"] * (4 * case["W"] + 12 * case["n"]), "flops": 4 * n}
    lin, att = _kinds(case.get("layers", 4))
    state = HV * DV * DK * 4
    if kind == "reorder":
        W = case["W"]
        written = W - 1                                           # expected over the parents that prepare() draws: beams that move, and the
        read = W * (1 - (1 - 1 / W) ** (W - 1))                   # different beams that they come from
        slot = lin * (state + 3 * CD * 2) + att * 2 * 2 * 512 * (case["pos"] - case["start"])
        return {"bytes": int(case["G"] * slot * (read + written)), "flops": 0}
    B, M = case["B"], case["M"]
    if kind == "attn":
        keys = B * (case["lo"] + max(case["hi"] - 1, case["lo"])) / 2
        row = (QKV + 2048 + 1024 if case["layer"] else 2048 * 2 + 1024 * 2) * 2        # a token's inputs, output and appended rows
        return {"bytes": int(keys * 2 * 2 * 512 + B * M * row), "flops": int(4 * 8 * 256 * M * (keys + B * M / 4))}
    if kind == "gdn":
        return {"bytes": B * (state + 3 * CD * 2 + M * ((CD + 32) * 2 + KD * 2)) + CD * 8, "flops": B * HV * M * (4 * DV * DK + 4 * DK * M // 2 + 4 * DV * M // 2)}
    n = _expected_path(M, case["D"])
    return {"bytes": int(B * (lin * (2 * state + 2 * 3 * CD * 2 + n * (2 * KD + 2 * KD + 64) * 2) + att * 2 * 2 * 2 * 512 * n)), "flops": int(B * lin * HV * n * 6 * DV * DK)}


def _expected_path(M, D):
    rng = np.random.default_rng(0)
    return float(np.mean([_paths(rng, _trees(rng, 8, M), D)[1].mean() for _ in range(8)]))


# ---- the same from the definitions in 64 bits ------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"select": _exact_select, "reorder": _exact_reorder, "attn": _exact_attn, "gdn": _exact_gdn, "commit": _exact_commit}[s.kind](s)


def _exact_select(s):
    p = torch.log_softmax(s.logits.double(), -1) + s.scores.double()[..., None]
    V = p.shape[-1]
    out, beam, tok = [], [], []
    for row in p:
        best, at = row.flatten().topk(s.n)
        out.append(best)
        beam.append(at // V)
        tok.append(at % V)
    return torch.stack(out), torch.stack(beam).int(), torch.stack(tok).int()


def _exact_reorder(s):
    slots, parents = s.slots.cpu().numpy(), s.parents.cpu().numpy()
    start, pos = s.start.cpu().numpy(), s.pos.cpu().numpy()

    def moved(pool, move):
        new = pool.double()
        for g in range(slots.shape[0]):
            for w in range(slots.shape[1]):
                move(new, pool, int(slots[g, w]), int(slots[g, parents[g, w]]), int(start[g]), int(pos[g]))
        return new

    def state(new, old, d, f, a, b):
        new[d] = old[f]

    def window(new, old, d, f, a, b):
        new[2 * d + b % 2] = old[2 * f + b % 2]

    def rows(new, old, d, f, a, b):
        new[d, :, a:b] = old[f, :, a:b]

    return [moved(p, window) for p in s.P.conv], [moved(p, state) for p in s.P.ssm], [moved(p, rows) for p in s.P.K], [moved(p, rows) for p in s.P.V]


def _np_bf(x):
    """to bf16 and back, to nearest even, on the bits"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return (((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)


def _np_sigmoid(x):
    e = _np_bf(np.exp(np.abs(x).astype(np.float64)).astype(np.float32))
    y = _np_bf(np.float32(1) / _np_bf(np.float32(1) + e))
    return np.where(x < 0, y, _np_bf(np.float32(1) - y))


def _np_core(x, p, b, a):
    """x [4, 6144]: a token's input rows, oldest first; b, a [16] -> q, k, v [16, 128], g, beta [16] in 64 bits"""
    f = np.float32
    w = p.cw.float().cpu().numpy().reshape(CD, 4)
    t = x[0] * w[:, 0]
    for i in (1, 2, 3):
        t = (t + x[i] * w[:, i]).astype(f)
    t = _np_bf(t)
    u = _np_bf(t * _np_sigmoid(t)).reshape(3, HV, 128)
    inv = f(128 ** -0.5)
    eps = f(f(f(1e-6) * inv) * inv)

    def unit(r, scale):
        ss = (r.astype(np.float64) ** 2).sum(-1, keepdims=True).astype(f)
        return _np_bf(_np_bf(r * (1 / np.sqrt((ss / f(128) + eps).astype(np.float64))).astype(f)) * _np_bf(scale))

    z = _np_bf(a + p.dtb.cpu().numpy())
    e = _np_bf(np.exp(-np.abs(z).astype(np.float64)).astype(f))
    up = f(1) + e
    ratio = np.log(up.astype(np.float64)).astype(f) / np.where(up == 1, f(1), up - f(1))
    sp = _np_bf(np.maximum(z, f(0)) + _np_bf(np.where(up == 1, e, e * ratio)))
    g = np.exp(-np.exp(p.A_log.cpu().numpy().astype(np.float64)) * sp)
    d = lambda v: torch.from_numpy(np.ascontiguousarray(v, np.float64)).cuda()  # noqa: E731
    return d(unit(u[0], inv * inv)), d(unit(u[1], inv)), d(u[2]), d(g), d(_np_sigmoid(b))


def _step64(S, k, v, g, beta):
    S = g[:, None, None] * S
    delta = beta[:, None] * (v - torch.einsum("hvk,hk->hv", S, k))
    return S + torch.einsum("hv,hk->hvk", delta, k)


def _exact_gdn(s):
    B, M = s.parents.shape
    proj, parents = s.proj.float().cpu().numpy().reshape(B, M, PW), s.parents.cpu().numpy()
    out = []
    for b in range(B):
        slot = int(s.slots[b])
        window = list(s.conv[2 * slot + int(s.pos[b]) % 2].float().cpu().numpy())
        S0 = s.ssm[slot].double()
        states, chains = [], []
        for j in range(M):
            i = int(parents[b, j])
            S, chain = (S0, window) if i < 0 else (states[i], chains[i])
            chain = chain[-3:] + [proj[b, j, :CD]]
            q, k, v, g, beta = _np_core(chain, s.p, proj[b, j, CD + KD:CD + KD + HV], proj[b, j, CD + KD + HV:])
            states.append(_step64(S, k, v, g, beta))
            chains.append(chain)
            out.append(torch.einsum("hvk,hk->hv", states[-1], q).flatten())
    return torch.stack(out)


def _exact_commit(s):
    B, D = s.path.shape
    path, count, slots, pos = (t.cpu().numpy() for t in (s.path, s.count, s.slots, s.pos))
    convs, ssms, Ks, Vs = [], [], [p.double() for p in s.P.K], [p.double() for p in s.P.V]
    for conv, ssm, proj, p in zip(s.P.conv, s.P.ssm, s.projs, s.p):
        new_conv, new_ssm = conv.double(), ssm.double()
        for b in range(B):
            slot, n = int(slots[b]), int(count[b])
            chain = list(conv[2 * slot + int(pos[b]) % 2].float().cpu().numpy())
            rows = proj.reshape(B, -1, PW)[b, s.path[b, :n].long()].float().cpu().numpy()
            for r in rows:
                chain.append(r[:CD])
                _, k, v, g, beta = _np_core(chain[-4:], p, r[CD + KD:CD + KD + HV], r[CD + KD + HV:])
                new_ssm[slot] = _step64(new_ssm[slot], k, v, g, beta)
            new_conv[2 * slot + (int(pos[b]) + n) % 2] = torch.from_numpy(np.stack(chain[-3:])).cuda().double()
        convs.append(new_conv)
        ssms.append(new_ssm)
    for new, old in list(zip(Ks, s.P.K)) + list(zip(Vs, s.P.V)):
        for b in range(B):
            for j in range(int(count[b])):
                new[int(slots[b]), :, int(pos[b]) + j] = old[int(slots[b]), :, int(pos[b]) + int(path[b, j])].double()
    return convs, ssms, Ks, Vs


def _exact_attn(s):
    B, M = s.parents.shape
    parents, slots, pos = (t.cpu().numpy() for t in (s.parents, s.slots, s.pos))
    Ks, Vs, out = s.Kp.double(), s.Vp.double(), []
    for b in range(B):
        at, n = int(slots[b]), int(pos[b])
        mine = []
        for j in range(M):
            mine.append((mine[parents[b, j]] if parents[b, j] >= 0 else []) + [j])
        seen = torch.zeros((M, M), dtype=torch.bool, device="cuda")
        for j in range(M):
            seen[j, torch.tensor(mine[j], device="cuda")] = True
        if s.layer:
            x = s.qkv[b * M:(b + 1) * M].double()
            heads = x[:, :4096].reshape(M, 8, 2, 256)
            where = torch.tensor([n + len(m) - 1 for m in mine], device="cuda").double()
            unit = lambda r, w: w.double() * r / (r.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731

            def turn(r):
                th = where[:, None, None] * (1e7 ** (-2.0 * torch.arange(32, device="cuda").double() / 64)).float().double()
                z = torch.complex(r[..., :32], r[..., 32:64]) * torch.polar(torch.ones_like(th), th)
                return torch.cat([z.real, z.imag, r[..., 64:]], -1)

            q, k, v, gate = turn(unit(heads[:, :, 0], s.q_norm)), turn(unit(x[:, 4096:4608].reshape(M, 2, 256), s.k_norm)), x[:, 4608:].reshape(M, 2, 256), heads[:, :, 1]
        else:
            q, k, v = (t[b * M:(b + 1) * M].double() for t in (s.q, s.k, s.v))
        Ks[at, :, n:n + M], Vs[at, :, n:n + M] = k.transpose(0, 1), v.transpose(0, 1)
        see = torch.cat([torch.ones((M, n), dtype=torch.bool, device="cuda"), seen], 1)
        o = torch.empty((M, 8, 256), dtype=F64, device="cuda")
        for h in range(8):
            x = (q[:, h] @ Ks[at, h // 4, :n + M].T / 16).masked_fill(~see, float("-inf"))
            o[:, h] = torch.softmax(x, -1) @ Vs[at, h // 4, :n + M]
        out.append((o * torch.sigmoid(gate)).reshape(M, KD) if s.layer else o)
    return torch.cat(out), Ks, Vs
