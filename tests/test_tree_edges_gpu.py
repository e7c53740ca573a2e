"""Drafted trees (batch_tree) where they can go wrong without the random cases of test_tree_gpu.py showing it: outputs in which opposite values cancel, states of which little
is left, paths that claim more tokens than there are, workgroups that go from one sequence to the next, masks under long caches, padding in a common slot, the largest batch."""
import numpy as np
import pytest
import torch

from oracle import gdn_oracle as O
from tests.test_tree_gpu import PoolSet, attn_run, gdn_case, gdn_reference, gdn_run, params, trees, way
from tests.util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


def attention64(c, parents=None):
    """float64 on the CPU, all sequences taking part -> o [R, 8, 256], sum of w |V| likewise, largest sum of |q k| of a key"""
    parents = c["parents"] if parents is None else parents
    B, M = parents.shape
    q, k, v = (c[n].cpu().double() for n in ("q", "k", "v"))
    o, a, most = torch.zeros((B * M, 8, 256), dtype=torch.float64), torch.zeros((B * M, 8, 256), dtype=torch.float64), 0.0
    for b in range(B):
        s, n, rows = int(c["slots"][b]), int(c["pos"][b]), slice(b * M, (b + 1) * M)
        see = torch.zeros((M, n + M), dtype=torch.bool)
        see[:, :n] = True
        for j in range(M):
            see[j, [n + i for i in way(parents[b], j)]] = True
        for h in range(2):
            K, V = (torch.cat([c[p][s, h, :n].cpu().double(), new[rows, h]]) for p, new in (("Kp", k), ("Vp", v)))
            x = q[rows, 4 * h:4 * h + 4].reshape(4 * M, 256)
            most = max(most, float((x.abs() @ K.abs().T).max()))
            w = torch.softmax((x @ K.T / 16).masked_fill(~see.repeat_interleave(4, 0), float("-inf")), -1)
            o[rows, 4 * h:4 * h + 4], a[rows, 4 * h:4 * h + 4] = (w @ V).reshape(M, 4, 256), (w @ V.abs()).reshape(M, 4, 256)
    return o, a, most


def attention_bound(c, ref, a, most):
    """|o - ref|: the output's rounding (bf16: 2^-8 of it); P as two bf16 terms (2^-16 of a weight); a score's sum of 256 products in float (2^-24 of the sum of their magnitudes each,
    1/16 of it in the exponent), its power of two (an argument of up to 2^-24 |x - max| log2 e, a result to 2^-23) and the sums over keys in float, which all change weights, in
    the numerator and in the sum below it"""
    keys = int(max(c["pos"])) + c["parents"].shape[1]
    weight = 256 * 2 ** -24 * most / 16 + 2 ** -24 * 2 * most / 16 * 1.4427 + 2 ** -23 + keys * 2 ** -24
    return 2 ** -8 * ref.abs() + (2 ** -16 + 2 * weight) * a


@pytest.mark.parametrize("M", [4, 12, 24, 33, 48, 64])
@pytest.mark.parametrize("pos", [0, 2, 40])
def test_attention_of_values_that_cancel(dev, M, pos):
    """nearly equal scores on opposite rows of V: what is left of the sum is small beside its terms, and so must be the error, at any number of tokens"""
    g = torch.Generator(dev).manual_seed(M + pos)
    r = lambda *s: torch.empty(s, device=dev).normal_(generator=g)  # noqa: E731
    Lmax = pos + M
    x, key = r(2, 256).to(BF16), r(2, 256)
    sign = lambda n: (1 - 2 * (torch.arange(n, device=dev) % 2)).to(BF16)  # noqa: E731
    c = {"q": (0.25 * r(M, 8, 256)).to(BF16), "k": (key + 0.05 * r(M, 2, 256)).to(BF16), "v": x * sign(M)[:, None, None],
         "Kp": (key[:, None] + 0.05 * r(3, 2, Lmax, 256)).to(BF16), "Vp": (x[:, None] * sign(Lmax)[:, None]).expand(3, 2, Lmax, 256).contiguous(),
         "slots": np.array([1], np.int32), "pos": np.array([pos], np.int32), "parents": trees(np.random.default_rng(M), 1, M, "star")}
    o, _, _ = attn_run(c, dev)
    ref, a, most = attention64(c)
    over = (o.cpu().double() - ref).abs() / attention_bound(c, ref, a, most)
    assert float(over.max()) <= 1.0, f"{float(over.max()):.2f} of the bound"


@pytest.mark.parametrize("M,D", [(6, 20), (1, 64), (9, 10), (20, 6)])
def test_commit_of_counts_beyond_the_tree(dev, M, D):
    """count > M, count > D, at the end of the pool: what count = min(D, M) does; the rows, heads and slots behind stay as they are"""
    import qwen_tailor_amd as qt
    gen = torch.Generator(dev).manual_seed(M)
    B, Lmax, most = 3, 2 * M + 5, min(D, M)
    P = PoolSet(gen, 1, 2, B, Lmax, dev)
    proj, p = torch.empty((B * M, PW), dtype=BF16, device=dev).normal_(generator=gen), params(gen, dev)
    i = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    path, slots, pos = i(np.random.default_rng(M).integers(0, M, (B, D))), i([2, 0, 1]), i([Lmax - M, Lmax - M, 1])
    got, want = P.clone(), P.clone()
    for pools, count in ((want, [most] * B), (got, [most + 1, 2 ** 31 - 1, max(M, D)])):
        qt.batch_tree.commit(pools, [proj], [p[0]], [p[1]], [p[2]], slots, pos, path, i(count))
    for name in ("conv", "ssm", "K", "V"):
        for a, b in zip(getattr(got, name), getattr(want, name)):
            check_tensors_equal(name, a, b)
    for name in ("K", "V"):
        for a, old in zip(getattr(got, name), getattr(P, name)):
            for s, n in zip(slots.tolist(), pos.tolist()):
                check_tensors_equal(f"{name}: rows before", a[s, :, :n], old[s, :, :n])
                check_tensors_equal(f"{name}: rows behind", a[s, :, n + most:], old[s, :, n + most:])
                check_tensors_equal(f"{name}: rows moved", a[s, :, n:n + most], old[s][:, (n + path[slots.tolist().index(s), :most]).long()])


@pytest.mark.parametrize("M", [1, 16, 17, 33, 64])
def test_gdn_step_of_states_that_cancel(dev, M):
    """rows of the state with two elements whose products with q are opposite, and that two bf16 terms would be 2^-17 off in the same direction: what is left has the precision
    of a float state.  (Equal tokens, so q is the same for all; beta = 0, so the outputs are gamma S q.)"""
    c = gdn_case(500 + M, 1, M, "chain")
    c["proj"][:] = c["proj"][:1]
    slot, pos = int(c["slots"][0]), int(c["pos"][0])
    c["conv"][2 * slot + (pos & 1)] = c["proj"][0, :CD]
    c["proj"][:, 8192:8208], c["proj"][:, 8208:8224] = -60.0, -8.0
    u = O.conv_silu(c["conv"][2 * slot + (pos & 1)], c["proj"][0, :CD], c["cw"])
    q, _ = O.normalize_qk(u[:2048].reshape(16, 128), u[2048:4096].reshape(16, 128))
    q = np.asarray(q, np.float64)
    two = lambda x: bf(x) + bf(x - bf(x))  # noqa: E731  (exact in float32: the terms do not overlap)
    rng = np.random.default_rng(M)
    S = np.zeros((16, 128, 128), np.float32)
    for h in range(16):
        big = np.argsort(-np.abs(q[h]))[:16]
        for v in range(128):
            i, j = rng.choice(big, 2, replace=False)
            a = (1.0 + rng.random(4000) * 2 ** -4).astype(np.float32)
            a = a[np.argmax((a - two(a)) * np.sign(q[h, i]))]                            # q_i times what two terms leave: positive
            b = (-q[h, i] * a / q[h, j] * (1 + (rng.random(4000) - 0.5) * 2 ** -13)).astype(np.float32)
            S[h, v, i], S[h, v, j] = a, b[np.argmax((b - two(b)) * np.sign(q[h, j]))]
    c["ssm"][slot] = S
    y, ref = to_np(gdn_run(c, dev)).astype(np.float64), gdn_reference(c)
    # the rounding of the output; six products and their sum in float, and gamma in float of a sum of at most 64 logarithms
    terms = np.einsum("hvk,hk->hv", np.abs(S.astype(np.float64)), np.abs(q)).ravel()
    over = np.abs(y - ref) / ((2 ** -8 + 2 ** -20) * np.abs(ref) + 12 * 2 ** -24 * terms)
    assert over.max() <= 1.0, f"{over.max():.2f} of the bound"


# ---- workgroups with several segments -------------------------------------------------------------------------------------

def visits(dev, B, M, pos):
    """the most segments (sequence, KV head) that one workgroup of the attention launch takes part in, from the launch's own plan, and how many segments there are"""
    rows = 32 if M <= 8 else 64 if M <= 16 else 128 if M <= 32 else 256
    extra, nwg = 2 + rows // 64, torch.cuda.get_device_properties(dev).multi_processor_count
    size = np.repeat([(n + 31) // 32 + (M + 31) // 32 + extra if n >= 0 else 0 for n in pos], 2)
    end = np.cumsum(size)
    per = max(2, -(-int(end[-1]) // nwg))
    most = 0
    for w in range(nwg):
        a, b = w * per, min((w + 1) * per, int(end[-1]))
        most = max(most, int(((end - size + extra < b) & (end > a) & (size > 0)).sum()))
    return most, 2 * B


def short_caches(B):
    return [(7 * k) % 40 for k in range(B)]


def one_long(B, n):
    return [n if k == B // 3 else (5 * k) % 33 for k in range(B)]


VISITS = [(200, 5, short_caches(200)), (200, 12, short_caches(200)), (300, 16, short_caches(300)), (32, 13, one_long(32, 40000)), (180, 24, short_caches(180)), (32, 20, one_long(32, 50000)),
          (150, 64, short_caches(150)), (300, 40, short_caches(300)), (32, 50, one_long(32, 60000))]


def visit_case(dev, B, M, pos):
    rng, g = np.random.default_rng(B + M), torch.Generator(dev).manual_seed(B + M)
    r = lambda *s: torch.empty(s, dtype=BF16, device=dev).normal_(generator=g)  # noqa: E731
    S, Lmax = B, max(pos) + M
    pos = np.array(pos, np.int32)
    slots = rng.permutation(S)[:B].astype(np.int32)
    pos[4], slots[6] = -1, S + 9                                 # two that are skipped
    most, segments = visits(dev, B, M, [int(p) if s < S else -1 for p, s in zip(pos, slots)])
    assert most >= 2, (most, segments)
    return {"qkv": r(B * M, 5120), "q_norm": r(256), "k_norm": r(256), "Kp": r(S, 2, Lmax, 256), "Vp": r(S, 2, Lmax, 256), "slots": slots, "pos": pos, "parents": trees(rng, B, M, "random")}


@pytest.mark.parametrize("B,M,pos", VISITS)
def test_attention_from_one_sequence_to_the_next(dev, B, M, pos):
    """workgroups with several visits, at every number of row tiles, with at most 64 segments and with more: against 64 bits, and the layer against attn_bt"""
    import qwen_tailor_amd as qt
    c = visit_case(dev, B, M, pos)
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    skipped = [4, 6]
    at = np.array([max(int(c["pos"][b]), 0) + len(way(c["parents"][b], j)) - 1 for b in range(B) for j in range(M)])
    c["q"], c["k"], c["v"] = qt.attention.qkv_prep(c["qkv"], c["q_norm"], c["k_norm"], i(at))
    c["v"].reshape(B, M, -1)[skipped] = float("nan")
    o, K, V = attn_run(c, dev)
    K2, V2 = c["Kp"].clone(), c["Vp"].clone()
    got = qt.batch_tree.attn_layer_bt(c["qkv"], c["q_norm"], c["k_norm"], K2, V2, i(c["slots"]), i(c["pos"]), i(c["parents"]))
    want = qt.attention.out_gate(o, c["qkv"]).reshape(B, M, -1)
    want[skipped] = 0
    check_tensors_equal("layer", got.reshape(B, M, -1), want)
    check_tensors_equal("layer: K", K2, K)
    check_tensors_equal("layer: V", V2, V)
    assert not bool(o.reshape(B, -1)[skipped].any())
    keep = [b for b in range(B) if b not in skipped]
    rows = [b * M + j for b in keep for j in range(M)]
    for name, pool, new in (("K", K, c["k"]), ("V", V, c["v"])):
        old = c[name + "p"].clone()
        for b in keep:
            old[c["slots"][b], :, c["pos"][b]:c["pos"][b] + M] = new[b * M:(b + 1) * M].transpose(0, 1)
        check_tensors_equal(name, pool, old)
    d = {"q": c["q"][rows], "k": c["k"][rows], "v": c["v"][rows], "Kp": c["Kp"], "Vp": c["Vp"], "slots": c["slots"][keep], "pos": c["pos"][keep], "parents": c["parents"][keep]}
    ref, a, most = attention64(d)
    over = (o[rows].cpu().double() - ref).abs() / attention_bound(d, ref, a, most)
    assert float(over.max()) <= 1.0, f"{float(over.max()):.2f} of the bound"


@pytest.mark.parametrize("M", [6, 16, 30, 64])
def test_masks_under_a_long_cache(dev, M):
    """the new keys carry most of the weight of a row, so that one that is wrongly seen or left out shows, however long the cache is.  (The bound notices: a mistake in the
    oracle's tree is beyond it in the rows that it concerns.)"""
    g = torch.Generator(dev).manual_seed(M)
    r = lambda *s: torch.empty(s, device=dev).normal_(generator=g)  # noqa: E731
    n, way_in = 20000, r(2, 256)
    c = {"q": (way_in.repeat_interleave(4, 0) + 0.1 * r(M, 8, 256)).to(BF16), "k": (0.9 * way_in + 0.05 * r(M, 2, 256)).to(BF16), "v": r(M, 2, 256).to(BF16), "Kp": r(2, 2, n + M, 256).to(BF16),
         "Vp": r(2, 2, n + M, 256).to(BF16), "slots": np.array([1], np.int32), "pos": np.array([n], np.int32), "parents": trees(np.random.default_rng(M), 1, M, "binary")}
    o, _, _ = attn_run(c, dev)
    ref, a, most = attention64(c)
    over = ((o.cpu().double() - ref).abs() / attention_bound(c, ref, a, most)).reshape(M, -1).amax(1)
    assert float(over.max()) <= 1.0, f"{float(over.max()):.2f} of the bound"
    wrong = c["parents"].copy()
    wrong[0, M - 1] = up = (int(wrong[0, M - 1]) + 1) % (M - 1)
    assert up != int(c["parents"][0, M - 1])
    bad, a, most = attention64(c, wrong)
    over = ((o.cpu().double() - bad).abs() / attention_bound(c, bad, a, most)).reshape(M, -1).amax(1)
    assert float(over[:M - 1].max()) <= 1.0 < float(over[M - 1])


# ---- padding --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("M", [5, 14, 40])
def test_padding_sequences_in_a_common_slot(dev, M):
    """sequences that pad a batch may all point at the pools' last slot, as in a decode step: the others' outputs and slots have the bits that they have when each has a slot of
    its own"""
    import qwen_tailor_amd as qt
    gen, B, Lmax = torch.Generator(dev).manual_seed(M), 6, 130
    P = PoolSet(gen, 1, 1, 9, Lmax, dev)
    r = lambda *s: torch.empty(s, dtype=BF16, device=dev).normal_(generator=gen)  # noqa: E731
    i = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    proj, qkv, p, ones = r(B * M, PW), r(B * M, 5120), params(gen, dev), torch.ones(256, dtype=BF16, device=dev)
    parents = i(trees(np.random.default_rng(M), B, M, "random"))
    pos, path, count = i([30, 77, 0, 0, 50, 12]), i([[0, 2, 4]] * B), i([3, 2, 3, 3, 1, 3])
    runs = []
    for slots in ([3, 8, 1, 8, 0, 8], [3, 8, 1, 7, 0, 6]):       # 1, 3 and 5 are padding
        Q, s = P.clone(), i(slots)
        y = qt.batch_tree.deltanet_bt(proj, Q.conv[0], *p, Q.ssm[0], s, pos, parents)
        o = qt.batch_tree.attn_layer_bt(qkv, ones, ones, Q.K[0], Q.V[0], s, pos, parents)
        qt.batch_tree.commit(Q, [proj], [p[0]], [p[1]], [p[2]], s, pos, path, count)
        real = [0, 2, 4]
        runs.append([t.reshape(B, M, -1)[real] for t in (y, o)] + [t[:6] for t in (Q.ssm[0], Q.K[0], Q.V[0])] + [Q.conv[0][:12]])
    for a, b in zip(*runs):
        check_tensors_equal("the others", a, b)


# ---- the largest batch ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("M", [3, 16, 17, 64])
def test_as_many_sequences_as_there_may_be(dev, M):
    """1024 sequences in one call: attention as that of 16 calls of 64 (its sums are split elsewhere: two roundings of the output apart), recurrent step and commit with their bits"""
    import qwen_tailor_amd as qt
    gen, B, Lmax, at = torch.Generator(dev).manual_seed(M), 1024, 40 + M, 64
    P = PoolSet(gen, 1, 1, B, Lmax, dev)
    r = lambda *s: torch.empty(s, dtype=BF16, device=dev).normal_(generator=gen)  # noqa: E731
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    rng = np.random.default_rng(M)
    proj, qkv, p, ones = r(B * M, PW), r(B * M, 5120), params(gen, dev), torch.ones(256, dtype=BF16, device=dev)
    slots, pos, parents = i(rng.permutation(B)), i(rng.integers(0, 41, B)), i(trees(rng, B, M, "random"))
    path, count = i(np.tile(np.arange(min(M, 5)), (B, 1))), i(rng.integers(0, 6, B))

    def run(Q, a, b):
        rows, s = slice(a * M, b * M), slice(a, b)
        y = qt.batch_tree.deltanet_bt(proj[rows], Q.conv[0], *p, Q.ssm[0], slots[s], pos[s], parents[s])
        o = qt.batch_tree.attn_layer_bt(qkv[rows], ones, ones, Q.K[0], Q.V[0], slots[s], pos[s], parents[s])
        qt.batch_tree.commit(Q, [proj[rows]], [p[0]], [p[1]], [p[2]], slots[s], pos[s], path[s], count[s])
        return y, o

    one, many = P.clone(), P.clone()
    y, o = run(one, 0, B)
    parts = [run(many, a, a + at) for a in range(0, B, at)]
    check_tensors_equal("y", y, torch.cat([q[0] for q in parts]))
    for name in ("conv", "ssm", "K", "V"):
        check_tensors_equal(name, getattr(one, name)[0], getattr(many, name)[0])
    want = torch.cat([q[1] for q in parts]).float()
    # o is rounded, then o times the gate: two steps each, and what float sums in another order leave where little is left (values of V are of size 1)
    assert bool(((o.float() - want).abs() <= 4 * 2 ** -8 * want.abs() + 1e-4).all())
