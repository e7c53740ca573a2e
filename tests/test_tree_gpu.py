"""Verification of drafted trees (batch_tree) against 64-bit restatements: attention over cache and ancestors, the GatedDeltaNet step of a tree, the
commit of the accepted path, and a round of all of them.  Sizes: one token to 64, tile borders, empty and long caches, chains, stars, forests, parents
that are none, padding that is not finite, sequences that are skipped."""
import numpy as np
import pytest
import torch

from oracle import gdn_oracle as O
from tests.util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu
NAN = float("nan")


def trees(rng, B, M, shape):
    p = np.full((B, M), -1, np.int32)
    for b in range(B):
        for j in range(1, M):
            p[b, j] = {"chain": j - 1, "star": 0, "forest": -1, "random": int(rng.integers(-1, j)), "deep": j - 1 - int(rng.integers(0, min(j, 2))),
                       "binary": (j - 1) // 2}[shape]
    return p


def up(p, j):
    """the parent that an entry counts as"""
    return int(p[j]) if 0 <= p[j] < j else -1


def way(p, j):
    w = []
    while j >= 0:
        w.append(j)
        j = up(p, j)
    return w[::-1]


# ---- attention ----------------------------------------------------------------------------------------------------------

def attn_reference(q, k, v, Kp, Vp, slots, pos, parents):
    """float64 torch on the GPU; the pools are updated.  -> o [R, 8, 256]"""
    B, M = parents.shape
    out = torch.zeros((B * M, 8, 256), dtype=torch.float64, device=q.device)
    S, Lmax = Kp.shape[0], Kp.shape[2]
    for b in range(B):
        s, n = int(slots[b]), int(pos[b])
        if not (0 <= s < S and 0 <= n <= Lmax - M):
            continue
        kb, vb = k[b * M:(b + 1) * M].double(), v[b * M:(b + 1) * M].double()
        for j in range(M):
            at = torch.tensor(way(parents[b], j), device=q.device)
            for h in range(2):
                K = torch.cat([Kp[s, h, :n].double(), kb[at, h]])
                V = torch.cat([Vp[s, h, :n].double(), vb[at, h]])
                x = q[b * M + j, 4 * h:4 * h + 4].double() @ K.T / 16
                out[b * M + j, 4 * h:4 * h + 4] = torch.softmax(x, -1) @ V
    for b in range(B):
        s, n = int(slots[b]), int(pos[b])
        if 0 <= s < S and 0 <= n <= Lmax - M:
            Kp[s, :, n:n + M], Vp[s, :, n:n + M] = k[b * M:(b + 1) * M].transpose(0, 1), v[b * M:(b + 1) * M].transpose(0, 1)
    return out


def attn_case(dev, seed, B, M, pos, Lmax, shape, scale=1.0):
    rng = np.random.default_rng(seed)
    g = torch.Generator(dev).manual_seed(seed)
    r = lambda *s: torch.empty(s, dtype=BF16, device=dev).normal_(0.0, scale, generator=g)  # noqa: E731
    S = B + 2
    return {"q": r(B * M, 8, 256), "k": r(B * M, 2, 256), "v": r(B * M, 2, 256), "Kp": r(S + 1, 2, Lmax, 256), "Vp": r(S + 1, 2, Lmax, 256),
            "slots": rng.permutation(S)[:B].astype(np.int32), "pos": np.asarray(pos, np.int32), "parents": trees(rng, B, M, shape)}


def attn_run(c, dev):
    import qwen_tailor_amd as qt
    K, V = c["Kp"].clone(), c["Vp"].clone()
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    o = qt.batch_tree.attn_bt(c["q"], c["k"], c["v"], K, V, i(c["slots"]), i(c["pos"]), i(c["parents"]))
    return o, K, V


# An output is a weighted mean of V rows: the rounding of the output is half a bf16 step (2^-9 of it, next to a power of two 2^-8), of P (up to 32 tokens
# two bf16 terms, beyond them one) at most 2^-9 of a weight each, of the scores' sum in float 256 * 2^-24 of |q||k| / 16 in the exponent.  Weights of
# independent V rows average out, so the error stays below 2^-8 |o| + 2^-9 max |V| sqrt(sum w^2) * 4; with softmax weights sum w^2 <= 1.
def check_attn(name, o, ref, vmax):
    d = (o.double() - ref).abs()
    bad = d > 2 ** -8 * ref.abs() + 2 ** -9 * vmax
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} elements off, largest {float(d.max()):.3e}"
    assert rel_l2(to_np(o), to_np(ref)) < 4e-3, name             # (an output's rounding alone: 2^-9 / sqrt(3) * about 1.5)


ATTN = [(1, 1, [0], 8, "star"), (1, 1, [1], 2, "star"), (1, 7, [300], 320, "random"), (2, 8, [31, 32], 64, "chain"), (3, 9, [33, 0, 64], 80, "random"),
        (2, 16, [500, 63], 600, "binary"), (2, 17, [129, 7], 200, "deep"), (1, 32, [1000], 1032, "random"), (2, 33, [95, 96], 129, "random"), (1, 48, [2000], 2048, "star"),
        (2, 64, [0, 1], 65, "chain"), (3, 64, [777, 31, 2500], 2600, "random"), (2, 63, [64, 1234], 1300, "forest"), (5, 3, [5000, 17, 900, 2, 4000], 5003, "random"),
        (40, 5, list(range(1, 400, 10)), 420, "random")]


@pytest.mark.parametrize("B,M,pos,Lmax,shape", ATTN)
def test_attention_of_a_tree(dev, B, M, pos, Lmax, shape):
    c = attn_case(dev, 100 * B + M, B, M, pos, Lmax, shape)
    o, K, V = attn_run(c, dev)
    rK, rV = c["Kp"].clone(), c["Vp"].clone()
    ref = attn_reference(c["q"], c["k"], c["v"], rK, rV, c["slots"], c["pos"], c["parents"])
    check_attn(f"{B} x {M}", o, ref, float(c["Vp"].float().abs().max()))
    check_tensors_equal("K pool", K, rK)
    check_tensors_equal("V pool", V, rV)


def test_attention_skips_and_repeats(dev):
    """slots and positions that do not fit: zero outputs, untouched pools; parents that are none count as -1; the same call gives the same bits"""
    c = attn_case(dev, 5, 6, 12, [10, -1, 50, 53, 20, 2 ** 31 - 1], 64, "random")
    c["slots"][0], c["slots"][4] = -1, 9
    c["parents"][2, :4] = [0, 1, 7, -5]                          # itself, itself, a later token, a negative one: all roots
    o, K, V = attn_run(c, dev)
    rK, rV = c["Kp"].clone(), c["Vp"].clone()
    ref = attn_reference(c["q"], c["k"], c["v"], rK, rV, c["slots"], c["pos"], c["parents"])
    assert not bool(o.reshape(6, -1)[[0, 1, 3, 4, 5]].any())
    check_attn("the others", o, ref, float(c["Vp"].float().abs().max()))
    check_tensors_equal("K pool", K, rK)
    check_tensors_equal("V pool", V, rV)
    for _ in range(3):
        o2, K2, V2 = attn_run(c, dev)
        check_tensors_equal("again", o2, o)


@pytest.mark.parametrize("M", [7, 24, 64])
def test_attention_keeps_what_is_not_finite_to_its_branch(dev, M):
    """NaN and infinities in padding, in other branches, behind the cache and in masked rows reach nothing; a token that sees them is NaN"""
    c = attn_case(dev, M, 1, M, [40], 40 + M + 8, "binary")
    clean, _, _ = attn_run(c, dev)
    bad = 2                                                      # its descendants: 5, 6, 11 ..
    hit = [j for j in range(M) if bad in way(c["parents"][0], j)]
    rest = [j for j in range(M) if j not in hit]
    for what, value in (("k", NAN), ("v", NAN), ("v", float("inf")), ("k", 3e38)):
        d = dict(c)
        d["Kp"], d["Vp"] = c["Kp"].clone(), c["Vp"].clone()
        d["Kp"][:, :, 40:], d["Vp"][:, :, 40:] = NAN, NAN        # never written rows
        d[what] = c[what].clone()
        d[what][bad] = value
        o, _, _ = attn_run(d, dev)
        check_tensors_equal(what, o[rest], clean[rest])
        if value != 3e38:
            assert bool(o[hit].isnan().all()), (what, value)


def test_attention_of_a_chain_is_the_verify_step(dev):
    """a tree that is a chain: what attn_b computes, to the rounding of the output; pools bit-exact"""
    import qwen_tailor_amd as qt
    c = attn_case(dev, 9, 4, 4, [100, 1000, 3, 64], 1100, "chain")
    o, K, V = attn_run(c, dev)
    K2, V2 = c["Kp"].clone(), c["Vp"].clone()
    i = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    o2 = qt.batch.attn_b(c["q"], c["k"], c["v"], K2, V2, i(c["slots"]), i(c["pos"]), 4)
    check_ulp("chain", to_np(o), to_np(o2), 1.0, rel_floor=1e-4)
    check_tensors_equal("K pool", K, K2)
    check_tensors_equal("V pool", V, V2)


def test_attention_large_scores_and_long_cache(dev):
    """scores of a few hundred (one key takes all) and a cache whose pool passes 2^31 bytes"""
    c = attn_case(dev, 3, 2, 20, [333, 90], 400, "random", scale=6.0)
    o, _, _ = attn_run(c, dev)
    ref = attn_reference(c["q"], c["k"], c["v"], c["Kp"].clone(), c["Vp"].clone(), c["slots"], c["pos"], c["parents"])
    check_attn("large scores", o, ref, float(c["Vp"].float().abs().max()))
    c = attn_case(dev, 4, 1, 3, [300000], 400000, "random")      # 4 slots x 2 x 400000 x 512 bytes = 1.6 GB a pool; slot 2 or 3 starts near or beyond 2^30 elements
    for slot in (0, 3):
        c["slots"][0] = slot
        o, K, V = attn_run(c, dev)
        rK, rV = c["Kp"].clone(), c["Vp"].clone()
        ref = attn_reference(c["q"], c["k"], c["v"], rK, rV, c["slots"], c["pos"], c["parents"])
        check_attn("long", o, ref, float(c["Vp"].float().abs().max()) / 8)
        check_tensors_equal("K pool", K, rK)


LAYER = [(1, 7, [300], 320, "random"), (3, 16, [100, 0, 777], 800, "binary"), (2, 40, [64, 500], 560, "deep"), (2, 64, [3, 1500], 1600, "random"), (4, 1, [0, 5, 31, 32], 40, "star"),
         (40, 5, list(range(1, 400, 10)), 420, "random"), (33, 12, [33 * (k % 7) for k in range(33)], 300, "deep"), (300, 2, [k % 50 for k in range(300)], 60, "chain"),
         (1, 16, [20000], 20016, "random")]


@pytest.mark.parametrize("B,M,pos,Lmax,shape", LAYER)
def test_attention_layer_of_a_tree(dev, B, M, pos, Lmax, shape):
    """attn_layer_bt is qkv_prep at the tokens' positions + attn_bt + out_gate: the same bits"""
    import qwen_tailor_amd as qt
    c = attn_case(dev, 7 * B + M, B, M, pos, Lmax, shape)
    g = torch.Generator(dev).manual_seed(M)
    qkv = torch.empty((B * M, 5120), dtype=BF16, device=dev).normal_(generator=g)
    qn, kn = ((1 + 0.1 * torch.empty(256, device=dev).normal_(generator=g)).to(BF16) for _ in range(2))
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    at = np.array([int(pos[b]) + len(way(c["parents"][b], j)) - 1 for b in range(B) for j in range(M)])
    q, k, v = qt.attention.qkv_prep(qkv, qn, kn, i(at))
    K, V = c["Kp"].clone(), c["Vp"].clone()
    o = qt.batch_tree.attn_bt(q, k, v, K, V, i(c["slots"]), i(pos), i(c["parents"]))
    want = qt.attention.out_gate(o, qkv)
    K2, V2 = c["Kp"].clone(), c["Vp"].clone()
    got = qt.batch_tree.attn_layer_bt(qkv, qn, kn, K2, V2, i(c["slots"]), i(pos), i(c["parents"]))
    check_tensors_equal("out", got, want)
    check_tensors_equal("K pool", K2, K)
    check_tensors_equal("V pool", V2, V)


@pytest.mark.parametrize("B,M,pos,Lmax,shape", [(2, 7, [300, 0], 320, "random"), (3, 16, [100, 31, 184], 200, "deep"), (2, 24, [64, 5], 100, "random")])
def test_attention_layer_without_a_whole_table(dev, B, M, pos, Lmax, shape):
    """the C entry with no table of rotary pairs, or one that ends early: the same bits"""
    import qwen_tailor_amd as qt
    c = attn_case(dev, 3 * B + M, B, M, pos, Lmax, shape)
    g = torch.Generator(dev).manual_seed(M)
    qkv = torch.empty((B * M, 5120), dtype=BF16, device=dev).normal_(generator=g)
    qn, kn = ((1 + 0.1 * torch.empty(256, device=dev).normal_(generator=g)).to(BF16) for _ in range(2))
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    idx = [i(c["slots"]), i(pos), i(c["parents"])]
    K, V = c["Kp"].clone(), c["Vp"].clone()
    want = qt.batch_tree.attn_layer_bt(qkv, qn, kn, K, V, *idx)
    ptr, n = qt._lib.ptr, qt._lib.lib().qt_gqa_tree_layer_workspace_bytes(B, M)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    short = torch.empty((Lmax - 1, 32, 2), device=dev)
    qt._lib.call("qt_rope_table_build", ptr(short), Lmax - 1, qt._lib.stream())
    for table, positions in ((None, 0), (short, Lmax - 1), (short, 40)):
        K2, V2, out = c["Kp"].clone(), c["Vp"].clone(), torch.empty_like(want)
        qt._lib.call("qt_gqa_tree_layer", ptr(qkv), ptr(qn), ptr(kn), ptr(table), positions, ptr(K2), ptr(V2), *[ptr(t) for t in idx], ptr(out), ptr(ws), n, B, M, Lmax,
                     K.shape[0], 1e-6, qt._lib.stream())
        check_tensors_equal("out", out, want)
        check_tensors_equal("K pool", K2, K)
        check_tensors_equal("V pool", V2, V)


@pytest.mark.parametrize("M", [5, 16])
def test_attention_layer_keeps_what_is_not_finite_to_its_branch(dev, M):
    """NaN in a drafted token's q, k or v row, in never written rows and in the rows of a skipped sequence"""
    import qwen_tailor_amd as qt
    B, Lmax = 2, 90
    c = attn_case(dev, M, B, M, [50, 0], Lmax, "binary")
    g = torch.Generator(dev).manual_seed(M)
    qkv = torch.empty((B * M, 5120), dtype=BF16, device=dev).normal_(generator=g)
    qn, kn = ((1 + 0.1 * torch.empty(256, device=dev).normal_(generator=g)).to(BF16) for _ in range(2))
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    c["slots"][1] = -1
    run = lambda x, K, V: qt.batch_tree.attn_layer_bt(x, qn, kn, K, V, i(c["slots"]), i([50, 0]), i(c["parents"]))  # noqa: E731
    clean = run(qkv, c["Kp"].clone(), c["Vp"].clone())
    assert not bool(clean[M:].any())
    hit = [j for j in range(M) if 2 in way(c["parents"][0], j)]
    for cols, touched in ((slice(0, 256), [2]), (slice(4096, 4352), hit), (slice(4608, 4864), hit)):
        x, K, V = qkv.clone(), c["Kp"].clone(), c["Vp"].clone()
        K[:, :, 50:], V[:, :, 50:] = NAN, NAN
        x[2, cols], x[M:] = NAN, NAN
        y = run(x, K, V)
        rest = [j for j in range(B * M) if j not in touched]
        check_tensors_equal(f"{cols}", y[rest], clean[rest])
        assert bool(y[touched][:, :256].isnan().all()), cols


# ---- the recurrent layers ------------------------------------------------------------------------------------------------

def gdn_case(seed, B, M, shape, scale=1.0):
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    cw, A_log, dtb, _ = layer_params(seed)
    return {"proj": rand_bf(gen, (B * M, PW), scale), "conv": rand_bf(gen, ((B + 1) * 2, 3, CD)), "ssm": (torch.randn((B + 1, 16, 128, 128), generator=gen) * 0.05).numpy(),
            "cw": cw, "A_log": A_log, "dtb": dtb, "slots": rng.permutation(B + 1)[:B].astype(np.int32), "pos": rng.integers(0, 1000, B).astype(np.int32),
            "parents": trees(rng, B, M, shape)}


def gdn_run(c, dev):
    import qwen_tailor_amd as qt
    conv, ssm = to_dev(c["conv"], dev, BF16), to_dev(c["ssm"], dev)
    y = qt.batch_tree.deltanet_bt(to_dev(c["proj"], dev, BF16), conv, to_dev(c["cw"], dev, BF16), to_dev(c["A_log"], dev), to_dev(c["dtb"], dev), ssm,
                                  to_dev(c["slots"], dev), to_dev(c["pos"], dev), to_dev(c["parents"], dev))
    check_equal("conv pool", to_np(conv), c["conv"])
    check_equal("ssm pool", to_np(ssm), c["ssm"])
    return y


def gdn_reference(c):
    """every token by the sequential oracle along its own path (states of shared ancestors are formed once)"""
    B, M = c["parents"].shape
    y = np.zeros((B * M, 2048))
    for b in range(B):
        slot = int(c["slots"][b])
        win = c["conv"][2 * slot + (int(c["pos"][b]) & 1)]
        ends = {-1: (win, c["ssm"][slot].astype(np.float64))}
        for j in range(M):
            w, S = ends[up(c["parents"][b], j)]
            cs, st, yy = step(c["proj"][b * M + j], w, S, c)
            ends[j] = (cs, st)
            y[b * M + j] = yy
    return y


def step(row, win, S, c):
    """one token of the layer core by the oracle's parts: bf16 prologue, float64 recurrence, unrounded output"""
    u = O.conv_silu(win, row[:CD], c["cw"])
    q, k = O.normalize_qk(u[:2048].reshape(16, 128), u[2048:4096].reshape(16, 128))
    v = u[4096:].reshape(16, 128)
    g, beta = O.gates(row[8208:8224], row[8192:8208], c["A_log"], c["dtb"])
    q, k, v, g, beta = (np.asarray(t, np.float64) for t in (q, k, v, g, beta))
    S = S * g[:, None, None]
    delta = (v - np.einsum("hvk,hk->hv", S, k)) * beta[:, None]
    S = S + delta[:, :, None] * k[:, None, :]
    return np.concatenate([win[1:], row[None, :CD]]), S, np.einsum("hvk,hk->hv", S, q).ravel()


GDN = [(1, 1, "star"), (1, 2, "chain"), (1, 7, "random"), (2, 15, "binary"), (2, 16, "random"), (1, 17, "chain"), (1, 31, "deep"), (2, 32, "random"), (1, 33, "star"),
       (1, 47, "random"), (1, 48, "chain"), (1, 49, "forest"), (1, 64, "chain"), (2, 64, "random"), (20, 5, "random")]


@pytest.mark.parametrize("B,M,shape", GDN)
def test_gdn_step_of_a_tree(dev, B, M, shape):
    """y in bf16: half a step of rounding (one where the oracle's lies next to a border), and what the state's two bf16 terms (2^-18 of an element) and float sums
    leave of 128 products: below 1e-4 of the largest output"""
    c = gdn_case(10 * M + B, B, M, shape)
    check_ulp(f"{B} x {M}", to_np(gdn_run(c, dev)), gdn_reference(c), 0.75, rel_floor=1e-4)


def test_gdn_step_equal_keys_and_slow_decay(dev):
    """a chain of 64 equal tokens (L is full, its powers grow) with hardly any decay: the solve has to stay exact"""
    c = gdn_case(77, 1, 64, "chain")
    c["proj"][:] = c["proj"][:1]
    c["conv"][:] = c["proj"][0, :CD]
    c["proj"][:, 8192:8208] = 8.0                                # beta = 1
    c["proj"][:, 8208:8224] = -8.0                               # g = 0.9997 ..
    check_ulp("equal keys", to_np(gdn_run(c, dev)), gdn_reference(c), 0.75, rel_floor=1e-4)


def test_gdn_step_forgetful_heads(dev):
    """decays whose products pass below the smallest float on the way down, beside heads that keep everything"""
    c = gdn_case(78, 1, 64, "deep")
    c["A_log"][::2] = 6.0
    c["proj"][::3, 8208:8224] = 30.0
    check_ulp("decay", to_np(gdn_run(c, dev)), gdn_reference(c), 0.75, rel_floor=1e-4)


def test_gdn_step_of_a_chain_is_the_verify_step(dev):
    import qwen_tailor_amd as qt
    B, M = 3, 6
    c = gdn_case(5, B, M, "chain")
    y = to_np(gdn_run(c, dev))
    sp = qt.batch_spec.SpecPools(qt.model.Cfg(layers=1), B, B, M, 8, device=dev)
    for b in range(B):
        sp.ssm[0][b, 0] = to_dev(c["ssm"][c["slots"][b]], dev)
        sp.conv[0][2 * b, 0] = to_dev(c["conv"][2 * c["slots"][b] + (c["pos"][b] & 1)], dev, BF16)
    z = torch.zeros(B, dtype=torch.int32, device=dev)
    y2 = qt.batch_spec.deltanet_bm(to_dev(c["proj"], dev, BF16), sp.conv[0], to_dev(c["cw"], dev, BF16), to_dev(c["A_log"], dev), to_dev(c["dtb"], dev), sp.ssm[0],
                                   torch.arange(B, dtype=torch.int32, device=dev), z, z, M)
    check_ulp("chain", y, to_np(y2), 1.0, rel_floor=1e-4)


@pytest.mark.parametrize("M", [10, 64])
def test_gdn_step_keeps_what_is_not_finite_to_its_branch(dev, M):
    c = gdn_case(M, 1, M, "binary")
    clean = gdn_run(c, dev)
    for at, value in ((100, NAN), (2048 + 5, float("inf")), (4096 + 130, NAN), (4096 + 130, 2.0 ** 126), (8192 + 1, NAN), (8208 + 1, NAN)):
        d = dict(c)
        d["proj"] = c["proj"].copy()
        d["proj"][2, at] = value
        y = gdn_run(d, dev)
        # the conv takes a token's row into the next three of its branch, so every descendant is met either way
        hit = [j for j in range(M) if 2 in way(c["parents"][0], j)]
        rest = [j for j in range(M) if j not in hit]
        head = (at % 2048) // 128 if at < 6144 else 1
        cols = slice(128 * head, 128 * head + 128)
        check_tensors_equal(f"{at}", y[rest], clean[rest])
        if value != 2.0 ** 126:
            assert bool(y[hit][:, cols].isnan().all()), (at, value)
        others = [k for k in range(2048) if not 128 * head <= k < 128 * head + 128]
        check_tensors_equal(f"{at}: the other heads", y[:, others], clean[:, others])


def test_gdn_step_skips(dev):
    c = gdn_case(3, 4, 9, "random")
    keep = c["slots"].copy()
    c["slots"][1], c["slots"][3] = -1, 5
    y = gdn_run(c, dev).reshape(4, -1)
    assert not bool(y[1].any()) and not bool(y[3].any())
    c["slots"] = keep
    check_tensors_equal("the others", y[[0, 2]], gdn_run(c, dev).reshape(4, -1)[[0, 2]])


@pytest.mark.parametrize("M", [16, 17, 33, 64])
def test_gdn_step_without_the_table(dev, M):
    """the C entry takes a null table of SiLU: it evaluates the function, the same bits"""
    import qwen_tailor_amd as qt
    c = gdn_case(300 + M, 2, M, "random", scale=3.0)
    want = gdn_run(c, dev)
    t = [to_dev(c["proj"], dev, BF16), to_dev(c["conv"], dev, BF16), to_dev(c["cw"], dev, BF16)] + [to_dev(c[n], dev) for n in ("A_log", "dtb", "ssm", "slots", "pos", "parents")]
    y = torch.empty_like(want)
    qt._lib.call("qt_gdn_tree_step", *[qt._lib.ptr(x) for x in t], None, qt._lib.ptr(y), 2, M, 3, qt._lib.stream())
    check_tensors_equal("y", y, want)


# ---- the commit ----------------------------------------------------------------------------------------------------------

class PoolSet:
    def __init__(self, gen, n_gdn, n_kv, slots, Lmax, dev):
        r = lambda shape, dt, s=1.0: torch.empty(shape, dtype=dt, device=dev).normal_(0.0, s, generator=gen)  # noqa: E731
        self.conv = [r((slots * 2, 3, CD), BF16) for _ in range(n_gdn)]
        self.ssm = [r((slots, 16, 128, 128), torch.float32, 0.05) for _ in range(n_gdn)]
        self.K = [r((slots, 2, Lmax, 256), BF16) for _ in range(n_kv)]
        self.V = [r((slots, 2, Lmax, 256), BF16) for _ in range(n_kv)]

    def clone(self):
        p = PoolSet.__new__(PoolSet)
        for name in ("conv", "ssm", "K", "V"):
            setattr(p, name, [t.clone() for t in getattr(self, name)])
        return p


def params(gen, dev):
    cw = torch.empty((CD, 4, 1), dtype=BF16, device=dev).normal_(0.0, 0.5, generator=gen)
    return cw, torch.empty(16, device=dev).uniform_(0.0, 2.7, generator=gen), torch.empty(16, device=dev).normal_(0.0, 0.1, generator=gen)


COMMIT = [(1, 7, 4, 3, 1), (3, 16, 16, 2, 2), (5, 64, 9, 1, 1), (2, 1, 1, 1, 1), (4, 33, 64, 1, 3), (2, 8, 3, 2, 0), (2, 8, 8, 0, 2), (2, 20, 5, 35, 1), (1, 5, 5, 1, 40)]


@pytest.mark.parametrize("B,M,D,n_gdn,n_kv", COMMIT)
def test_commit_is_so_many_decode_steps(dev, B, M, D, n_gdn, n_kv):
    """states and windows: the bits of single decode steps; K / V rows moved, everything else untouched; counts from 0 to the whole path"""
    import qwen_tailor_amd as qt
    rng = np.random.default_rng(B * M + D)
    gen = torch.Generator(dev).manual_seed(M)
    Lmax = 2 * M + 20
    P = PoolSet(gen, n_gdn, n_kv, B + 2, Lmax, dev)
    parents = trees(rng, B, M, "random" if M < 20 else "deep")
    path, count = np.zeros((B, D), np.int32), np.zeros(B, np.int32)
    for b in range(B):
        w = max((way(parents[b], j) for j in range(M)), key=len)[:D]
        path[b, :len(w)] = w
        count[b] = len(w) if b != 1 else 0
    pos = rng.integers(0, Lmax - M + 1, B).astype(np.int32)
    slots = rng.permutation(B + 2)[:B].astype(np.int32)
    projs = [torch.empty((B * M, PW), dtype=BF16, device=dev).normal_(generator=gen) for _ in range(n_gdn)]
    ps = [params(gen, dev) for _ in range(n_gdn)]
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    want = P.clone()
    for b in range(B):
        for l in range(n_gdn):
            cw, A, dt = ps[l]
            for t in range(count[b]):
                qt.batch.deltanet_b(projs[l][b * M + int(path[b, t])][None], want.conv[l], cw, A, dt, want.ssm[l], i(slots[b:b + 1]), i(pos[b:b + 1] + t))
        for pool, old in list(zip(want.K, P.K)) + list(zip(want.V, P.V)):
            for t in range(count[b]):
                pool[slots[b], :, pos[b] + t] = old[slots[b], :, pos[b] + path[b, t]]
    got = P.clone()
    qt.batch_tree.commit(got, projs, [p[0] for p in ps], [p[1] for p in ps], [p[2] for p in ps], i(slots), i(pos), i(path), i(count), M=M)
    for name in ("ssm", "K", "V"):
        for a, b in zip(getattr(got, name), getattr(want, name)):
            check_tensors_equal(name, a, b)
    for l in range(n_gdn):                                       # (the buffers that no step will read hold what single steps have left there)
        live = [2 * s + ((p + n) & 1) for s, p, n in zip(slots.tolist(), pos.tolist(), count.tolist())]
        check_tensors_equal("conv", got.conv[l][live], want.conv[l][live])
        rest = [k for k in range(2 * (B + 2)) if k // 2 not in slots.tolist()]
        check_tensors_equal("other conv", got.conv[l][rest], P.conv[l][rest])


def test_commit_skips(dev):
    """slots that are none, counts below zero, positions whose rows do not fit, path entries that are no token"""
    import qwen_tailor_amd as qt
    gen = torch.Generator(dev).manual_seed(1)
    B, M, Lmax = 5, 6, 40
    P = PoolSet(gen, 1, 1, 7, Lmax, dev)
    proj, p = torch.empty((B * M, PW), dtype=BF16, device=dev).normal_(generator=gen), params(gen, dev)
    i = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    got = P.clone()
    qt.batch_tree.commit(got, [proj], [p[0]], [p[1]], [p[2]], i([-1, 7, 2, 3, 4]), i([3, 3, 35, -2, 5]), i([[0, 1, 2]] * B), i([3, 3, 3, 3, -1]))
    for name in ("conv", "ssm", "K", "V"):
        check_tensors_equal(name, getattr(got, name)[0], getattr(P, name)[0])
    a, b = P.clone(), P.clone()                                  # (an entry that is none counts as token 0)
    qt.batch_tree.commit(a, [proj], [p[0]], [p[1]], [p[2]], i([0, 1, 2, 3, 4]), i([3] * 5), i([[0, 99, -1]] * B), i([3] * 5))
    qt.batch_tree.commit(b, [proj], [p[0]], [p[1]], [p[2]], i([0, 1, 2, 3, 4]), i([3] * 5), i([[0, 0, 0]] * B), i([3] * 5))
    for name in ("conv", "ssm"):
        check_tensors_equal(name, getattr(a, name)[0], getattr(b, name)[0])


def test_commit_gathers_whatever_the_path_says(dev):
    """K / V rows of a path that goes down no tree (backwards, repeated): every row as it was before the call"""
    import qwen_tailor_amd as qt
    gen = torch.Generator(dev).manual_seed(2)
    B, M, D, Lmax = 2, 64, 64, 100
    P = PoolSet(gen, 0, 2, 3, Lmax, dev)
    path = torch.stack([torch.arange(63, -1, -1), torch.arange(64) // 5 * 3]).to(torch.int32).to(dev)
    slots, pos, count = (torch.tensor(a, dtype=torch.int32, device=dev) for a in ([2, 0], [36, 5], [64, 41]))
    got = P.clone()
    qt.batch_tree.commit(got, [], [], [], [], slots, pos, path, count, M=M)
    for name in ("K", "V"):
        for a, old in zip(getattr(got, name), getattr(P, name)):
            want = old.clone()
            for b, (s, p, n) in enumerate([(2, 36, 64), (0, 5, 41)]):
                want[s, :, p:p + n] = old[s][:, (p + path[b, :n]).long()]
            check_tensors_equal(name, a, want)


# ---- a round ------------------------------------------------------------------------------------------------------------

def test_a_round_of_drafting_leaves_what_decode_steps_would(dev):
    """two layers (one recurrent, one attention), two sequences: the tree step's outputs along the accepted path are those of single decode steps, and
    after the commit so are pools and the next step.  Once eagerly, and as a captured graph replayed three times with other work in between"""
    import qwen_tailor_amd as qt
    gen = torch.Generator(dev).manual_seed(11)
    rng = np.random.default_rng(11)
    B, M, Lmax = 2, 13, 200
    P = PoolSet(gen, 1, 1, B + 1, Lmax, dev)
    r = lambda *s: torch.empty(s, dtype=BF16, device=dev).normal_(generator=gen)  # noqa: E731
    proj, qkv, nxt, nqkv = r(B * M, PW), r(B * M, 5120), r(B, PW), r(B, 5120)
    cw, A, dt = params(gen, dev)
    qn, kn = ((1 + 0.1 * r(256).float()).to(BF16) for _ in range(2))
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    parents = trees(rng, B, M, "random")
    parents[0, 1:5], parents[1, 1:8] = [0, 1, 2, 3], [0, 1, 1, 3, 4, 5, 6]
    ways = [[0, 1, 2, 3, 4], [0, 1, 3, 4, 5, 6, 7]]
    path, count = np.zeros((B, 8), np.int32), np.array([5, 7], np.int32)
    for b in range(B):
        path[b, :count[b]] = ways[b]
    slots, pos = i([2, 0]), i([77, 100])
    dparents, dpath, dcount = i(parents), i(path), i(count)
    W = P.clone()
    y_ref, o_ref = [[], []], [[], []]
    for b in range(B):
        for t, j in enumerate(ways[b]):
            at = pos[b:b + 1] + t
            y_ref[b].append(qt.batch.deltanet_b(proj[b * M + j][None], W.conv[0], cw, A, dt, W.ssm[0], slots[b:b + 1], at))
            o_ref[b].append(qt.batch.attn_layer_b(qkv[b * M + j][None], qn, kn, W.K[0], W.V[0], slots[b:b + 1], at))
    pos2 = pos + dcount
    want_next = (qt.batch.deltanet_b(nxt, W.conv[0], cw, A, dt, W.ssm[0], slots, pos2), qt.batch.attn_layer_b(nqkv, qn, kn, W.K[0], W.V[0], slots, pos2))

    T = P.clone()

    def a_round():
        y = qt.batch_tree.deltanet_bt(proj, T.conv[0], cw, A, dt, T.ssm[0], slots, pos, dparents)
        o = qt.batch_tree.attn_layer_bt(qkv, qn, kn, T.K[0], T.V[0], slots, pos, dparents)
        qt.batch_tree.commit(T, [proj], [cw], [A], [dt], slots, pos, dpath, dcount)
        return y, o

    def reset():
        for name in ("conv", "ssm", "K", "V"):
            for a, b in zip(getattr(T, name), getattr(P, name)):
                a.copy_(b)

    def check(y, o):
        for b in range(B):
            at = [b * M + j for j in ways[b]]
            check_ulp("y", to_np(y[at]), to_np(torch.cat(y_ref[b])), 1.0, rel_floor=1e-4)
            check_ulp("o", to_np(o[at]), to_np(torch.cat(o_ref[b])), 2.0, rel_floor=1e-4)      # (a step of o, through the gate)
        check_tensors_equal("ssm", T.ssm[0], W0.ssm[0])
        for name in ("K", "V"):
            for b, s in enumerate(slots.tolist()):
                n = int(pos2[b])
                check_tensors_equal(name, getattr(T, name)[0][s, :, :n], getattr(W, name)[0][s, :, :n])
        Z = T.clone()
        z = (qt.batch.deltanet_b(nxt, Z.conv[0], cw, A, dt, Z.ssm[0], slots, pos2), qt.batch.attn_layer_b(nqkv, qn, kn, Z.K[0], Z.V[0], slots, pos2))
        check_tensors_equal("next y", z[0], want_next[0])
        check_tensors_equal("next o", z[1], want_next[1])

    W0 = P.clone()                                               # the state before the next step
    for b in range(B):
        for t, j in enumerate(ways[b]):
            qt.batch.deltanet_b(proj[b * M + j][None], W0.conv[0], cw, A, dt, W0.ssm[0], slots[b:b + 1], pos[b:b + 1] + t)
    y, o = a_round()
    check(y, o)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        reset()
        a_round()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            gy, go = a_round()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        check(gy, go)
        check_tensors_equal("y again", gy, y)
        check_tensors_equal("o again", go, o)


def both_layers(case, P, dev):
    """one tree step of a recurrent and an attention layer, as a function of nothing"""
    import qwen_tailor_amd as qt
    proj, qkv, p, qn, kn, slots, pos, parents = case
    return (qt.batch_tree.deltanet_bt(proj, P.conv[0], *p, P.ssm[0], slots, pos, parents), qt.batch_tree.attn_layer_bt(qkv, qn, kn, P.K[0], P.V[0], slots, pos, parents),
            qt.batch_tree.attn_bt(qkv[:, :2048].reshape(-1, 8, 256).contiguous(), qkv[:, 4096:4608].reshape(-1, 2, 256).contiguous(),
                                  qkv[:, 4608:].reshape(-1, 2, 256).contiguous(), P.K[0], P.V[0], slots, pos, parents))


def layer_case(gen, seed, B, M, Lmax, dev):
    rng = np.random.default_rng(seed)
    r = lambda *s: torch.empty(s, dtype=BF16, device=dev).normal_(generator=gen)  # noqa: E731
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    qn, kn = ((1 + 0.1 * r(256).float()).to(BF16) for _ in range(2))
    return r(B * M, PW), r(B * M, 5120), params(gen, dev), qn, kn, i(rng.permutation(B + 1)[:B]), i(rng.integers(0, Lmax - M, B)), i(trees(rng, B, M, "random"))


SHAPES = [(1, 7, 100), (3, 24, 700), (2, 64, 300)]


def test_calls_from_threads_on_streams_of_their_own(dev):
    """the same bits as one after the other: no scratch in common between streams"""
    import threading
    gen = torch.Generator(dev).manual_seed(21)
    cases = [(layer_case(gen, k, B, M, L, dev), PoolSet(gen, 1, 1, B + 1, L, dev)) for k, (B, M, L) in enumerate(SHAPES)]
    want = [both_layers(c, P, dev) for c, P in cases]
    torch.cuda.synchronize()
    got, errors = [None] * len(cases), []

    def work(k):
        try:
            with torch.cuda.device(dev), torch.cuda.stream(torch.cuda.Stream()):
                got[k] = [both_layers(*cases[k], dev) for _ in range(10)]
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for w, g in zip(want, got):
        for again in g:
            for a, b in zip(again, w):
                check_tensors_equal("out", a, b)


def test_graphs_captured_on_one_stream_replayed_side_by_side(dev):
    """each graph has scratch of its own: replayed on two streams at once, with eager calls between, the outputs are those of eager calls"""
    gen = torch.Generator(dev).manual_seed(22)
    cases = [(layer_case(gen, k, B, M, L, dev), PoolSet(gen, 1, 1, B + 1, L, dev)) for k, (B, M, L) in enumerate(SHAPES)]
    want = [both_layers(c, P, dev) for c, P in cases]
    side, graphs, outs = torch.cuda.Stream(), [], []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c, P in cases:
            both_layers(c, P, dev)
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(both_layers(c, P, dev))
            graphs.append(g)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(4):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
            graphs[1].replay()
        with torch.cuda.stream(other):
            graphs[2].replay()
        eager = both_layers(*cases[1], dev)                      # (the pool rows that it writes are those that the graph writes: the same values)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for a, b in zip(o, w):
                check_tensors_equal("replayed", a, b)
        for a, b in zip(eager, want[1]):
            check_tensors_equal("eager", a, b)


# ---- refusals ------------------------------------------------------------------------------------------------------------

def test_refusals(dev):
    import qwen_tailor_amd as qt
    T, z = qt.batch_tree, lambda *s, dt=BF16: torch.zeros(s, dtype=dt, device=dev)  # noqa: E731
    i = lambda *s: z(*s, dt=torch.int32)  # noqa: E731
    good = dict(proj=z(8, PW), conv=z(6, 3, CD), cw=z(CD, 4), A=z(16, dt=torch.float32), dt=z(16, dt=torch.float32), ssm=z(3, 16, 128, 128, dt=torch.float32),
                slots=i(2), pos=i(2), parents=i(2, 4))
    for key, value, err in (("proj", z(9, PW), ValueError), ("proj", z(8, PW).float(), TypeError), ("proj", z(8, 2 * PW)[:, ::2], ValueError), ("conv", z(5, 3, CD), ValueError),
                            ("cw", z(CD, 3), ValueError), ("A", z(15, dt=torch.float32), ValueError), ("ssm", z(3, 16, 128, 128), TypeError), ("slots", i(3), ValueError),
                            ("pos", z(2, dt=torch.int64), TypeError), ("parents", i(8), ValueError), ("parents", i(1, 4), ValueError)):
        with pytest.raises(err):
            T.deltanet_bt(*{**good, key: value}.values())
    with pytest.raises(ValueError):
        T.deltanet_bt(*{**good, "proj": z(130, PW), "parents": i(2, 65)}.values())
    a = dict(q=z(8, 8, 256), k=z(8, 2, 256), v=z(8, 2, 256), K=z(3, 2, 20, 256), V=z(3, 2, 20, 256), slots=i(2), pos=i(2), parents=i(2, 4))
    for key, value, err in (("q", z(8, 8, 128), ValueError), ("k", z(7, 2, 256), ValueError), ("V", z(3, 2, 21, 256), ValueError), ("K", z(3, 2, 20, 256).half(), TypeError),
                            ("parents", i(4, 4), ValueError), ("slots", i(1), ValueError), ("v", z(2, 8, 256).transpose(0, 1), ValueError)):
        with pytest.raises(err):
            T.attn_bt(*{**a, key: value}.values())
    with pytest.raises(ValueError):
        T.attn_bt(*{**a, "q": z(1025, 8, 256), "k": z(1025, 2, 256), "v": z(1025, 2, 256), "slots": i(1025), "pos": i(1025), "parents": i(1025, 1)}.values())
    with pytest.raises(ValueError):
        T.attn_layer_bt(z(8, 5119), z(256), z(256), a["K"], a["V"], a["slots"], a["pos"], a["parents"])
    P = qt.batch.Pools(qt.model.Cfg(layers=4), 2, 20, device=dev)
    c = dict(projs=[z(8, PW)] * 3, cws=[z(CD, 4)] * 3, As=[z(16, dt=torch.float32)] * 3, dts=[z(16, dt=torch.float32)] * 3, slots=i(2), pos=i(2), path=i(2, 3), count=i(2))
    for key, value, err in (("projs", [z(8, PW)] * 2, ValueError), ("projs", [z(7, PW)] * 3, ValueError), ("path", i(2, 65), ValueError), ("count", i(3), ValueError),
                            ("projs", [z(130, PW)] * 3, ValueError), ("As", [z(16, dt=torch.float32)], ValueError)):
        with pytest.raises(err):
            T.commit(P, *{**c, key: value}.values())
    with pytest.raises(ValueError):
        T.commit(P, *c.values(), M=5)
    # no sequences
    assert T.deltanet_bt(*{**good, "proj": z(0, PW), "slots": i(0), "pos": i(0), "parents": i(0, 4)}.values()).shape == (0, 2048)
    assert T.attn_bt(*{**a, "q": z(0, 8, 256), "k": z(0, 2, 256), "v": z(0, 2, 256), "slots": i(0), "pos": i(0), "parents": i(0, 4)}.values()).shape == (0, 8, 256)
    T.commit(P, [z(0, PW)] * 3, c["cws"], c["As"], c["dts"], i(0), i(0), i(0, 3), i(0))
