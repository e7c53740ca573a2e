"""Beam search on the pools (batch_beam): the selection over beams and vocabulary against float64, and the reordering of states against indexing."""
import numpy as np
import pytest
import torch

from tests.util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def reference(logits, scores, n):
    """float64 on the CPU: (scores, parents, tokens), and all candidates' scores [G, W V]"""
    x, s = logits.detach().cpu().double(), scores.detach().cpu().double()
    G, W, V = x.shape
    top = x.amax(-1, keepdim=True)
    c = (s[..., None] + ((x - top) - torch.log(torch.exp(x - top).sum(-1, keepdim=True)))).reshape(G, W * V)
    c = torch.where(c.isnan(), torch.tensor(-INF, dtype=torch.float64), c)
    best, at = c.sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    if best.shape[1] < n:
        best = torch.cat([best, torch.full((G, n - best.shape[1]), -INF, dtype=torch.float64)], 1)
        at = torch.cat([at, torch.zeros((G, n - at.shape[1]), dtype=at.dtype)], 1)
    none = best == -INF
    return best, torch.where(none, -1, at // V), torch.where(none, -1, at % V), c


# The sum of up to 2^18 exponentials in float, lanes' sums of a few hundred terms first: below 2^-24 * 128 of it, and the exponential's argument in float (2^-24 of
# a logit difference of up to 30, times log2 e): together below 1.5e-5 of l; the score is rounded to float once.
TOL = 2e-5


def check(logits, scores, n):
    import qwen_tailor_amd as qt
    got = qt.batch_beam.select(logits, scores, n)
    best, w, t, every = reference(logits, scores, n)
    gs, gw, gt = got[0].cpu().double(), got[1].cpu().long(), got[2].cpu().long()
    V = logits.shape[2]
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int32
    assert torch.equal(gs == -INF, best == -INF), "number of candidates"
    for g in range(gs.shape[0]):
        k = int((best[g] > -INF).sum())
        assert (gw[g, k:] == -1).all() and (gt[g, k:] == -1).all()
        if not k:
            continue
        flat = gw[g, :k] * V + gt[g, :k]
        assert len(set(flat.tolist())) == k, "a candidate twice"
        err = (gs[g, :k] - best[g, :k]).abs()
        assert float(err.max()) <= TOL * max(1.0, float(best[g, :k].abs().max())), float(err.max())
        # places of two candidates may only be changed where their scores lie closer than the scores are known (candidates of one beam never)
        same = (gw[g, :k] == w[g, :k]) & (gt[g, :k] == t[g, :k])
        for i in torch.nonzero(~same).flatten().tolist():
            assert abs(float(every[g, flat[i]]) - float(best[g, i])) <= TOL, (g, i)
            assert int(gw[g, i]) != int(w[g, i]), "order within a beam"
    return got


def case(dev, seed, G, W, V, dtype, scale=2.5):
    g = torch.Generator(dev).manual_seed(seed)
    x = torch.empty((G, W, V), dtype=dtype, device=dev).normal_(0.0, scale, generator=g)
    return x, torch.empty((G, W), device=dev).uniform_(-12.0, -2.0, generator=g)


SIZES = [(1, 1, 1, 1), (1, 1, 2, 3), (1, 3, 5, 20), (2, 1, 63, 4), (1, 2, 64, 64), (3, 4, 1000, 5), (1, 1, 2047, 8), (2, 5, 4097, 10), (1, 64, 3001, 64), (4, 16, 32003, 16),
         (1, 1, 248320, 8), (2, 4, 248320, 4), (1, 1, 262143, 64), (33, 2, 50257, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("G,W,V,n", SIZES)
def test_select(dev, G, W, V, n, dtype):
    check(*case(dev, G + W + V + n, G, W, V, dtype), n)


@pytest.mark.parametrize("V", [300, 9001, 100003])
@pytest.mark.parametrize("n", [1, 7, 64])
def test_select_orders_that_fill_the_lists(dev, V, n):
    """rising logits (every one enters), falling, all equal, two values, one spike"""
    up = torch.arange(V, device=dev, dtype=torch.float32) * 1e-4
    s = torch.tensor([[-1.0, -1.0]], device=dev)
    for row in (up, up.flip(0), torch.zeros(V, device=dev), (torch.arange(V, device=dev) % 3 == 1).float(), torch.nn.functional.one_hot(torch.tensor(V - 1, device=dev), V).float() * 9):
        for dtype in (torch.float32, torch.bfloat16):
            x = torch.stack([row, row])[None].to(dtype)          # two equal beams: ties between them go to the first
            got = check(x, s, n)
            if dtype == torch.float32 and row is up:
                assert got[2][0, 0] == V - 1 and got[1][0, 0] == 0


def test_select_values_at_the_edges(dev):
    """masked logits, beams that are none, rows without a candidate, NaN and infinities, the smallest and largest values"""
    x, s = case(dev, 3, 6, 4, 5000, torch.float32)
    x[0, :, 100:] = -INF                                         # a grammar's mask
    x[0, 1] = -INF                                               # a beam without a token
    s[1, 2] = -INF
    s[2, :] = -INF                                               # nothing to select
    x[3, 0, 17] = NAN                                            # log-softmax of this beam is NaN
    x[3, 1, 18] = INF
    s[3, 3] = NAN
    x[4] = -INF
    x[4, 2, 4999] = 3.0                                          # one candidate
    x[5, 0] = torch.finfo(torch.float32).min                     # masks of the type's lowest value
    x[5, 0, 7] = 0.0
    x[5, 1] = torch.finfo(torch.float32).min
    for n in (3, 40):
        got = check(x, s, n)
        assert (got[1][2] == -1).all() and (got[1][3] == 2).all()
        assert (got[0][4, 1:] == -INF).all() and got[2][4, 0] == 4999
    xb = x.to(torch.bfloat16)
    check(xb, s, 5)
    z = torch.zeros((1, 2, 300), device=dev)
    z[0, 0, ::2] = -0.0                                          # both zeros are equal
    got = check(z, torch.zeros((1, 2), device=dev), 9)
    assert got[2][0].tolist() == list(range(9))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_select_strides(dev, dtype):
    """padded vocabularies, rows that start at any element, beams in another order, a broadcast beam"""
    x, s = case(dev, 8, 3, 4, 5003, dtype)
    for lo, hi in ((0, 5000), (1, 5003), (3, 4098), (7, 8)):
        v = x[:, :, lo:hi]
        a, b = check(v, s, 6), check(v.contiguous(), s, 6)
        for p, q in zip(a, b):
            check_tensors_equal("view", p, q)
    check(x.transpose(0, 1), s.T.contiguous(), 6)
    check(x[:, :1].expand(3, 4, 5003), s, 6)
    check(x[::2, 1::2], s[::2, 1::2].contiguous(), 6)


def test_select_is_repeatable_and_runs_in_graphs(dev):
    import qwen_tailor_amd as qt
    x, s = case(dev, 9, 4, 4, 100000, torch.bfloat16)
    y, _ = case(dev, 10, 4, 4, 100000, torch.bfloat16)
    want, other = qt.batch_beam.select(x, s, 8), qt.batch_beam.select(y, s, 8)
    buf = x.clone()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qt.batch_beam.select(buf, s, 8)
        side.synchronize()
        with torch.cuda.graph(g, stream=side):
            out = qt.batch_beam.select(buf, s, 8)
    for src, ref in ((x, want), (y, other), (x, want), (y, other)):
        buf.copy_(src)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        again = qt.batch_beam.select(src, s, 8)
        for a, b, c in zip(out, ref, again):
            check_tensors_equal("replay", a, b)
            check_tensors_equal("eager", c, b)
    assert qt.batch_beam.select(x[:0], s[:0], 8)[0].shape == (0, 8)


# ---- reordering -----------------------------------------------------------------------------------------------------------

class PoolSet:
    def __init__(self, gen, n_gdn, n_kv, slots, Lmax, dev):
        r = lambda shape, dt: torch.empty(shape, dtype=dt, device=dev).normal_(generator=gen)  # noqa: E731
        self.conv = [r((slots * 2, 3, CD), BF16) for _ in range(n_gdn)]
        self.ssm = [r((slots, 16, 128, 128), torch.float32) for _ in range(n_gdn)]
        self.K = [r((slots, 2, Lmax, 256), BF16) for _ in range(n_kv)]
        self.V = [r((slots, 2, Lmax, 256), BF16) for _ in range(n_kv)]


REORDER = [(1, 1, 1, 1), (1, 2, 1, 1), (1, 4, 3, 1), (3, 3, 2, 2), (2, 8, 1, 1), (2, 9, 1, 1), (1, 16, 1, 1), (1, 17, 1, 1), (1, 32, 1, 1), (2, 4, 0, 1), (2, 4, 1, 0), (1, 2, 50, 1), (1, 2, 1, 50)]


@pytest.mark.parametrize("G,W,n_gdn,n_kv", REORDER)
def test_reorder(dev, G, W, n_gdn, n_kv):
    """any map of beams to beams, rotations and swaps among them; K / V rows of the range only; the conv buffer that the next step reads"""
    import qwen_tailor_amd as qt
    rng = np.random.default_rng(G * W)
    gen = torch.Generator(dev).manual_seed(W)
    Lmax = 37
    P = PoolSet(gen, n_gdn, n_kv, G * W + 2, Lmax, dev)
    slots = rng.permutation(G * W + 2)[:G * W].reshape(G, W).astype(np.int32)
    maps = [rng.integers(0, W, (G, W)), np.tile(np.roll(np.arange(W), 1), (G, 1)), np.tile(np.arange(W)[::-1], (G, 1)), np.zeros((G, W), int), np.tile(np.arange(W), (G, 1))]
    i = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    for m in maps:
        m = m.astype(np.int32)
        if W > 2:
            m[0, 1] = -1                                         # stays
            m[0, 2] = W + 3                                      # is none: stays
        start, pos = rng.integers(0, Lmax, G), rng.integers(0, Lmax + 1, G)
        want = {k: [t.clone() for t in getattr(P, k)] for k in ("conv", "ssm", "K", "V")}
        for g in range(G):
            for w in range(W):
                p = int(m[g, w])
                if not 0 <= p < W:
                    continue
                d, f, a, b = int(slots[g, w]), int(slots[g, p]), int(start[g]), int(pos[g])
                for l in range(n_gdn):
                    want["ssm"][l][d] = P.ssm[l][f]
                    want["conv"][l][2 * d + b % 2] = P.conv[l][2 * f + b % 2]
                for l in range(n_kv):
                    want["K"][l][d, :, a:b], want["V"][l][d, :, a:b] = P.K[l][f, :, a:b], P.V[l][f, :, a:b]
        qt.batch_beam.reorder(P, i(slots), i(m), i(start), i(pos))
        for k in want:
            for a, b in zip(getattr(P, k), want[k]):
                check_tensors_equal(k, a, b)


def test_reorder_stays_within_the_pools(dev):
    """slots that are none, ranges beyond the pool, several padding beams in the trash slot"""
    import qwen_tailor_amd as qt
    gen = torch.Generator(dev).manual_seed(5)
    P = PoolSet(gen, 1, 1, 5, 10, dev)
    Q = {k: [t.clone() for t in getattr(P, k)] for k in ("conv", "ssm", "K", "V")}
    i = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    qt.batch_beam.reorder(P, i([[0, 1, 4, 4], [2, -1, 9, 4]]), i([[1, 1, 2, 3], [1, 0, 0, -1]]), i([-3, 5]), i([99, 3]))
    Q["ssm"][0][0], Q["conv"][0][1] = Q["ssm"][0][1].clone(), Q["conv"][0][3].clone()
    Q["K"][0][0], Q["V"][0][0] = Q["K"][0][1].clone(), Q["V"][0][1].clone()
    for k in Q:
        check_tensors_equal(k, getattr(P, k)[0], Q[k][0])


def test_a_beam_search_step(dev):
    """select and reorder as a program calls them: after them every beam decodes as its parent would have"""
    import qwen_tailor_amd as qt
    gen = torch.Generator(dev).manual_seed(21)
    G, W, n = 2, 4, 60
    P = PoolSet(gen, 1, 1, G * W + 1, 80, dev)
    r = lambda *s: torch.empty(s, dtype=BF16, device=dev).normal_(generator=gen)  # noqa: E731
    slots = torch.randperm(G * W, generator=gen, device=dev).to(torch.int32).reshape(G, W)
    start, pos = torch.tensor([50, 0], dtype=torch.int32, device=dev), torch.tensor([n, n + 3], dtype=torch.int32, device=dev)
    for t in P.K + P.V:                                          # a common prompt
        t[slots[0].long(), :, :50] = t[int(slots[0, 0]), :, :50].clone()
    logits, scores = r(G, W, 5000), torch.zeros((G, W), device=dev)
    _, parents, _ = qt.batch_beam.select(logits, scores, W)
    proj, qkv, ones = r(G * W, PW), r(G * W, 5120), torch.ones(256, dtype=BF16, device=dev)
    cw, A, dt = r(CD, 4), torch.rand(16, device=dev), torch.zeros(16, device=dev)
    at = pos.repeat_interleave(W)
    from_slots = slots.long().gather(1, parents.long()).to(torch.int32)
    want = []
    for g in range(G):
        for w in range(W):                                       # one at a time on copies: several beams continue from one
            K, V, S, C = P.K[0].clone(), P.V[0].clone(), P.ssm[0].clone(), P.conv[0].clone()
            s, p, row = from_slots[g, w][None], at[g * W + w][None], slice(g * W + w, g * W + w + 1)
            want.append((qt.batch.deltanet_b(proj[row], C, cw, A, dt, S, s, p), qt.batch.attn_layer_b(qkv[row], ones, ones, K, V, s, p)))
    qt.batch_beam.reorder(P, slots, parents, start, pos)
    for g in range(G):
        for w in range(W):
            s, p, row = slots[g, w][None], at[g * W + w][None], slice(g * W + w, g * W + w + 1)
            check_tensors_equal("y", qt.batch.deltanet_b(proj[row], P.conv[0], cw, A, dt, P.ssm[0], s, p), want[g * W + w][0])
            check_tensors_equal("o", qt.batch.attn_layer_b(qkv[row], ones, ones, P.K[0], P.V[0], s, p), want[g * W + w][1])


def test_refusals(dev):
    import qwen_tailor_amd as qt
    z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device=dev)  # noqa: E731
    i = lambda *s: z(*s, dt=torch.int32)  # noqa: E731
    sel = qt.batch_beam.select
    for x, s, n, err in ((z(2, 3), z(2, 3), 1, ValueError), (z(2, 3, 4, dt=torch.float64), z(2, 3), 1, TypeError), (z(2, 3, 4), z(2, 4), 1, ValueError), (z(2, 3, 4), z(2, 3), 0, ValueError),
                         (z(2, 3, 4), z(2, 3), 65, ValueError), (z(2, 65, 4), z(2, 65), 1, ValueError), (z(2, 3, 0), z(2, 3), 1, ValueError),
                         (z(2, 3, 8)[:, :, ::2], z(2, 3), 1, ValueError), (z(2000, 64, 1), z(2000, 64), 1, ValueError), (z(2, 3, 4), z(2, 3, dt=torch.float16), 1, TypeError),
                         (z(2, 3, 4), z(2, 3), 1.5, TypeError)):
        with pytest.raises(err):
            sel(x, s, n)
    P = qt.batch.Pools(qt.model.Cfg(layers=4), 4, 20, device=dev)
    good = dict(slots=i(1, 4), parents=i(1, 4), start=i(1), pos=i(1))
    for key, value, err in (("slots", i(4), ValueError), ("parents", i(1, 3), ValueError), ("start", i(2), ValueError), ("pos", z(1), TypeError)):
        with pytest.raises(err):
            qt.batch_beam.reorder(P, *{**good, key: value}.values())
    with pytest.raises(ValueError):
        qt.batch_beam.reorder(P, i(1, 33), i(1, 33), i(1), i(1))
    P.K[0] = P.K[0][:, :, :10]
    with pytest.raises(ValueError):
        qt.batch_beam.reorder(P, *good.values())
    P.K, P.V, P.ssm, P.conv = [], [], [], []
    with pytest.raises(ValueError):
        qt.batch_beam.reorder(P, *good.values())
