"""Drafted trees (batch_tree) where they can go wrong without the random cases of test_tree_gpu.py showing it: outputs in which opposite values cancel,
paths that claim more tokens than there are."""
import numpy as np
import pytest
import torch

from tests.test_tree_gpu import PoolSet, attn_run, params, trees, way
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
