"""The scratch memory that the operators keep for a stream, under batches that grow."""
import numpy as np
import pytest
import torch

from tests.test_tree_gpu import layer_case, PoolSet
from tests.util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


def held_after(dev, calls):
    """device memory that stays allocated once the calls have been made, on a stream of their own, and their results are gone"""
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().synchronize()
        before = torch.cuda.memory_allocated(dev)
        for call in calls:
            call()
        torch.cuda.current_stream().synchronize()
        return torch.cuda.memory_allocated(dev) - before


@pytest.mark.parametrize("layer", [False, True])
def test_tree_attention_of_a_growing_batch(dev, layer):
    """one buffer for a stream, at most half as large again as the largest call needs: none of those that were outgrown"""
    import qwen_tailor_amd as qt
    gen, M, most = torch.Generator(dev).manual_seed(1), 64, 12
    P = PoolSet(gen, 0, 1, most + 1, 100, dev)
    cases = [layer_case(gen, B, B, M, 100, dev) for B in range(1, most + 1)]
    heads = lambda x, a, n: x[:, a:a + 256 * n].reshape(-1, n, 256).contiguous()  # noqa: E731

    def call(c):
        _, qkv, _, qn, kn, slots, pos, parents = c
        if layer:
            return qt.batch_tree.attn_layer_bt(qkv, qn, kn, P.K[0], P.V[0], slots, pos, parents)
        return qt.batch_tree.attn_bt(heads(qkv, 0, 8), heads(qkv, 4096, 2), heads(qkv, 4608, 2), P.K[0], P.V[0], slots, pos, parents)

    call(cases[0])                                               # (the rotary table is built by the first call on a device)
    need = qt._lib.lib().qt_gqa_tree_layer_workspace_bytes(most, M) if layer else qt._lib.lib().qt_gqa_tree_workspace_bytes(most, M)
    assert held_after(dev, [lambda c=c: call(c) for c in cases]) <= 1.5 * need + (2 << 20)


def test_selection_of_a_growing_batch(dev):
    import qwen_tailor_amd as qt
    x = torch.zeros((64, 16, 9000), dtype=BF16, device=dev)
    s = torch.zeros((64, 16), device=dev)
    lib = qt._lib.lib()
    need = max(lib.qt_beam_select_workspace_bytes(G, 16, 9000, 64, 2) for G in range(1, 65))
    assert held_after(dev, [lambda G=G: qt.batch_beam.select(x[:G], s[:G], 64) for G in range(1, 65)]) <= 1.5 * max(need, 1 << 20) + (2 << 20)


def test_results_and_graphs_across_the_growth(dev):
    """a call's outputs do not change when the scratch grows between two of them, nor do a graph's that was captured before"""
    import qwen_tailor_amd as qt
    gen = torch.Generator(dev).manual_seed(3)
    cases = [(layer_case(gen, B, B, M, 90, dev), PoolSet(gen, 0, 1, B + 1, 90, dev)) for B, M in ((1, 7), (3, 20), (9, 64), (2, 40))]
    run = lambda c, P: qt.batch_tree.attn_layer_bt(c[1], c[3], c[4], P.K[0], P.V[0], c[5], c[6], c[7])  # noqa: E731
    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        run(*cases[0])
        side.synchronize()
        with torch.cuda.graph(g, stream=side):
            out = run(*cases[1])
        for _ in range(3):
            got = [run(*c) for c in cases]
            out.zero_()
            g.replay()
            filler = torch.full((64 << 20,), 255, dtype=torch.uint8, device=dev)       # (what was given back is used by something else)
            side.synchronize()
            for a, b in zip(got, want):
                check_tensors_equal("eager", a, b)
            check_tensors_equal("replay", out, want[1])
            del filler
