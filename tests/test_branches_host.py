"""What the operators of several branches (batch_tree, batch_beam) refuse, and their plans, without a GPU."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    import qwen_tailor_amd as qt
    x = torch.zeros((2, 8224), dtype=torch.bfloat16)
    i = torch.zeros((2, 1), dtype=torch.int32)
    P = qt.batch.Pools(qt.model.Cfg(layers=4), 2, 16, device="cpu")
    for call in (lambda: qt.batch_tree.deltanet_bt(x, x, x, x, x, x, i, i, i), lambda: qt.batch_tree.attn_bt(x, x, x, x, x, i, i, i),
                 lambda: qt.batch_tree.attn_layer_bt(x, x, x, x, x, i, i, i), lambda: qt.batch_tree.commit(P, [x] * 3, [x] * 3, [x] * 3, [x] * 3, i, i, i, i),
                 lambda: qt.batch_beam.select(x, x, 1), lambda: qt.batch_beam.reorder(P, i, i, i, i)):
        with pytest.raises(TypeError):
            call()


def test_error_codes():
    import qwen_tailor_amd as qt
    lib = qt._lib.lib()
    z, p, odd = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(8)
    step = lambda *a: lib.qt_gdn_tree_step(*a)  # noqa: E731
    assert step(p, p, p, p, p, p, p, p, z, p, p, 1, 4, 1, z) == -3
    assert step(p, p, p, p, p, p, p, p, p, z, p, 1, 65, 1, z) == -4 and step(p, p, p, p, p, p, p, p, p, z, p, 1, 0, 1, z) == -4
    assert step(p, p, p, p, p, p, p, p, p, z, p, -1, 4, 1, z) == -1 and step(p, p, p, p, p, p, p, p, p, z, p, 1, 4, 0, z) == -1
    assert step(p, p, p, p, p, p, p, p, p, odd, p, 1, 4, 1, z) == -2
    assert step(odd, p, p, p, p, p, p, p, p, z, p, 1, 4, 1, z) == -2
    assert step(p, p, p, p, p, p, p, p, p, z, p, 0, 4, 1, z) == 0                       # nothing to do: no launch
    need = lib.qt_gqa_tree_workspace_bytes(2, 16)
    assert lib.qt_gqa_tree_workspace_bytes(1025, 4) == -1 and lib.qt_gqa_tree_workspace_bytes(1, 65) == -1 and lib.qt_gqa_tree_layer_workspace_bytes(1, 0) == -1
    assert lib.qt_gqa_tree_layer_workspace_bytes(2, 16) >= need + 2 * 16 * 12 * 256 * 2
    attn = lambda ws, n, B, M, L, S: lib.qt_gqa_tree_attn(p, p, p, p, p, p, p, p, p, ws, n, B, M, L, S, z)  # noqa: E731
    assert attn(z, need, 2, 16, 64, 3) == -3 and attn(p, need - 1, 2, 16, 64, 3) == -6 and attn(odd, need, 2, 16, 64, 3) == -2
    assert attn(p, 1 << 40, 2, 65, 64, 3) == -4 and attn(p, 1 << 40, 1025, 4, 64, 3) == -4 and attn(p, 1 << 40, 2, 16, 0, 3) == -1
    assert attn(p, 1 << 40, 0, 16, 64, 3) == 0
    layer = lambda t, n, M: lib.qt_gqa_tree_layer(p, p, p, t, n, p, p, p, p, p, p, p, 1 << 40, 1, M, 64, 3, 1e-6, z)  # noqa: E731
    assert layer(z, 64, 4) == -1 and layer(p, -1, 4) == -1 and layer(p, 64, 65) == -4
    assert lib.qt_gqa_tree_layer(p, z, p, p, 64, p, p, p, p, p, p, p, 1 << 40, 1, 4, 64, 3, 1e-6, z) == -3


def test_error_codes_of_tables():
    import qwen_tailor_amd as qt
    lib = qt._lib.lib()
    z, p = ctypes.c_void_p(0), ctypes.c_void_p(16)
    t, bad, null = (ctypes.c_void_p * 1)(16), (ctypes.c_void_p * 1)(8), (ctypes.c_void_p * 1)(0)
    commit = lambda ssm=t, kv=t, n=1, B=1, M=4, D=4, L=64, path=p: lib.qt_tree_commit(t, t, t, t, t, ssm, n, kv, n, p, p, path, p, B, M, D, 3, L, z)  # noqa: E731
    assert commit(ssm=bad) == -2 and commit(kv=bad) == -2 and commit(ssm=null) == -3 and commit(kv=null) == -3 and commit(path=z) == -3
    assert commit(M=65) == -4 and commit(D=65) == -4 and commit(D=0) == -4 and commit(L=0) == -1 and commit(n=-1) == -1
    assert commit(B=0) == 0
    reorder = lambda ssm=t, kv=t, n=1, G=1, W=4, L=64: lib.qt_beam_reorder(ssm, t, n, kv, n, p, p, p, p, G, W, 3, L, z)  # noqa: E731
    assert reorder(ssm=bad) == -2 and reorder(kv=bad) == -2 and reorder(ssm=null) == -3 and reorder(W=33) == -4 and reorder(W=0) == -4
    assert reorder(L=0) == -1 and reorder(G=-1) == -1 and reorder(G=0) == 0
    ws = lib.qt_beam_select_workspace_bytes
    assert ws(1, 65, 10, 1, 2) == -1 and ws(1, 1, 10, 65, 2) == -1 and ws(1, 1, 10, 0, 2) == -1 and ws(1, 1, 0, 1, 2) == -1 and ws(1, 1, 10, 1, 3) == -1
    assert ws(2000, 64, 10, 1, 2) == -1 and ws(0, 4, 10, 1, 2) == 0 and ws(1, 1, 248320, 8, 2) > 0
    select = lambda x=p, d=0, w=p, n=1 << 40, G=1, W=2, V=100, k=4: lib.qt_beam_select(x, d, 200, 100, p, p, p, p, w, n, G, W, V, k, z)  # noqa: E731
    assert select(x=z) == -3 and select(w=z) == -3 and select(d=3) == -4 and select(W=65) == -1 and select(k=0) == -1
    assert select(x=ctypes.c_void_p(17)) == -2 and select(x=ctypes.c_void_p(18), d=2) == -2 and select(n=16) == -6 and select(G=0) == 0
