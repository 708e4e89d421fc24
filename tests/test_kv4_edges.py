"""Operators of the 4-bit key/value cache at their edges: captured steps beside growing workspaces, values that a token must
not see, scores at the end of the f32 range, aliased buffers, sizes at the end of the index range.

The definitions and the bound on a score's error (ds) are those of test_kv4.py. A slot that a token does not see has no
part in its output, whatever its bits: the definition here sums over the visible slots alone.
"""
import numpy as np
import pytest

import sparrow_b200.kernels as K
from test_kv4 import _random_cache, _torch, _up


# ------------------------------------------------- captured steps

def _replay_beside_a_larger_call(step, outs, larger):
    """Capture `step` behind an eager run of it, make a larger call, fill whatever memory that gave back, replay: the outputs
    are the eager run's, bit for bit, and the memory that others hold by then is as they left it."""
    torch = _torch()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    step(st)
    K.sync(st)
    ref = [x.clone() for x in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step(st)
    larger(st)
    K.sync(st)
    torch.cuda.empty_cache()
    others = [torch.full((n,), 0x5A, dtype=torch.uint8, device="cuda") for n in [1 << 12, 1 << 16, 1 << 20] * 20 + [24 << 20] * 40]
    for _ in range(2):
        for x in outs:
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, r in zip(outs, ref):
            assert torch.equal(x.view(torch.uint8), r.view(torch.uint8))
    assert all((x == 0x5A).all() for x in others)
    K.sync(st)
    del graph


@pytest.mark.gpu
@pytest.mark.parametrize("d,group", [(64, 2), (128, 4), (256, 3)])
@pytest.mark.parametrize("weights", [False, True])
def test_captured_attention_beside_a_larger_call(kernels, d, group, weights):
    """A decode step is captured; then a prompt's call needs more of every workspace."""
    torch = _torch()
    K.sync()
    K.shutdown()  # the workspaces of earlier calls go
    K.init(0)
    rng = np.random.default_rng(d)
    n_seq, n_kv, cap = 2, 4, 5000
    _, cache = _random_cache(rng, n_seq, n_kv, cap, d, [cap] * n_seq, bad=False)
    length = _up(np.array([cap, 777], np.int32))

    def make(m):
        q = _up(rng.standard_normal((n_seq * m, n_kv * group * d)).astype(np.float32))
        out = torch.empty_like(q)
        w = torch.zeros((n_seq, n_kv, cap), device="cuda") if weights else None
        return [out] + ([w] if weights else []), lambda st: K.kv4_attn_dev(cache, q, length, out, m, n_kv * group, 0.1,
                                                                           w_out=w, stream=st)

    outs, step = make(1)
    _replay_beside_a_larger_call(step, outs, make(60)[1])


@pytest.mark.gpu
def test_captured_gemm_beside_a_larger_call(kernels):
    """The other operators' workspaces are kept by the same rule."""
    torch = _torch()
    K.sync()
    K.shutdown()
    K.init(0)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    n, k = 256, 512
    w = (torch.randn((n, k), generator=g, device="cuda") * 0.05).to(torch.bfloat16)

    def make(m):
        x, y = torch.randn((m, k), generator=g, device="cuda"), torch.empty((m, n), device="cuda")

        def step(st):
            for _ in range(2):  # an even number: the calls use two flag words in turn
                K.gemm_nt_bf16_dev(x, w, y, m, n, k, stream=st)
        return [y], step

    outs, step = make(200)
    _replay_beside_a_larger_call(step, outs, make(4000)[1])
