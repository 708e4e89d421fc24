"""Operators of the 4-bit key/value cache at their edges: captured steps beside growing workspaces, values that a token must
not see, scores at the end of the f32 range, aliased buffers, sizes at the end of the index range.

The definitions and the bound on a score's error (ds) are those of test_kv4.py. A slot that a token does not see has no
part in its output, whatever its bits: the definition here sums over the visible slots alone.
"""
import ctypes

import numpy as np
import pytest

import sparrow_b200.kernels as K
from sparrow_b200._lib import VmlmError
from test_kv4 import EPS, _cache, _random_cache, _rc, _tables, _torch, _up, np_attention, np_keep, np_norm_rope, np_values


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


# ------------------------------------------------- the end of the index range

def test_attention_refuses_sizes_whose_product_wraps():
    """n_seq * m * n_q is 2^65: below 2^31 in 64 bits."""
    c = _cache(n_seq=1 << 25, n_kv=1)
    rc, msg = _rc("vmlm_kv4_attn_dev", ctypes.byref(c), 4096, 64 << 15, 4096, 1 << 28, 64 << 15, 1 << 25, 1 << 15, 0.125, None,
                  None, None)
    assert rc == 2 and "n_seq * m * n_q" in msg


def test_refuses_slots_that_a_step_would_carry_past_32_bits():
    """A kernel's walk steps by a tile or by a block of threads from slots below cap, and by units of 32 columns over what an
    eviction keeps."""
    T = 1 << 40

    def cache(**kw):
        return _cache(**{**dict(k=T, v=2 * T, ks=3 * T, vs=4 * T, n_kv=1), **kw})

    for cap in ((1 << 31) - 1, (1 << 31) - 8191):
        c = cache(cap=cap)
        rc, msg = _rc("vmlm_kv4_attn_dev", ctypes.byref(c), 4096, 64, 4096, 1 << 28, 64, 1, 1, 0.125, None, None, None)
        assert rc == 2 and "cap" in msg
        assert _rc("vmlm_kv4_read_dev", ctypes.byref(c), 4096, 4096, 1, 4096, 4096, None)[0] == 2
    assert _rc("vmlm_kv4_read_dev", ctypes.byref(cache()), 4096, 4096, (1 << 31) - 1, 4096, 4096, None)[0] == 2
    for d, keep in ((64, 1 << 30), (128, 1 << 29), (256, 1 << 28)):
        s, t = cache(cap=keep + 8, d=d), cache(k=5 * T, v=6 * T, ks=7 * T, vs=8 * T, cap=keep, d=d)
        rc, msg = _rc("vmlm_kv4_evict_dev", ctypes.byref(s), ctypes.byref(t), 9 * T, 10 * T, keep, 0, 0, 11 * T, None, 12 * T, None)
        assert rc == 2 and "keep" in msg


# ------------------------------------------------- aliased buffers

def test_eviction_refuses_outputs_that_overlap():
    """One CTA a sequence writes its new length, perhaps before another head's has read the old one; no output may lie on an
    input or on another output."""
    n, M = 1 << 12, 1 << 20  # every buffer below has at most 4096 bytes: n_seq 2, n_kv 2, 8 slots of 64, 4 kept

    def evict(**at):
        p = dict(k=1, v=2, ks=3, vs=4, dk=5, dv=6, dks=7, dvs=8, w=9, length=10, idx=11, w_out=12, len_out=13)
        p = {x: M + n * y for x, y in p.items()}
        for x, y in at.items():
            p[x] = p[y] if isinstance(y, str) else p[y[0]] + y[1]
        s = _cache(k=p["k"], v=p["v"], ks=p["ks"], vs=p["vs"], n_seq=2)
        t = _cache(k=p["dk"], v=p["dv"], ks=p["dks"], vs=p["dvs"], n_seq=2)
        return _rc("vmlm_kv4_evict_dev", ctypes.byref(s), ctypes.byref(t), p["w"], p["length"], 4, 1, 2, p["idx"], p["w_out"],
                   p["len_out"], None)

    rc, msg = evict(len_out="length")
    assert rc == 1 and "an output overlaps an input" in msg
    assert evict(len_out=("length", 4))[0] == 1 and evict(w_out="w")[0] == 1 and evict(w_out=("w", 120))[0] == 1
    assert evict(idx="w")[0] == 1 and evict(idx="length")[0] == 1 and evict(dks="vs")[0] == 1 and evict(dv="w")[0] == 1
    rc, msg = evict(idx="w_out")
    assert rc == 1 and "two outputs overlap" in msg
    assert evict(len_out=("idx", 60))[0] == 1 and evict(dk="dv")[0] == 1


def test_attention_refuses_an_output_over_its_queries():
    P = 1 << 20

    def attn(q, ldq, out, ldo, m=1, w_in=None, w_out=None):
        c = _cache(k=1 << 24, v=2 << 24, ks=3 << 24, vs=4 << 24, n_seq=3)
        return _rc("vmlm_kv4_attn_dev", ctypes.byref(c), q, ldq, 1 << 28, out, ldo, m, 4, 0.125, w_in, w_out, None)

    rc, msg = attn(P, 256, P, 256)
    assert rc == 1 and "out overlaps q" in msg
    assert attn(P, 256, P + 2 * 256 * 4 + 255 * 4, 256)[0] == 1      # its last value
    assert attn(P + 255 * 4, 256, P, 256)[0] == 1
    assert attn(P, 600, P + 255 * 4, 600)[0] == 1 and attn(P, 600, P + 345 * 4, 600)[0] == 1  # rows between rows, one too far
    assert attn(P, 300, P + 256 * 4, 400)[0] == 1                    # other strides over the same span
    rc, msg = attn(P, 256, 2 * P, 256, w_in=3 * P, w_out=3 * P + 64)
    assert rc == 1 and "w_in and w_out overlap" in msg


def test_norm_and_append_refuse_partly_shared_rows():
    P = 1 << 20

    def norm(q=P, ldq=128, k=2 * P, ldk=128, qo=3 * P, ldqo=128, ko=4 * P, ldko=128):
        return _rc("vmlm_qk_norm_rope_dev", q, ldq, k, ldk, None, None, 1e-5, None, qo, ldqo, ko, ldko, 5, 2, 2, 64, None)

    rc, msg = norm(qo=P, ldqo=256)
    assert rc == 1 and "qo and q overlap" in msg
    assert norm(qo=P + 4)[0] == 1 and norm(ko=2 * P - 4)[0] == 1 and norm(ko=2 * P + 512)[0] == 1
    rc, msg = norm(qo=2 * P)
    assert rc == 1 and "queries and keys overlap" in msg
    assert norm(ko=P)[0] == 1 and norm(qo=4 * P + 4 * 512)[0] == 1

    def app(qo, ldqo):
        c = _cache(k=1 << 24, v=2 << 24, ks=3 << 24, vs=4 << 24, n_seq=3)
        return _rc("vmlm_kv4_append_dev", ctypes.byref(c), P, 512, qo, ldqo, 2, P + 512, 512, P + 1024, 512, None, None, 1e-5,
                   None, 1 << 28, 1, None)

    assert app(P, 300)[0] == 1 and app(P + 4, 512)[0] == 1 and app(P + 512, 512)[0] == 1 and app(P + 1024 + 508, 512)[0] == 1


@pytest.mark.gpu
def test_buffers_between_each_other(kernels):
    """What may share memory: queries and outputs as slices of one matrix, rows in place, histories in place, one row with any
    stride."""
    torch = _torch()
    rng = np.random.default_rng(1)
    n_seq, n_kv, group, cap, d, m = 2, 2, 2, 300, 64, 3
    width = n_kv * group * d
    _, cache = _random_cache(rng, n_seq, n_kv, cap, d, [cap] * n_seq, bad=False)
    lens = _up(np.array([cap, 40], np.int32))
    both = _up(rng.standard_normal((n_seq * m, 2 * width)).astype(np.float32))
    q = both[:, :width].clone()
    st = torch.cuda.current_stream()
    ref = torch.empty_like(q)
    K.kv4_attn_dev(cache, q, lens, ref, m, n_kv * group, 0.1, stream=st)
    K.kv4_attn_dev(cache, both[:, :width], lens, both[:, width:], m, n_kv * group, 0.1, stream=st)
    assert torch.equal(both[:, width:], ref) and torch.equal(both[:, :width], q)
    x = both.clone()
    y, g = torch.empty_like(x), _up(rng.uniform(0.5, 1.5, d).astype(np.float32))
    K.qk_norm_rope_dev(x[:, :width], x[:, width:], g, g, EPS, None, y[:, :width], y[:, width:], n_seq * m, n_kv * group,
                       n_kv * group, d, stream=st)
    K.qk_norm_rope_dev(x[:, :width], x[:, width:], g, g, EPS, None, x[:, :width], x[:, width:], n_seq * m, n_kv * group,
                       n_kv * group, d, stream=st)
    K.qk_norm_rope_dev(x[:1, :d], None, None, None, EPS, None, x[:1, :d], None, 1, 1, 0, d, stream=st)
    assert torch.equal(x, y)
    K.sync(st)
    idx, w = torch.empty((n_seq, n_kv, 8), dtype=torch.int32, device="cuda"), torch.ones((n_seq, n_kv, cap), device="cuda")
    _, small = _random_cache(rng, n_seq, n_kv, 8, d, [8] * n_seq, bad=False)
    with pytest.raises(VmlmError):
        K.kv4_evict_dev(cache, small, w, lens, 8, 0, 0, idx, None, lens, stream=st)
    K.kv4_evict_dev(cache, small, w, lens, 8, 0, 0, idx, None, torch.empty_like(lens), stream=st)
    K.sync(st)


# ------------------------------------------------- what a token does not see

def _visible_attention(q, k, v, seen, scale):
    """q [rows, d], k, v [n, d] f64, seen [rows]: output and weights [rows, n], each row from its visible slots alone."""
    out, p = np.zeros((len(q), v.shape[1])), np.zeros((len(q), len(k)))
    for r, n in enumerate(seen):
        if n <= 0:
            continue
        z = scale * (k[:n] @ q[r])
        e = np.exp(z - z.max())
        p[r, :n] = e / e.sum()
        with np.errstate(invalid="ignore"):
            out[r] = p[r, :n] @ v[:n]
    return out, p


@pytest.mark.gpu
@pytest.mark.parametrize("d,group,m,n_seq,n_kv,cap", [
    (64, 1, 2, 2, 2, 100), (64, 1, 33, 2, 3, 400), (64, 3, 5, 3, 2, 900), (64, 1, 130, 1, 2, 300), (64, 5, 2, 2, 1, 4000),
    (128, 1, 3, 2, 2, 70), (128, 4, 5, 3, 2, 700), (128, 2, 40, 1, 2, 3000), (256, 1, 4, 2, 2, 65), (256, 2, 9, 2, 1, 500),
    (256, 16, 5, 8, 2, 3000), (256, 4, 8, 8, 2, 3000), (256, 1, 45, 8, 2, 3000)])
@pytest.mark.parametrize("weights", [False, True])
def test_attention_hidden_values_that_are_not_finite(kernels, d, group, m, n_seq, n_kv, cap, weights):
    """NaN and infinite values, and codes whose value overflows a half, in the newest tokens: a token that does not see
    them has a finite output; one that does has them in their columns and nowhere else."""
    torch = _torch()
    rng = np.random.default_rng(d + m + cap)
    lens = np.array([max(m, cap - 13 * b) for b in range(n_seq)], np.int32)
    host, _ = _random_cache(rng, n_seq, n_kv, cap, d, lens)
    (kc, ks, kb), (vc, vs, vb) = host
    for b, n in enumerate(lens):
        vs[b, 0, n - 1, 0] = np.nan                 # the last token, its first 32 columns
        vb[b, :, n - 1, d // 32 - 1] = -np.inf      # and its last 32
        vs[b, n_kv - 1, n - m + 1, 1] = 4000        # the second token: codes from 1 on are infinite
        vb[b, n_kv - 1, n - m + 1, 1] = 0
        if n > m + 3:
            vs[b, 0, 1, 1] = np.nan                 # a slot that every token sees
    cache = K.Kv4Cache(_up(kc[..., 0::2] | (kc[..., 1::2] << 4)), _up(vc[..., 0::2] | (vc[..., 1::2] << 4)),
                       _up(np.stack((ks, kb), -1)), _up(np.stack((vs, vb), -1)))
    n_q, scale = n_kv * group, 1 / np.sqrt(d)
    q = rng.standard_normal((n_seq * m, n_q * d)).astype(np.float32)
    out = torch.full((n_seq * m, n_q * d), 7.0, device="cuda")
    w_out = torch.full((n_seq, n_kv, cap), 7.0, device="cuda") if weights else None
    st = torch.cuda.current_stream()
    K.kv4_attn_dev(cache, _up(q), _up(lens), out, m, n_q, scale, w_out=w_out, stream=st)
    K.sync(st)
    got = out.cpu().numpy().reshape(n_seq, m, n_q, d)
    q = q.reshape(n_seq, m, n_q, d).astype(np.float64)
    for b, n in enumerate(lens):
        seen = np.repeat(n - (m - 1 - np.arange(m)), group)
        for h in range(n_kv):
            k = np_values(kc[b, h, :n], ks[b, h, :n], kb[b, h, :n])
            with np.errstate(over="ignore", invalid="ignore"):
                v = np_values(vc[b, h, :n], vs[b, h, :n], vb[b, h, :n])
            rows = q[b, :, h * group:(h + 1) * group].reshape(m * group, d)
            ref, p = _visible_attention(rows, k, v, seen, scale)
            _, _, ds = np_attention(rows, k, np.zeros_like(v), seen, scale)
            y = got[b, :, h * group:(h + 1) * group].reshape(m * group, d)
            assert np.array_equal(np.isfinite(y), np.isfinite(ref)), (b, h)
            for r in range(m * group):
                x = v[:seen[r]]
                vmax = np.abs(x[np.isfinite(x)]).max()
                ok = np.isfinite(ref[r])
                assert (np.abs(y[r, ok] - ref[r, ok]) <= (2 * ds[r] + 2.0 ** -18) * vmax).all(), (b, h, r)
            if weights:
                tol = ((2 * ds + 2.0 ** -18)[:, None] * p).sum(0) + 2.0 ** -22 * p.sum(0) + 1e-12
                assert (np.abs(w_out[b, h].cpu().numpy()[:n] - p.sum(0)) <= tol).all(), (b, h)


# ------------------------------------------------- scores at the end of the f32 range

#: d, query heads a kv head, sequences, kv heads, slots: one to sixteen rows a warp, items shared by warps and by CTAs, the
#: kernel for many rows of 256
SCORE_CASES = [(64, 1, 1, 2, 50), (64, 12, 1, 1, 6000), (128, 4, 2, 2, 333), (128, 7, 1, 1, 9000), (256, 2, 1, 2, 700),
               (256, 32, 8, 2, 3000)]


def _one_sign(d, group, n_seq, n_kv, n, size, scale):
    """Attention with weights where every key is positive and every query has the sign of `size`, so that all scores have
    it, and one slot of each head is far ahead of the others (by more than a thousandth of the scores). Returns the output
    [n_seq, n_kv, group, d], the weight that was added [n_seq, n_kv, n], and the slot and its values [n_seq, n_kv, d]."""
    torch = _torch()
    rng = np.random.default_rng(d + n)
    host, _ = _random_cache(rng, n_seq, n_kv, n, d, [n] * n_seq)
    (kc, ks, kb), (vc, vs, vb) = host
    ks[:], kb[:] = rng.uniform(0.1, 2.0, ks.shape).astype(np.float16), np.float16(0.5)
    best = rng.integers(0, n - 1, (n_seq, n_kv))
    for b in range(n_seq):
        for h in range(n_kv):
            ks[b, h, best[b, h]] = np.float16(5.0 if size * scale > 0 else 0.0)
    cache = K.Kv4Cache(_up(kc[..., 0::2] | (kc[..., 1::2] << 4)), _up(vc[..., 0::2] | (vc[..., 1::2] << 4)),
                       _up(np.stack((ks, kb), -1)), _up(np.stack((vs, vb), -1)))
    q = (size * rng.uniform(0.5, 1.0, (n_seq, n_kv * group * d))).astype(np.float32)
    out = torch.full((n_seq, n_kv * group * d), 7.0, device="cuda")
    w = torch.full((n_seq, n_kv, n), 7.0, device="cuda")
    st = torch.cuda.current_stream()
    K.kv4_attn_dev(cache, _up(q), _up(np.full(n_seq, n, np.int32)), out, 1, n_kv * group, scale, w_out=w, stream=st)
    K.sync(st)
    v = np_values(vc, vs, vb)
    return (out.cpu().numpy().reshape(n_seq, n_kv, group, d), w.cpu().numpy(), best,
            np.take_along_axis(v, best[..., None, None], 2)[:, :, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("case", SCORE_CASES)
def test_attention_scores_of_minus_infinity(kernels, case):
    """Every score overflows to -inf: nothing is left to weigh, for the output and for the weights alike."""
    out, w, _, _ = _one_sign(*case, size=-3e38, scale=1.0)
    assert (out == 0).all() and (w == 0).all()


def _check_one_slot(case, size, scale):
    """The slot in front has all of the weight: its lead is above 2^-10 of the scores, and ds below 2^-16 of them."""
    d, group = case[:2]
    out, w, best, v = _one_sign(*case, size=size, scale=scale)
    assert (np.abs(out - v[:, :, None]) <= 2.0 ** -18 * np.abs(v).max()).all()
    for b in range(w.shape[0]):
        for h in range(w.shape[1]):
            want = np.zeros(w.shape[2])
            want[best[b, h]] = group
            assert (np.abs(w[b, h] - want) <= 2.0 ** -18 * want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", SCORE_CASES)
@pytest.mark.parametrize("size", [3e3, 1e5, 3e6, 1e8, 1e12, 1e30, -3e5, -1e8])
def test_attention_scores_of_any_size(kernels, case, size):
    """Scores whose neighbours in f32 lie further apart than a weight's room to grow."""
    _check_one_slot(case, size, 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("case", SCORE_CASES)
def test_attention_with_a_scale_that_is_no_number(kernels, case):
    """softmax(NaN) is NaN, in the output and in the weights."""
    out, w, _, _ = _one_sign(*case, size=1.0, scale=float("nan"))
    assert np.isnan(out).all() and np.isnan(w).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", SCORE_CASES)
@pytest.mark.parametrize("size", [-1e28, -1e30, -3e33])
def test_attention_scores_far_below_zero(kernels, case, size):
    """Scores down to -1e37: the largest of them still leads."""
    _check_one_slot(case, size, 0.125)


# ------------------------------------------------- workspaces

@pytest.mark.gpu
def test_workspace_grows_into_what_is_left(kernels):
    """A call that needs a little more workspace than the one before it runs where that fits, although twice the old size
    (what the library asks for, so that growing stays rare) does not."""
    torch = _torch()
    rng = np.random.default_rng(3)
    d, n_seq, n_kv, group, cap = 64, 2, 4, 4, 4000
    m = 512
    _, cache = _random_cache(rng, n_seq, n_kv, cap, d, [cap] * n_seq, bad=False)
    st = torch.cuda.current_stream()
    w = torch.zeros((n_seq, n_kv, cap), device="cuda")
    lens = _up(np.full(n_seq, cap, np.int32))

    def call(m):
        q = torch.ones((n_seq * m, n_kv * group * d), device="cuda")
        out = torch.empty_like(q)
        K.kv4_attn_dev(cache, q, lens, out, m, n_kv * group, 0.1, w_out=w, stream=st)
        K.sync(st)
        return out

    K.sync(st)
    K.shutdown()  # the workspaces of earlier tests go
    K.init(0)
    call(m)  # scores: 2 * 4 * 2048 rows * 4000 slots * 4 bytes = 262 MB
    torch.cuda.empty_cache()
    need = n_seq * n_kv * (m + 64) * group * cap * 4
    free = torch.cuda.mem_get_info()[0]
    old = n_seq * n_kv * m * group * cap * 4
    held = torch.empty(free + old - need - (96 << 20), dtype=torch.uint8, device="cuda")  # all but what is needed and 96 MB
    try:
        out = call(m + 64)
        assert torch.isfinite(out).all()
    finally:
        del held
        torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["bf16", "f32", "attention"])
def test_a_call_that_cannot_grow_leaves_the_workspace(kernels, what):
    """A larger call inside a capture is an error, and calls of the old size go on as before, behind a graph that holds the
    workspace and without one."""
    torch = _torch()
    K.sync()
    K.shutdown()
    K.init(0)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    n, k = 256, 512
    _, cache = _random_cache(np.random.default_rng(1), 2, 4, 600, 64, [600] * 2, bad=False)
    length = _up(np.array([600, 77], np.int32))
    wb = (torch.randn((n, k), generator=g, device="cuda") * 0.05).to(torch.bfloat16)
    wf = wb.float()

    def make(m):
        if what == "attention":
            q = torch.randn((2 * m, 4 * 64), generator=g, device="cuda")
            out, w = torch.empty_like(q), torch.zeros((2, 4, 600), device="cuda")
            return [out, w], lambda st: K.kv4_attn_dev(cache, q, length, out, m, 4, 0.1, w_out=w, stream=st)
        x, y = torch.randn((m, k), generator=g, device="cuda"), torch.empty((m, n), device="cuda")
        if what == "bf16":
            return [y], lambda st: K.gemm_nt_bf16_dev(x, wb, y, m, n, k, stream=st)
        return [y], lambda st: K.gemm_nt_f32_dev(x, wf, y, m, n, k, stream=st)

    cuda = ctypes.CDLL("libcuda.so.1")
    outs, step = make(200)
    _, larger = make(4000)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    step(st)
    K.sync(st)
    ref = [x.clone() for x in outs]
    for held in (False, True):
        if held:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                step(st)
                step(st)
        handle, made = ctypes.c_void_p(st.cuda_stream), ctypes.c_void_p()
        assert cuda.cuStreamBeginCapture_v2(handle, 1) == 0  # of this thread
        with pytest.raises(VmlmError):
            larger(st)
        assert cuda.cuStreamEndCapture(handle, ctypes.byref(made)) == 901 and not made.value  # the capture is void
        torch.cuda.synchronize()
        for _ in range(2):
            for x in outs:
                x.zero_()
            torch.cuda.synchronize()
            step(st)
            K.sync(st)
            assert all(torch.equal(x, r) for x, r in zip(outs, ref))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, r) for x, r in zip(outs, ref))
    del graph


# ------------------------------------------------- idle sequences

@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_append_asks_no_position_of_an_idle_sequence(kernels, d):
    """Positions that follow the lengths, as a decode step has them: -1 for an idle sequence is no error, and one outside
    the table of a sequence in use is one all the same."""
    torch = _torch()
    rng = np.random.default_rng(d)
    n_seq, n_kv, cap = 4, 2, 9
    _, cache = _random_cache(rng, n_seq, n_kv, cap, d, [cap] * n_seq, bad=False)
    x = rng.standard_normal((n_seq, 3 * n_kv * d)).astype(np.float32)
    length = np.array([3, -1, 8, -7], np.int32)
    tc, ts = _tables(cap, d)
    before = cache.k.clone()
    xd, g = _up(x), _up(np.ones(d, np.float32))
    qo = torch.full((n_seq, n_kv * d), 7.0, device="cuda")
    st = torch.cuda.current_stream()

    def append(pos):
        K.kv4_append_dev(cache, xd[:, n_kv * d:2 * n_kv * d], xd[:, 2 * n_kv * d:], _up(length), 1, q=xd[:, :n_kv * d], qo=qo,
                         n_q=n_kv, gq=g, gk=g, eps=EPS, rope=K.Rope(_up(tc), _up(ts), _up(pos)), stream=st)
        K.sync(st)

    append(length)
    got = qo.cpu().numpy()
    ref = np_norm_rope(x[[0, 2], :n_kv * d].reshape(2, n_kv, d), np.ones(d, np.float32), tc[[3, 8]], ts[[3, 8]], False)
    assert np.abs(got[[0, 2]].reshape(ref.shape) - ref).max() < 1e-5 and (got[[1, 3]] == 7).all()
    assert torch.equal(cache.k[[1, 3]], before[[1, 3]]) and not torch.equal(cache.k[0, :, 3], before[0, :, 3])
    with pytest.raises(VmlmError) as e:
        append(np.array([3, -1, 9, -1], np.int32))
    assert e.value.status == 8 and "position" in str(e.value)


# ------------------------------------------------- what is no tensor on the GPU

@pytest.mark.parametrize("bad", [None, np.zeros((1, 64), np.float32), [0.0] * 64, 1.5])
def test_python_says_which_argument_is_no_cuda_tensor(bad):
    from types import SimpleNamespace
    c = SimpleNamespace(n_seq=1, n_kv=1, cap=4, d=64, ref=None)
    for call in (lambda: K.kv4_attn_dev(c, bad, 8, bad, 1, 1, 0.1), lambda: K.kv4_append_dev(c, bad, bad, 8, 1),
                 lambda: K.qk_norm_rope_dev(bad, None, None, None, EPS, None, bad, None, 1, 1, 0, 64)):
        with pytest.raises(ValueError, match="^[qk]: expected a float32 CUDA tensor"):
            call()
    if bad is not None:
        with pytest.raises(ValueError, match="^start: "):
            K.kv4_read_dev(c, bad, 8, 1, 16, 16)
        with pytest.raises(ValueError, match="^w: "):
            K.kv4_evict_dev(c, c, bad, 8, 1, 0, 0, 8, None, 8)


# ------------------------------------------------- eviction from shares that outgrow shared memory

@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["spread", "ties", "late"])
def test_eviction_keys_read_again(kernels, kind):
    """More heads than SMs, so that one CTA has all of a head: 24576 of its keys lie in shared memory and those behind are
    read again in every pass. Lengths on both sides of that, ties across it, all of the weight behind it."""
    torch = _torch()
    rng = np.random.default_rng(len(kind))
    n_seq, n_kv, d, cap, keep, first, recent = 150, 1, 64, 24700, 300, 4, 20
    lens = rng.integers(24570, cap + 1, n_seq).astype(np.int32)
    lens[:6] = [24576, 24577, 24575, cap, 300, 0]
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    codes = lambda n: [torch.randint(0, 256, (n_seq, n_kv, n, d // 2), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
                       for _ in range(2)]
    scales = lambda n: [torch.randn((n_seq, n_kv, n, d // 32, 2), generator=g, device="cuda").half() for _ in range(2)]  # noqa: E731
    src, dst = K.Kv4Cache(*codes(cap), *scales(cap)), K.Kv4Cache(*codes(keep), *scales(keep))
    w = rng.random((n_seq, n_kv, cap)).astype(np.float32)
    if kind == "ties":
        w = np.where(w < 0.995, 0.0, np.where(np.arange(cap) < 24500, np.float32(0.5), np.float32(0.25))).astype(np.float32)
        w[:, :, 24560:24600] = 0.25
    elif kind == "late":
        w[:, :, :24570] *= 1e-6
    idx = torch.empty((n_seq, n_kv, keep), dtype=torch.int32, device="cuda")
    w_out = torch.empty((n_seq, n_kv, keep), device="cuda")
    len_out = torch.empty(n_seq, dtype=torch.int32, device="cuda")
    st = torch.cuda.current_stream()
    K.kv4_evict_dev(src, dst, _up(w), _up(lens), keep, first, recent, idx, w_out, len_out, stream=st)
    K.sync(st)
    assert np.array_equal(len_out.cpu().numpy(), np.minimum(lens, keep))
    ix, wo = idx.cpu().numpy()[:, 0], w_out.cpu().numpy()[:, 0]
    for b in range(n_seq):
        at = np_keep(w[b, 0], int(lens[b]), keep, first, recent)
        assert np.array_equal(ix[b, :len(at)], at) and (ix[b, len(at):] == -1).all(), b
        assert np.array_equal(wo[b, :len(at)], w[b, 0, at]) and (wo[b, len(at):] == 0).all(), b
        t = torch.from_numpy(at).cuda()
        for x, y in ((src.k, dst.k), (src.v, dst.v), (src.ks.view(torch.int16), dst.ks.view(torch.int16)),
                     (src.vs.view(torch.int16), dst.vs.view(torch.int16))):
            assert torch.equal(y[b, 0, :len(at)], x[b, 0, t]), b


# ------------------------------------------------- the example

def test_decode_example_refuses_what_cannot_fit():
    import importlib.util
    import os

    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("kv4_decode", os.path.join(ROOT, "examples", "kv4_decode.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    for bad in (dict(prompt=49, cap=48), dict(prompt=10, cap=48, keep=48), dict(tokens=0), dict(prompt=0)):
        with pytest.raises(ValueError, match="the prompt has to fit"):
            example.run(**bad)


@pytest.mark.gpu
@pytest.mark.parametrize("d,group,m,n_seq,n_kv,cap", [(64, 1, 3, 1, 2, 300), (64, 2, 9, 2, 2, 2500), (128, 4, 4, 2, 2, 700),
                                                      (256, 1, 5, 1, 2, 90), (256, 16, 5, 8, 2, 3000)])
def test_weights_of_slots_that_a_query_of_nan_does_not_see(kernels, d, group, m, n_seq, n_kv, cap):
    """The first token's query is NaN: its outputs are, and the weights of the slots that it sees; the newer tokens have
    their outputs, and their own slots the weights that they give them."""
    torch = _torch()
    rng = np.random.default_rng(d + m)
    host, cache = _random_cache(rng, n_seq, n_kv, cap, d, [cap] * n_seq)
    q = rng.standard_normal((n_seq * m, n_kv * group * d)).astype(np.float32)
    q[0::m] = np.nan
    out = torch.empty((n_seq * m, n_kv * group * d), device="cuda")
    w = torch.zeros((n_seq, n_kv, cap), device="cuda")
    st = torch.cuda.current_stream()
    K.kv4_attn_dev(cache, _up(q), _up(np.full(n_seq, cap, np.int32)), out, m, n_kv * group, 0.1, w_out=w, stream=st)
    K.sync(st)
    got, w = out.cpu().numpy().reshape(n_seq, m, n_kv, group, d), w.cpu().numpy()
    assert np.isnan(got[:, 0]).all() and np.isnan(w[:, :, :cap - m + 1]).all()
    q = q.reshape(n_seq, m, n_kv, group, d).astype(np.float64)
    seen = np.repeat(cap - (m - 1 - np.arange(1, m)), group)
    for b in range(n_seq):
        for h in range(n_kv):
            k, v = (np_values(c[b, h], s[b, h], x[b, h]) for c, s, x in host)
            ref, p, ds = np_attention(q[b, 1:, h].reshape(-1, d), k, v, seen, 0.1)
            y = got[b, 1:, h].reshape(-1, d)
            assert (np.abs(y - ref) <= ((2 * ds + 2.0 ** -18) * np.abs(v).max())[:, None]).all(), (b, h)
            new = slice(cap - m + 1, cap)
            tol = ((2 * ds + 2.0 ** -18)[:, None] * p[:, new]).sum(0) + 2.0 ** -22 * p[:, new].sum(0) + 1e-12
            assert (np.abs(w[b, h, new] - p[:, new].sum(0)) <= tol).all(), (b, h)
