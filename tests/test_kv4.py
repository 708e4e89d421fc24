"""The 4-bit key/value cache of a decode step, through the C ABI: per-head norm
and rotation, append, read, attention and eviction.

The CPU tests check what the entry points refuse. The GPU tests compare with
plain implementations in f64 (or, where every step of the definition is one f32
operation, with the same steps in numpy f32, bit for bit).

Tolerances. Attention: queries are split into two halves (2^-22 of a row's
largest value), a score is an f32 sum of at most 256 exact products in chains of
at most 16 tensor-core sums (16 * 2^-23 of the sum of magnitudes), so
|ds| <= 2^-18 * scale * max|q| * sum|k| bounds a score's error with a factor 2
to spare; weights move by at most the factor exp(+-ds) each way, and are kept to
2^-21; the output is a convex combination, so |dout| <= (2 ds + 2^-18) max|v|.
The accumulated weight of a slot moves by (2 ds + 2^-18) of the weight received.
Norm and rotation: a tree of 8 sums, a root, a division, three products and a sum:
16 * 2^-24 of the two rotated values' magnitudes.
"""
import numpy as np
import pytest

import sparrow_b200.kernels as K
from sparrow_b200 import _lib
from sparrow_b200._lib import Kv4, RopeTable, VmlmError

EPS = 1e-5


# ------------------------------------------------------------ definitions

def np_quantise(x):
    """The format's definition in f32 steps: codes, step, base (f16) of x [..., d]."""
    f = np.float32
    g = np.clip(x.astype(f), f(-16384), f(16384)).reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    step = ((hi - lo) * (f(1) / f(15))).astype(np.float16)
    s = step.astype(f)
    base = (lo - f(16) * s).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(s > 0, f(1) / s, f(0)).astype(f)
        c = np.clip(np.rint((g - base.astype(f)) * inv) - f(16), f(0), f(15))
    c = np.where(np.isnan(c), 0, c)
    return c.astype(np.uint8).reshape(x.shape), step[..., 0], base[..., 0]


def np_values(codes, step, base):
    """f64 of half(step * (16 + c) + base): codes [..., d], step and base [..., d/32]."""
    c = codes.astype(np.float64).reshape(*codes.shape[:-1], codes.shape[-1] // 32, 32)
    v = step.astype(np.float64)[..., None] * (16 + c) + base.astype(np.float64)[..., None]
    return v.astype(np.float16).astype(np.float64).reshape(codes.shape)


def np_norm_rope(x, gain, cos, sin, inter):
    y = x.astype(np.float64)
    if gain is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + EPS) * gain.astype(np.float64)
    y = y.copy()
    if cos is not None:
        rot = 2 * cos.shape[-1]
        i, j = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
        a, b, c, s = y[..., i].copy(), y[..., j].copy(), cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
        y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    return y


def np_attention(q, k, v, seen, scale):
    """q [rows, d], k, v [n, d] f64, seen [rows]: output, weights [rows, n], score error bound [rows]."""
    n = k.shape[0]
    z = scale * (q @ k.T)
    z = np.where(np.arange(n)[None] < seen[:, None], z, -np.inf)
    top = np.where(seen > 0, z.max(-1, initial=-np.inf), 0)
    e = np.exp(z - top[:, None])
    p = e / np.maximum(e.sum(-1, keepdims=True), 1e-300)
    ds = 2.0 ** -18 * abs(scale) * np.abs(q).max(-1) * (np.abs(k).sum(-1).max() if n else 0)
    return p @ v, p, ds


def np_keep(w, n, keep, first, recent):
    if n <= keep:
        return np.arange(max(n, 0))
    must = np.r_[np.arange(first), np.arange(n - recent, n)]
    rest = np.arange(first, n - recent)
    x = np.where(np.isnan(w[rest]), -np.inf, w[rest].astype(np.float64))
    best = rest[np.lexsort((rest, np.isnan(w[rest]), -x))][:keep - first - recent]
    return np.sort(np.r_[must, best])


# --------------------------------------------------------- CPU: refusals

def _cache(**kw):
    c = dict(k=256, v=512, ks=1024, vs=2048, n_seq=1, n_kv=2, cap=8, d=64)
    c.update(kw)
    return Kv4(**c)


def _rc(fn, *args):
    L = _lib.lib()
    return getattr(L, fn)(*args), L.vmlm_last_error().decode()


def test_refusals_of_the_cache():
    import ctypes
    P = 4096

    def attn(c, q=P, ldq=128, ln=P, out=P, ldo=128, m=1, n_q=2, w_in=None, w_out=None):
        return _rc("vmlm_kv4_attn_dev", ctypes.byref(c) if c else None, q, ldq, ln, out, ldo, m, n_q, 0.125, w_in, w_out,
                   None)

    assert attn(None) == (1, "kv4_attn_dev: null cache")
    for d in (0, 32, 80, 96, 512):
        rc, msg = attn(_cache(d=d))
        assert rc == 2 and "head size" in msg
    assert attn(_cache(n_kv=0))[0] == 1
    assert attn(_cache(cap=1 << 31))[0] == 2 and attn(_cache(n_seq=1 << 30))[0] == 2
    for x in ("k", "v", "ks", "vs"):
        assert attn(_cache(**{x: None}))[0] == 1
        rc, msg = attn(_cache(**{x: 264}))
        assert rc == 1 and "16-byte" in msg
    rc, msg = attn(_cache(), n_q=3)
    assert rc == 2 and "evenly" in msg
    assert attn(_cache(), q=None)[0] == 1 and attn(_cache(), out=None)[0] == 1 and attn(_cache(), ln=None)[0] == 1
    rc, msg = attn(_cache(), ldq=127)
    assert rc == 1 and "row stride of q" in msg
    assert attn(_cache(), ldo=0)[0] == 1
    rc, msg = attn(_cache(), w_in=P)
    assert rc == 1 and "w_out" in msg
    assert attn(_cache(), m=1 << 31)[0] == 2
    assert attn(_cache(), m=0)[0] == 0 and attn(_cache(n_seq=0))[0] == 0 and attn(_cache(), n_q=0)[0] == 0


def test_refusals_of_append_read_and_rotation():
    import ctypes
    P = 4096

    def app(c=None, q=None, qo=None, n_q=0, k=P, ldk=128, v=P, ldv=128, rope=None, ln=P, m=1):
        return _rc("vmlm_kv4_append_dev", ctypes.byref(c or _cache()), q, 128, qo, 128, n_q, k, ldk, v, ldv, None, None,
                   1e-5, ctypes.byref(rope) if rope else None, ln, m, None)

    def table(**kw):
        t = dict(cos_t=P, sin_t=P, pos=P, n_pos=16, rot=64, interleaved=0)
        t.update(kw)
        return RopeTable(**t)

    assert app(k=None)[0] == 1 and app(v=None)[0] == 1 and app(ln=None)[0] == 1
    assert app(ldk=64)[0] == 1 and app(n_q=2)[0] == 1 and app(n_q=2, q=P)[0] == 1
    for bad in (dict(rot=0), dict(rot=8), dict(rot=24), dict(rot=80), dict(rot=128), dict(n_pos=0), dict(cos_t=None),
                dict(sin_t=None), dict(pos=None)):
        assert app(rope=table(**bad))[0] == 1, bad
    assert app(m=0)[0] == 0
    assert app(c=_cache(cap=0))[0] == 1
    assert app(m=1 << 31)[0] == 2

    def read(c=None, start=P, end=P, count=1, k=P, v=P):
        return _rc("vmlm_kv4_read_dev", ctypes.byref(c or _cache()), start, end, count, k, v, None)

    assert read(start=None)[0] == 1 and read(end=None)[0] == 1 and read(k=None)[0] == 1
    assert read(k=P + 2)[0] == 1 and read(count=0)[0] == 0 and read(count=1 << 31)[0] == 2

    def rows(q=P, k=P, qo=P, ko=P, d=64, n_q=1, n_kv=1, tokens=1, ld=64, rope=None):
        return _rc("vmlm_qk_norm_rope_dev", q, ld, k, ld, None, None, 1e-5, ctypes.byref(rope) if rope else None, qo, ld,
                   ko, ld, tokens, n_q, n_kv, d, None)

    assert rows(q=None)[0] == 1 and rows(qo=None)[0] == 1 and rows(k=None)[0] == 1 and rows(ko=None)[0] == 1
    assert rows(d=96)[0] == 2 and rows(ld=63)[0] == 1 and rows(n_q=65536)[0] == 2
    assert rows(tokens=0)[0] == 0 and rows(n_q=0, n_kv=0)[0] == 0
    assert rows(rope=table(rot=128))[0] == 1


def test_refusals_of_eviction():
    import ctypes
    P = 4096

    def evict(s=None, t=None, w=P, ln=P, keep=4, first=1, recent=2, idx=P, lo=P):
        s, t = s or _cache(), t or _cache(k=4096, v=8192, ks=16384, vs=32768)
        return _rc("vmlm_kv4_evict_dev", ctypes.byref(s), ctypes.byref(t), w, ln, keep, first, recent, idx, None, lo, None)

    assert evict(w=None)[0] == 1 and evict(ln=None)[0] == 1 and evict(idx=None)[0] == 1 and evict(lo=None)[0] == 1
    rc, msg = evict(keep=9)
    assert rc == 2 and "holds 8" in msg
    rc, msg = evict(first=3)
    assert rc == 1 and "above keep" in msg
    assert evict(first=1 << 63, recent=1 << 63)[0] == 1
    other = dict(k=4096, v=8192, ks=16384, vs=32768)
    assert evict(t=_cache(**other, n_kv=1))[0] == 2 and evict(t=_cache(**other, d=128))[0] == 2
    rc, msg = evict(t=_cache())
    assert rc == 1 and "overlap" in msg
    # the second half of src's codes
    rc, msg = evict(t=_cache(k=256 + 256, v=8192, ks=16384, vs=32768))
    assert rc == 1 and "overlap" in msg
    assert evict(s=_cache(n_seq=0), t=_cache(**other, n_seq=0))[0] == 0


def test_python_mirror_checks_its_tensors():
    import torch
    with pytest.raises(ValueError):
        K.Kv4Cache(*(torch.zeros(1, 1, 4, 32, dtype=torch.uint8) for _ in range(2)),
                   *(torch.zeros(1, 1, 4, 2, 2, dtype=torch.float16) for _ in range(2)))  # not on the GPU
    with pytest.raises(ValueError):
        K.qk_norm_rope_dev(torch.zeros(1, 64), None, None, None, EPS, None, torch.zeros(1, 64), None, 1, 1, 0, 64)


def test_definition_of_the_format():
    # the packed values are within half a step and the roundings of step, base and value to halves
    rng = np.random.default_rng(0)
    for scale, off in ((1.0, 0.0), (1e-3, 0.0), (3000.0, 0.0), (0.1, 40.0)):
        x = (rng.standard_normal((200, 64)) * scale + off).astype(np.float32)
        c, s, b = np_quantise(x)
        got = np_values(c, s, b)
        step = np.repeat(s.astype(np.float64), 32, -1)
        base = np.abs(np.repeat(b.astype(np.float64), 32, -1))
        bound = 0.5 * step + 2.0 ** -11 * (base + 31 * step) + 2.0 ** -11 * np.abs(x) + 2.0 ** -24 * 16
        assert (np.abs(got - x) <= bound).all()


# ------------------------------------------------------------------- GPU

def _torch():
    import torch
    torch.cuda.set_device(0)
    return torch


def _up(x):
    torch = _torch()
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _tables(n_pos, rot):
    a = np.arange(n_pos)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def _random_cache(rng, n_seq, n_kv, cap, d, lens, bad=True):
    """numpy codes, step, base of K and V, and the cache on the GPU; slots behind a length hold NaN and Inf."""
    torch = _torch()
    host, dev = [], []
    for _ in range(2):
        c = rng.integers(0, 16, (n_seq, n_kv, cap, d)).astype(np.uint8)
        s = (0.27 * np.exp(0.5 * rng.standard_normal((n_seq, n_kv, cap, d // 32)))).astype(np.float16)
        b = (-23.5 * s.astype(np.float64) + 0.2 * rng.standard_normal(s.shape)).astype(np.float16)
        if bad:
            for i, n in enumerate(lens):
                s[i, :, max(n, 0):] = np.nan
                b[i, :, max(n, 0):] = np.inf
        host.append((c, s, b))
        dev.append((_up(c[..., 0::2] | (c[..., 1::2] << 4)), _up(np.stack((s, b), -1))))
    cache = K.Kv4Cache(dev[0][0], dev[1][0], dev[0][1], dev[1][1])
    torch.cuda.synchronize()
    return host, cache


@pytest.mark.gpu
@pytest.mark.parametrize("d,n_q,n_kv,rot,inter,norm,tokens,slice_", [
    (64, 36, 36, 64, False, True, 1, False), (64, 3, 1, 32, True, True, 7, True), (128, 32, 8, 128, False, True, 33, True),
    (128, 5, 5, 64, False, False, 2, False), (128, 4, 2, 16, True, True, 129, True), (256, 16, 1, 256, False, True, 5, True),
    (256, 2, 2, 128, True, True, 3, False), (128, 8, 0, 128, False, True, 4, False), (64, 0, 3, 16, False, True, 4, False),
    (64, 2, 2, 0, False, True, 9, False), (256, 1, 1, 16, False, False, 70, False)])
def test_norm_and_rotation(kernels, d, n_q, n_kv, rot, inter, norm, tokens, slice_):
    torch = _torch()
    rng = np.random.default_rng(d + n_q + rot)
    width = (n_q + n_kv) * d + (1 if slice_ else 0)  # an odd row stride takes the value-by-value loads
    x = rng.standard_normal((tokens, width)).astype(np.float32) * 3
    gq, gk = (rng.uniform(0.5, 1.5, d).astype(np.float32) for _ in range(2)) if norm else (None, None)
    pos = rng.integers(0, 100, tokens).astype(np.int32)
    xd = _up(x)
    rope = cos = sin = None
    if rot:
        tc, ts = _tables(100, rot)
        cos, sin = tc[pos], ts[pos]
        rope = K.Rope(_up(tc), _up(ts), _up(pos), interleaved=inter)
    qo = torch.full((tokens + 1, max(1, n_q) * d), 7.0, device="cuda")
    ko = torch.full((tokens + 1, max(1, n_kv) * d), 7.0, device="cuda")
    st = torch.cuda.current_stream()
    K.qk_norm_rope_dev(xd[:, :n_q * d], xd[:, n_q * d:], _up(gq) if norm else None, _up(gk) if norm else None, EPS, rope,
                       qo, ko, tokens, n_q, n_kv, d, stream=st)
    K.sync(st)
    for got, heads, at, g in ((qo, n_q, 0, gq), (ko, n_kv, n_q * d, gk)):
        if not heads:
            continue
        src = x[:, at:at + heads * d].reshape(tokens, heads, d)
        ref = np_norm_rope(src, g, cos, sin, inter)
        plain = np.abs(np_norm_rope(src, g, None, None, False))
        mag = plain.copy()
        if rot:
            half = rot // 2
            if inter:
                both = plain[..., 0:rot:2] + plain[..., 1:rot:2]
                mag[..., 0:rot:2], mag[..., 1:rot:2] = both, both
            else:
                both = plain[..., :half] + plain[..., half:rot]
                mag[..., :half], mag[..., half:rot] = both, both
        y = got[:tokens].cpu().numpy().reshape(tokens, heads, d)
        assert (np.abs(y - ref) <= 16 * 2.0 ** -24 * mag + 1e-30).all()
    assert (qo[tokens] == 7).all() and (ko[tokens] == 7).all()


def np_norm_rope_f32(x, gain, cos, sin, inter):
    """The definition step by step in f32: squares added in halves, every operation rounded on its own."""
    f = np.float32
    sq = x * x
    while sq.shape[-1] > 1:
        h = sq.shape[-1] // 2
        sq = sq[..., :h] + sq[..., h:]
    y = x * (f(1) / np.sqrt(sq / f(x.shape[-1]) + f(EPS))) * gain
    rot = 2 * cos.shape[-1]
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b, c, s = y[..., i].copy(), y[..., j].copy(), cos[:, None], sin[:, None]
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("d,rot,inter,tokens", [(64, 64, False, 300), (64, 32, True, 300), (128, 128, False, 300),
                                                (128, 64, False, 1000), (128, 96, False, 50), (256, 256, True, 200),
                                                (256, 48, False, 9), (128, 128, True, 3)])
def test_norm_rotation_and_append_bit_for_bit(kernels, d, rot, inter, tokens):
    # a code must not depend on fused or reordered operations: queries, and the codes of keys and values, are numpy's
    torch = _torch()
    rng = np.random.default_rng(d + rot)
    n_q, n_kv, cap = 4, 3, tokens + 5
    x = (rng.standard_normal((tokens, (n_q + 2 * n_kv) * d)) * np.exp(rng.standard_normal((n_q + 2 * n_kv) * d))).astype(np.float32)
    gq, gk = (rng.uniform(0.5, 1.5, d).astype(np.float32) for _ in range(2))
    pos = rng.integers(0, 2000, tokens).astype(np.int32)
    tc, ts = _tables(2000, rot)
    _, cache = _random_cache(rng, 1, n_kv, cap, d, [0])
    xd = _up(x)
    qo = torch.empty((tokens, n_q * d), device="cuda")
    st = torch.cuda.current_stream()
    K.kv4_append_dev(cache, xd[:, n_q * d:(n_q + n_kv) * d], xd[:, (n_q + n_kv) * d:], _up(np.array([2], np.int32)), tokens,
                     q=xd[:, :n_q * d], qo=qo, n_q=n_q, gq=_up(gq), gk=_up(gk), eps=EPS,
                     rope=K.Rope(_up(tc), _up(ts), _up(pos), interleaved=inter), stream=st)
    K.sync(st)
    q = np_norm_rope_f32(x[:, :n_q * d].reshape(tokens, n_q, d), gq, tc[pos], ts[pos], inter)
    assert np.array_equal(qo.cpu().numpy().reshape(q.shape), q)
    k = np_norm_rope_f32(x[:, n_q * d:(n_q + n_kv) * d].reshape(tokens, n_kv, d), gk, tc[pos], ts[pos], inter)
    v = x[:, (n_q + n_kv) * d:].reshape(tokens, n_kv, d)
    for ref, codes, sb in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):
        c, s, b = np_quantise(ref.transpose(1, 0, 2))
        got = codes[0, :, 2:2 + tokens].cpu().numpy()
        assert np.array_equal(got & 15, c[..., 0::2]) and np.array_equal(got >> 4, c[..., 1::2])
        sbg = sb[0, :, 2:2 + tokens].cpu().numpy()
        assert np.array_equal(sbg[..., 0], s) and np.array_equal(sbg[..., 1], b)


@pytest.mark.gpu
def test_norm_and_rotation_in_place_and_bad_position(kernels):
    torch = _torch()
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 4 * 128)).astype(np.float32)
    g = np.ones(128, np.float32)
    tc, ts = _tables(10, 128)
    pos = np.array([0, 9, 10, 3, -1, 2], np.int32)
    q, k = _up(x[:, :256]), _up(x[:, 256:])
    st = torch.cuda.current_stream()
    K.qk_norm_rope_dev(q, k, _up(g), _up(g), EPS, K.Rope(_up(tc), _up(ts), _up(pos)), q, k, 6, 2, 2, 128, stream=st)
    with pytest.raises(VmlmError) as e:
        K.sync(st)
    assert e.value.status == 8 and "position" in str(e.value)
    K.sync(st)  # the word is cleared
    ok = np.array([0, 1, 3, 5])
    ref = np_norm_rope(x.reshape(6, 4, 128)[ok], g, tc[pos[ok]], ts[pos[ok]], False).reshape(4, -1)
    got = torch.cat((q, k), 1).cpu().numpy()
    assert np.abs(got[ok] - ref).max() < 1e-5
    assert np.array_equal(got[[2, 4]], x[[2, 4]])  # rows of a bad position are left alone


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n_seq,n_kv,cap,m", [(1, 1, 1, 1), (3, 2, 40, 7), (2, 5, 300, 130)])
def test_append_values_bit_for_bit(kernels, d, n_seq, n_kv, cap, m):
    # without norm and rotation every step is one f32 operation: codes, step and base are numpy's
    torch = _torch()
    rng = np.random.default_rng(d + cap)
    k, v = (rng.standard_normal((n_seq * m, n_kv * d)).astype(np.float32) * np.exp(rng.standard_normal((n_seq * m, 1)) * 3)
            .astype(np.float32) for _ in range(2))
    v[0, :32] = 2.5          # a constant group
    k[-1, -32:] = 1e30       # saturates
    k[0, 5] = -np.inf
    start = rng.integers(0, cap - m + 1, n_seq).astype(np.int32)
    host, cache = _random_cache(rng, n_seq, n_kv, cap, d, [cap] * n_seq, bad=False)
    st = torch.cuda.current_stream()
    K.kv4_append_dev(cache, _up(k), _up(v), _up(start), m, stream=st)
    out = [torch.empty((n_seq, n_kv, cap, d), dtype=torch.float16, device="cuda") for _ in range(2)]
    K.kv4_read_dev(cache, _up(np.zeros(n_seq, np.int32)), _up(np.full(n_seq, cap, np.int32)), cap, *out, stream=st)
    K.sync(st)
    for x, (c0, s0, b0), codes, sb, got in ((k, host[0], cache.k, cache.ks, out[0]), (v, host[1], cache.v, cache.vs, out[1])):
        rows = x.reshape(n_seq, m, n_kv, d).transpose(0, 2, 1, 3)
        c, s, b = np_quantise(rows)
        c1, s1, b1 = c0.copy(), s0.copy(), b0.copy()
        for i in range(n_seq):
            at = slice(start[i], start[i] + m)
            c1[i, :, at], s1[i, :, at], b1[i, :, at] = c[i], s[i], b[i]
        cd = codes.cpu().numpy()
        assert np.array_equal(cd & 15, c1[..., 0::2]) and np.array_equal(cd >> 4, c1[..., 1::2])
        sbd = sb.cpu().numpy()
        assert np.array_equal(sbd[..., 0], s1) and np.array_equal(sbd[..., 1], b1)
        ref = np_values(c1, s1, b1)
        assert np.array_equal(got.cpu().numpy().astype(np.float64), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("d,n_q,n_kv,rot,inter,odd", [(64, 4, 4, 64, False, False), (128, 6, 2, 64, True, True),
                                                      (256, 4, 1, 256, False, False)])
def test_append_with_norm_and_rotation(kernels, d, n_q, n_kv, rot, inter, odd):
    torch = _torch()
    rng = np.random.default_rng(d)
    n_seq, m, cap = 3, 5, 16
    x = rng.standard_normal((n_seq * m, (n_q + 2 * n_kv) * d + (3 if odd else 0))).astype(np.float32)
    gq, gk = (rng.uniform(0.8, 1.2, d).astype(np.float32) for _ in range(2))
    start = np.array([0, 11, 4], np.int32)
    pos = (start[:, None] + np.arange(m)).reshape(-1).astype(np.int32)
    tc, ts = _tables(32, rot)
    rope = K.Rope(_up(tc), _up(ts), _up(pos), interleaved=inter)
    _, cache = _random_cache(rng, n_seq, n_kv, cap, d, [0] * n_seq)
    xd = _up(x)
    qo = torch.empty((n_seq * m, n_q * d), device="cuda")
    st = torch.cuda.current_stream()
    K.kv4_append_dev(cache, xd[:, n_q * d:(n_q + n_kv) * d], xd[:, (n_q + n_kv) * d:], _up(start), m, q=xd[:, :n_q * d],
                     qo=qo, n_q=n_q, gq=_up(gq), gk=_up(gk), eps=EPS, rope=rope, stream=st)
    kr, vr = (torch.empty((n_seq, n_kv, m, d), dtype=torch.float16, device="cuda") for _ in range(2))
    K.kv4_read_dev(cache, _up(start), _up(start + np.array([m, m, m - 2], np.int32)), m, kr, vr, stream=st)
    K.sync(st)
    parts = x[:, :n_q * d], x[:, n_q * d:(n_q + n_kv) * d], x[:, (n_q + n_kv) * d:(n_q + 2 * n_kv) * d]
    ref = np_norm_rope(parts[0].reshape(-1, n_q, d), gq, tc[pos], ts[pos], inter)
    assert np.abs(qo.cpu().numpy().reshape(ref.shape) - ref).max() <= 32 * 2.0 ** -24 * np.abs(ref).max()
    key = np_norm_rope(parts[1].reshape(-1, n_kv, d), gk, tc[pos], ts[pos], inter)
    key = key.reshape(n_seq, m, n_kv, d).transpose(0, 2, 1, 3)
    _, s, b = np_quantise(key)
    step = np.repeat(s.astype(np.float64), 32, -1)
    bound = 0.5 * step + 2.0 ** -11 * (np.abs(np.repeat(b.astype(np.float64), 32, -1)) + 33 * step) + 2.0 ** -10 * np.abs(key)
    k_got, v_got = kr.cpu().numpy().astype(np.float64), vr.cpu().numpy().astype(np.float64)
    val = parts[2].reshape(n_seq, m, n_kv, d).transpose(0, 2, 1, 3)
    v_ref = np_values(*np_quantise(val))
    k_got[2, :, m - 2:] = key[2, :, m - 2:]
    assert (kr[2, :, m - 2:] == 0).all() and (vr[2, :, m - 2:] == 0).all()  # behind `end`
    v_ref[2, :, m - 2:] = 0
    assert (np.abs(k_got - key) <= bound).all()
    assert np.array_equal(v_got, v_ref)


@pytest.mark.gpu
def test_append_nan_idle_and_full(kernels):
    torch = _torch()
    rng = np.random.default_rng(2)
    d, n_kv, cap, m = 64, 2, 4, 2
    k = rng.standard_normal((3 * m, n_kv * d)).astype(np.float32)
    v = k.copy()
    k[0, 3] = np.nan
    host, cache = _random_cache(rng, 3, n_kv, cap, d, [cap] * 3, bad=False)
    before = cache.k.clone()
    st = torch.cuda.current_stream()
    K.kv4_append_dev(cache, _up(k), _up(v), _up(np.array([1, -1, 3], np.int32)), m, stream=st)
    with pytest.raises(VmlmError) as e:
        K.sync(st)
    assert e.value.status == 8 and "slot" in str(e.value)
    kr, vr = (torch.empty((3, n_kv, cap, d), dtype=torch.float16, device="cuda") for _ in range(2))
    K.kv4_read_dev(cache, _up(np.zeros(3, np.int32)), _up(np.full(3, cap, np.int32)), cap, kr, vr, stream=st)
    K.sync(st)
    got = kr.cpu().numpy()
    assert np.isnan(got[0, 0, 1, :32]).all() and not np.isnan(got[0, 0, 1, 32:]).any() and not np.isnan(got[0, 1]).any()
    assert torch.equal(cache.k[1], before[1])                      # idle: untouched
    assert torch.equal(cache.k[2, :, :3], before[2, :, :3])        # only slot 3 of a full cache was written
    assert np.array_equal(vr[2, :, 3].cpu().numpy().astype(np.float64),
                          np_values(*np_quantise(v[4].reshape(n_kv, d))))


def _check_attention(rng, d, n_seq, n_kv, group, cap, lens, m, weights, w_null=False, odd=False, in_place=False):
    torch = _torch()
    n_q = n_kv * group
    lens = np.asarray(lens, np.int32)
    host, cache = _random_cache(rng, n_seq, n_kv, cap, d, lens)
    q = rng.standard_normal((n_seq * m, n_q * d + (1 if odd else 0))).astype(np.float32)
    scale = 1 / np.sqrt(d)
    out = torch.full((n_seq * m + 1, n_q * d + (3 if odd else 0)), 7.0, device="cuda")
    w = np.exp(rng.standard_normal((n_seq, n_kv, cap))).astype(np.float32)
    for b, n in enumerate(lens):
        w[b, :, max(0, n - m):] = np.nan  # what is not history is not read
    w_in = None if w_null or not weights else _up(w)
    w_out = None
    if weights:
        w_out = w_in if in_place and w_in is not None else torch.full((n_seq, n_kv, cap), 7.0, device="cuda")
    st = torch.cuda.current_stream()
    K.kv4_attn_dev(cache, _up(q), _up(lens), out, m, n_q, scale, w_in=w_in, w_out=w_out, stream=st)
    K.sync(st)
    got = out.cpu().numpy()
    assert (got[-1] == 7).all() and (got[:, n_q * d:] == 7).all()
    got = got[:-1, :n_q * d].reshape(n_seq, m, n_q, d)
    q = q[:, :n_q * d].reshape(n_seq, m, n_q, d).astype(np.float64)
    for b in range(n_seq):
        n = max(0, int(lens[b]))
        seen = np.maximum(0, n - (m - 1 - np.arange(m)))
        for h in range(n_kv):
            kv = [np_values(c[b, h, :n], s[b, h, :n], x[b, h, :n]) for c, s, x in host]
            rows = q[b, :, h * group:(h + 1) * group].reshape(m * group, d)
            ref, p, ds = np_attention(rows, kv[0], kv[1], np.repeat(seen, group), scale)
            vmax = np.abs(kv[1]).max() if n else 0.0
            y = got[b, :, h * group:(h + 1) * group].reshape(m * group, d)
            assert (np.abs(y - ref) <= ((2 * ds + 2.0 ** -18) * vmax)[:, None] + 1e-30).all(), (b, h)
            if not weights:
                continue
            hist = np.zeros(cap)
            if not w_null:
                hist[:max(0, n - m)] = w[b, h, :max(0, n - m)]
            want = hist[:n] + p.sum(0)
            tol = ((2 * ds + 2.0 ** -18)[:, None] * p).sum(0) + 2.0 ** -22 * np.abs(want) + 1e-12
            gw = w_out[b, h].cpu().numpy()
            assert (np.abs(gw[:n] - want) <= tol).all(), (b, h)
            if not in_place:
                assert (gw[n:] == 7).all()


LENGTHS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257, 511, 1000]


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 12])
def test_attention_one_token(kernels, d, group):
    rng = np.random.default_rng(d * 100 + group)
    _check_attention(rng, d, len(LENGTHS), 2, group, 1000, LENGTHS, 1, weights=group % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("d,group,m,weights", [(64, 1, 2, True), (64, 1, 33, True), (128, 4, 5, False), (128, 4, 16, True),
                                               (256, 16, 5, True), (128, 8, 64, False), (64, 3, 7, True),
                                               (128, 1, 130, True)])
def test_attention_several_tokens(kernels, d, group, m, weights):
    # lengths below m leave the first tokens with nothing to see; 0 and negative lengths leave all of them
    rng = np.random.default_rng(d + group + m)
    lens = [0, 1, m - 1, m, m + 1, 3 * m + 5, -1, 200]
    _check_attention(rng, d, len(lens), 3, group, max(200, 3 * m + 5), lens, m, weights)


@pytest.mark.gpu
@pytest.mark.parametrize("d,n_kv,group,n,weights", [(128, 8, 4, 20011, True), (64, 36, 1, 4097, True), (256, 1, 16, 9001, False),
                                                    (64, 1, 1, 70001, True), (128, 1, 2, 33333, False)])
def test_attention_long(kernels, d, n_kv, group, n, weights):
    rng = np.random.default_rng(n)
    _check_attention(rng, d, 1, n_kv, group, n + 3, [n], 1, weights)


@pytest.mark.gpu
@pytest.mark.parametrize("d,group,m", [(64, 5, 1), (64, 9, 1), (64, 12, 1), (64, 1, 15), (64, 3, 9), (64, 33, 1), (128, 5, 1),
                                       (128, 3, 4), (128, 33, 1), (256, 2, 3), (256, 1, 24)])
@pytest.mark.parametrize("weights", [False, True])
def test_attention_rows_over_long_caches(kernels, d, group, m, weights):
    """Every count of rows that a warp takes at a time, where items are shared by warps and by CTAs."""
    rng = np.random.default_rng(d + group + m)
    _check_attention(rng, d, 5, 4, group, 5001, [5001, 4990, 0, 2177, 63], m, weights)
    _check_attention(rng, d, 1, 1, group, 20011, [20009], m, weights)


@pytest.mark.gpu
@pytest.mark.parametrize("n_seq,group,m,weights", [(4, 7, 4, True), (4, 1, 45, False), (4, 64, 1, True), (4, 16, 5, True),
                                                  (8, 16, 5, False), (8, 27, 3, True)])
def test_attention_many_rows_of_256(kernels, n_seq, group, m, weights):
    rng = np.random.default_rng(group + m)
    lens = [3001, 3000, 1723, 2944, 0, m - 1, 65, 2999][:n_seq]
    _check_attention(rng, 256, n_seq, 4, group, 3001, lens, m, weights)


@pytest.mark.gpu
def test_attention_many_ragged(kernels):
    rng = np.random.default_rng(11)
    lens = rng.integers(0, 700, 70)
    lens[5] = 0
    _check_attention(rng, 128, 70, 4, 2, 700, lens, 1, True)
    _check_attention(rng, 64, 70, 1, 1, 700, lens, 3, True)


@pytest.mark.gpu
def test_attention_strides_null_history_and_in_place(kernels):
    rng = np.random.default_rng(3)
    _check_attention(rng, 128, 2, 2, 3, 100, [77, 100], 2, True, odd=True)
    _check_attention(rng, 64, 2, 2, 3, 100, [77, 100], 2, True, w_null=True)
    _check_attention(rng, 64, 2, 2, 3, 100, [77, 100], 2, True, in_place=True)
    _check_attention(rng, 64, 2, 1, 1, 3, [0, 0], 1, True)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_peaked_and_wide_scores(kernels, d):
    """One slot takes nearly all of the weight, and many that follow or come before it share what is left: their small
    weights have to add up; large and tiny queries keep their scores."""
    torch = _torch()
    rng = np.random.default_rng(d)
    n = 6000
    for peak, size in ((0, 1.0), (n - 1, 1.0), (2500, 30.0), (77, 1e-6), (5, 1e-30)):
        host, cache = _random_cache(rng, 1, 1, n, d, [n])
        (kc, ks, kb), (vc, vs, vb) = host
        ks[:] = np.float16(0.01)
        kb[:] = np.float16(-0.235)
        ks[0, 0, peak] = np.float16(1.5)
        kb[0, 0, peak] = np.float16(-24)
        kc[0, 0, peak] = 15
        vs[:], vb[:] = np.float16(0.1), np.float16(0.4)  # one sign: nothing cancels
        cache = K.Kv4Cache(_up(kc[..., 0::2] | (kc[..., 1::2] << 4)), _up(vc[..., 0::2] | (vc[..., 1::2] << 4)),
                           _up(np.stack((ks, kb), -1)), _up(np.stack((vs, vb), -1)))
        q = np.full((1, d), size * 17.0 / (22.5 * np.sqrt(d)), np.float32) * rng.uniform(0.9, 1.1, (1, d)).astype(np.float32)
        out = torch.empty((1, d), device="cuda")
        w = torch.zeros((1, 1, n), device="cuda")
        st = torch.cuda.current_stream()
        K.kv4_attn_dev(cache, _up(q), _up(np.array([n], np.int32)), out, 1, 1, 1 / np.sqrt(d), w_out=w, stream=st)
        K.sync(st)
        k, v = np_values(kc[0, 0], ks[0, 0], kb[0, 0]), np_values(vc[0, 0], vs[0, 0], vb[0, 0])
        ref, p, ds = np_attention(q.astype(np.float64), k, v, np.array([n]), 1 / np.sqrt(d))
        assert (np.abs(out.cpu().numpy() - ref) <= (2 * ds[0] + 2.0 ** -18) * np.abs(v).max()).all()
        assert (np.abs(w.cpu().numpy()[0, 0] - p[0]) <= (2 * ds[0] + 2.0 ** -18) * p[0] + 1e-30).all()


@pytest.mark.gpu
def test_attention_extreme_queries_and_lengths(kernels):
    torch = _torch()
    rng = np.random.default_rng(8)
    d, n = 128, 300
    _, cache = _random_cache(rng, 3, 1, n, d, [n, n, n], bad=False)
    q = rng.standard_normal((3, d)).astype(np.float32)
    q[0, 7] = np.nan
    q[1] = 0.0
    lens = np.array([n, n, n + 1], np.int32)
    out = torch.empty((3, d), device="cuda")
    st = torch.cuda.current_stream()
    K.kv4_attn_dev(cache, _up(q), _up(lens), out, 1, 1, 0.1, stream=st)
    with pytest.raises(VmlmError) as e:
        K.sync(st)
    assert e.value.status == 8  # a length above cap is reported, and taken as cap
    got = out.cpu().numpy()
    assert np.isnan(got[0]).all() and np.isfinite(got[1:]).all()
    lens[2] = n
    out2 = torch.empty_like(out)
    K.kv4_attn_dev(cache, _up(q), _up(lens), out2, 1, 1, 0.1, stream=st)
    K.sync(st)
    assert torch.equal(out[1:], out2[1:])  # the same call gives the same bits


@pytest.mark.gpu
def test_attention_on_other_streams_and_repeated(kernels):
    torch = _torch()
    rng = np.random.default_rng(9)
    d, n = 128, 5000
    _, cache = _random_cache(rng, 2, 4, n, d, [n, 1234], bad=False)
    q, lens = _up(rng.standard_normal((2, 16 * d)).astype(np.float32)), _up(np.array([n, 1234], np.int32))
    outs = []
    torch.cuda.synchronize()
    for st in (torch.cuda.Stream(), None, torch.cuda.current_stream(), torch.cuda.Stream()):
        out, w = torch.empty_like(q), torch.zeros((2, 4, n), device="cuda")
        torch.cuda.synchronize()
        K.kv4_attn_dev(cache, q, lens, out, 1, 16, 0.1, w_out=w, stream=st)
        K.sync(st)
        outs.append((out, w))
    for out, w in outs[1:]:
        assert torch.equal(out, outs[0][0]) and torch.equal(w, outs[0][1])


def _check_eviction(rng, d, n_seq, n_kv, cap, keep, first, recent, lens, w, spare=0, w_null=False):
    torch = _torch()
    lens = np.asarray(lens, np.int32)
    host, src = _random_cache(rng, n_seq, n_kv, cap, d, lens)
    _, dst = _random_cache(rng, n_seq, n_kv, keep + spare, d, [keep + spare] * n_seq, bad=False)
    before = [x.clone() for x in (dst.k, dst.v, dst.ks, dst.vs)]
    idx = torch.full((n_seq, n_kv, keep), 7, dtype=torch.int32, device="cuda")
    w_out = None if w_null else torch.full((n_seq, n_kv, keep), 7.0, device="cuda")
    len_out = torch.full((n_seq,), 7, dtype=torch.int32, device="cuda")
    st = torch.cuda.current_stream()
    K.kv4_evict_dev(src, dst, _up(w), _up(lens), keep, first, recent, idx, w_out, len_out, stream=st)
    K.sync(st)
    assert np.array_equal(len_out.cpu().numpy(), np.clip(lens, 0, keep))
    ix = idx.cpu().numpy()
    for b in range(n_seq):
        for h in range(n_kv):
            at = np_keep(w[b, h], int(lens[b]), keep, first, recent)
            assert np.array_equal(ix[b, h, :len(at)], at) and (ix[b, h, len(at):] == -1).all(), (b, h)
            if not w_null:
                wo = w_out[b, h].cpu().numpy()
                assert np.array_equal(wo[:len(at)], w[b, h, at], equal_nan=True) and (wo[len(at):] == 0).all()
            t = torch.from_numpy(at).cuda()
            for x, y, z in ((src.k, dst.k, before[0]), (src.v, dst.v, before[1]), (src.ks, dst.ks, before[2]),
                            (src.vs, dst.vs, before[3])):
                bits = [u[b, h].view(torch.uint8 if u.dtype == torch.uint8 else torch.int16) for u in (x, y, z)]
                assert torch.equal(bits[1][:len(at)], bits[0][t])
                assert torch.equal(bits[1][len(at):], bits[2][len(at):])  # nothing else is written


@pytest.mark.gpu
@pytest.mark.parametrize("d,n_seq,n_kv,cap,keep,first,recent", [
    (64, 3, 2, 1, 1, 0, 0), (64, 4, 3, 50, 7, 1, 2), (128, 4, 2, 1023, 512, 4, 64), (128, 2, 2, 1025, 1, 0, 0),
    (256, 3, 1, 2500, 2400, 0, 0), (64, 2, 36, 1100, 512, 4, 64), (64, 4, 1, 300, 20, 20, 0), (64, 4, 1, 300, 20, 0, 20),
    (64, 4, 1, 300, 20, 12, 8), (128, 1, 1, 40000, 4096, 4, 256), (64, 1, 2, 70001, 333, 4, 16), (128, 2, 1, 3000, 0, 0, 0),
    (64, 9, 8, 9000, 1000, 4, 32)])
def test_eviction(kernels, d, n_seq, n_kv, cap, keep, first, recent):
    rng = np.random.default_rng(cap + keep)
    lens = ([cap, max(1, cap // 2), min(keep, cap), min(keep + 1, cap), 0, -1, cap] * 2)[:n_seq]
    w = np.exp(2 * rng.standard_normal((n_seq, n_kv, cap))).astype(np.float32)
    _check_eviction(rng, d, n_seq, n_kv, cap, keep, first, recent, lens, w, spare=cap % 3, w_null=cap % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "signs", "odd values", "descending"])
@pytest.mark.parametrize("cap", [257, 5000, 20000])
def test_eviction_ties_and_odd_weights(kernels, kind, cap):
    rng = np.random.default_rng(cap)
    w = np.full((2, 2, cap), 0.25, np.float32)
    if kind == "few":
        w = rng.integers(0, 4, w.shape).astype(np.float32)
    elif kind == "zeros":
        w = np.where(rng.random(w.shape) < 0.9, rng.choice([0.0, -0.0], w.shape), rng.random(w.shape)).astype(np.float32)
    elif kind == "signs":
        w = rng.standard_normal(w.shape).astype(np.float32)
    elif kind == "odd values":
        w = rng.choice(np.array([np.nan, np.inf, -np.inf, 0, 1e-42, -1e-42, 3e38, -3e38], np.float32), w.shape)
    elif kind == "descending":
        w = np.broadcast_to(np.arange(cap, 0, -1, dtype=np.float32), w.shape).copy()
    _check_eviction(rng, 64, 2, 2, cap, cap // 3, 3, 10, [cap, cap - 7], w)


@pytest.mark.gpu
def test_eviction_reports_a_length_above_cap(kernels):
    torch = _torch()
    rng = np.random.default_rng(1)
    _, src = _random_cache(rng, 1, 1, 8, 64, [8])
    _, dst = _random_cache(rng, 1, 1, 4, 64, [4])
    idx, lo = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (4, 1))
    st = torch.cuda.current_stream()
    K.kv4_evict_dev(src, dst, _up(np.arange(8, dtype=np.float32)), _up(np.array([9], np.int32)), 4, 0, 0, idx, None, lo,
                    stream=st)
    with pytest.raises(VmlmError):
        K.sync(st)
    assert idx.cpu().tolist() == [4, 5, 6, 7] and lo.item() == 4


@pytest.mark.gpu
def test_calls_in_a_graph(kernels):
    """One eager step sizes the workspace; captured, the same step gives the same bits on every replay."""
    torch = _torch()
    rng = np.random.default_rng(4)
    d, n_kv, n_q, cap = 128, 2, 8, 400
    _, cache = _random_cache(rng, 2, n_kv, cap, d, [cap] * 2, bad=False)
    _, small = _random_cache(rng, 2, n_kv, 100, d, [100] * 2, bad=False)
    x = _up(rng.standard_normal((2, (n_q + 2 * n_kv) * d)).astype(np.float32))
    had = _up(np.array([300, 17], np.int32))
    now = had + 1
    tc, ts = _tables(cap, d)
    rope = K.Rope(_up(tc), _up(ts), had)
    g = _up(np.ones(d, np.float32))
    qo, out = torch.empty((2, n_q * d), device="cuda"), torch.empty((2, n_q * d), device="cuda")
    w_in, w = torch.ones((2, n_kv, cap), device="cuda"), torch.zeros((2, n_kv, cap), device="cuda")
    idx = torch.empty((2, n_kv, 100), dtype=torch.int32, device="cuda")
    lo = torch.empty(2, dtype=torch.int32, device="cuda")
    st = torch.cuda.Stream()

    def step():
        K.kv4_append_dev(cache, x[:, n_q * d:(n_q + n_kv) * d], x[:, (n_q + n_kv) * d:], had, 1, q=x[:, :n_q * d], qo=qo,
                         n_q=n_q, gq=g, gk=g, eps=EPS, rope=rope, stream=st)
        K.kv4_attn_dev(cache, qo, now, out, 1, n_q, 0.1, w_in=w_in, w_out=w, stream=st)
        K.kv4_evict_dev(cache, small, w, now, 100, 4, 10, idx, None, lo, stream=st)

    torch.cuda.synchronize()
    step()
    K.sync(st)
    ref = [t.clone() for t in (qo, out, w, idx, lo, small.k, small.vs)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step()
    for _ in range(3):
        for t in (qo, out, idx):
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for t, r in zip((qo, out, w, idx, lo, small.k, small.vs), ref):
            assert torch.equal(t.view(torch.uint8), r.view(torch.uint8))
    K.sync(st)
    del graph


@pytest.mark.gpu
def test_decode_example(kernels):
    """The block of examples/kv4_decode.py: prompt, decode and evictions together. Keys and values are off by at most half a
    code step of their 32 columns (a step is about 4.1 / 15 of their deviation, so 0.08 of it in the mean square), which
    averages out over the slots of a row: 0.2 leaves room for rows that see few slots."""
    import importlib.util
    import os

    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("kv4_decode", os.path.join(ROOT, "examples", "kv4_decode.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.run(prompt=90, tokens=40, n_seq=3, cap=100, keep=60, recent=16, check=True)
    assert got["evictions"] == 1 and 0 < got["error"] < 0.2
    got = example.run(prompt=33, tokens=50, n_seq=1, cap=48, keep=40, recent=8, check=True)
    assert got["evictions"] == 5 and 0 < got["error"] < 0.2
