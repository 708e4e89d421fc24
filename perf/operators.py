"""The operators between the q/k/v projections and the output projection of a decode step, as cases to time.

    rope    per-head RMSNorm of queries and keys and the position rotation, in one pass
    append  the same, and keys and values written to a cache that holds them in 4 bits
    attn    attention of the newest tokens over that cache, with the weight that each slot received where asked for
    evict   the slots with the most accumulated weight kept, moved to another cache

A cache row of d values is d/2 bytes of codes (column p in byte p/2, the low nibble when p is even) and, for every 32
columns, (step, base) as two halves; a code c stands for half(step * (16 + c) + base). Activations are f32.

`own` chooses between the plain form of each operator (elementary torch operations in f32) and the calls that a user
makes of this package. `exact` is the same from the definitions in f64.
"""
import math

import numpy as np
import torch

own = False

GROUP = 32
CLAMP = 16384.0
EPS = 1e-5

# The 36 x 64 cases are the attention heads of this repository's own 2304-wide decoder (no grouping of heads);
# 32 query heads over 8 kv heads of 128 columns is a generic grouped layout, 16 over 1 of 256 a generic shared one.
CASES = [
    # one decoded token of one user: the smallest call there is, all latency
    dict(name="rope_token_36x64", op="rope", n_seq=1, m=1, n_q=36, n_kv=36, d=64, rot=64, inter=False),
    # a prompt of odd length, half of each head rotated
    dict(name="rope_prompt_gqa128", op="rope", n_seq=1, m=2047, n_q=32, n_kv=8, d=128, rot=64, inter=True),
    # a decode step of 24 users, each token appended behind its own history
    dict(name="append_batch_36x64", op="append", n_seq=24, m=1, n_q=36, n_kv=36, d=64, rot=64, inter=False, cap=640),
    # a long prompt written to an empty cache
    dict(name="append_prompt_gqa128", op="append", n_seq=1, m=8191, n_q=32, n_kv=8, d=128, rot=128, inter=False,
         cap=8192),
    # one token of one user over a short history: latency
    dict(name="attn_token_36x64", op="attn", n_seq=1, m=1, n_q=36, n_kv=36, d=64, cap=1024, len="one:777",
         weights=False),
    # one token over a very long history: bandwidth, with few rows to split the work by
    dict(name="attn_long_gqa128", op="attn", n_seq=1, m=1, n_q=32, n_kv=8, d=128, cap=131072, len="one:131071",
         weights=False),
    # a decode step of many users with histories of all lengths: the ordinary serving call
    dict(name="attn_ragged_gqa128", op="attn", n_seq=48, m=1, n_q=32, n_kv=8, d=128, cap=8192, len="ragged",
         weights=False),
    # the last window of a prompt, whose weights choose what the cache keeps
    dict(name="attn_window_weights_36x64", op="attn", n_seq=2, m=33, n_q=36, n_kv=36, d=64, cap=4097, len="full",
         weights=True),
    # a decode step that accumulates the weights
    dict(name="attn_token_weights_gqa128", op="attn", n_seq=8, m=1, n_q=32, n_kv=8, d=128, cap=16384, len="ragged",
         weights=True),
    # a few drafted tokens checked at once, one shared kv head
    dict(name="attn_draft_mqa256", op="attn", n_seq=16, m=5, n_q=16, n_kv=1, d=256, cap=3001, len="ragged",
         weights=False),
    # a small budget for one user
    dict(name="evict_36x64", op="evict", n_seq=1, n_kv=36, d=64, cap=1100, keep=512, first=4, recent=64, len="full"),
    # long prompts of several users cut to a budget
    dict(name="evict_long_gqa128", op="evict", n_seq=8, n_kv=8, d=128, cap=32768, keep=4096, first=4, recent=256,
         len="ragged"),
]

#: What no drawn case exceeds: cache values (n_seq * n_kv * length * d), scores (n_seq * n_q * m * cap), activation
#: values (and values of kept rows).
MOST_CACHE, MOST_SCORES, MOST_ROWS = 200_000_000, 12_000_000, 33_000_000


def listed():
    return [dict(c) for c in CASES]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attn", "attn", "attn", "evict"])
    d = rng.choice([64, 128, 128, 256])
    n_kv = rng.choice([1, 2, 3, 4, 8, 8, 36])
    group = rng.choice([1, 2, 3, 4, 4, 6, 8, 16]) if n_kv < 36 else 1
    n_seq = _spread(rng, 1, 64)
    case = dict(op=op, n_seq=n_seq, n_kv=n_kv, d=d)
    if op in ("rope", "append"):
        m = _spread(rng, 1, 8191)
        row = n_kv * (group + 2) * d
        m = max(1, min(m, MOST_ROWS // (row * n_seq)))
        case.update(m=m, n_q=n_kv * group, rot=rng.choice([d, d // 2]), inter=rng.random() < 0.3)
        if op == "append":
            case["cap"] = m + _spread(rng, 1, 512)
        return case
    cap = _spread(rng, 1, 131072)
    case["len"] = rng.choice(["ragged", "full"])
    if op == "evict":
        cap = max(2, min(cap, MOST_CACHE // (n_seq * n_kv * d)))
        keep = max(1, min(int(cap * rng.uniform(0.05, 0.8)), MOST_ROWS // (n_seq * n_kv * d)))
        case.update(cap=cap, keep=keep, first=min(4, keep), recent=min(_spread(rng, 1, 256), max(0, keep - 4)))
        return case
    m = rng.choice([1, 1, 1, rng.randint(2, 8), _spread(rng, 9, 64)])
    cap = max(1, min(cap, MOST_CACHE // (n_seq * n_kv * d), MOST_SCORES // (n_seq * n_kv * group * m)))
    case.update(cap=cap, m=m, n_q=n_kv * group, weights=rng.random() < 0.4)
    return case


def _lengths(case):
    """Slots in use of each sequence: of the case alone, so that its work is known without a seed."""
    n, cap, how = case["n_seq"], case["cap"], case["len"]
    if how == "full":
        return [cap] * n
    if how == "ragged":  # spread evenly over 1..cap, in no order
        return [1 + int((cap - 1) * ((b * 0.6180339887498949 + 0.97) % 1.0)) for b in range(n)]
    return [int(how.split(":")[1])] * n


def work(case):
    d, n_kv = case["d"], case["n_kv"]
    row = 1.25 * d  # codes, steps and bases of one slot, K and V together
    if case["op"] in ("rope", "append"):
        tokens, n_q = case["n_seq"] * case["m"], case["n_q"]
        values = tokens * (n_q + n_kv) * d
        table = tokens * case["rot"] * 4 + tokens * 4
        if case["op"] == "rope":
            return {"bytes": 8.0 * values + table, "flops": 10.0 * values}
        # q in and out, k and v in, the cache rows out, and the values that they stand for (halves)
        moved = tokens * (8 * n_q * d + 8 * n_kv * d + n_kv * row + 4 * n_kv * d)
        return {"bytes": float(moved + table), "flops": 10.0 * values + 8.0 * tokens * n_kv * d}
    total = sum(_lengths(case))
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in _lengths(case)) * n_kv
        # scores in; kept rows read and written; index and score of each out; all rows' values out (halves)
        out = case["n_seq"] * n_kv * case["keep"]
        return {"bytes": 4.0 * total * n_kv + kept * 2 * row + out * (8 + 4 * d), "flops": 2.0 * total * n_kv}
    rows = case["n_seq"] * case["m"] * case["n_q"]
    seen = sum(max(0, n - (case["m"] - 1 - t)) for n in _lengths(case) for t in range(case["m"]))
    moved = total * n_kv * row + rows * d * 8 + (8.0 * total * n_kv if case["weights"] else 0)
    return {"bytes": float(moved), "flops": 4.0 * seen * case["n_q"] * d}


# ------------------------------------------------------------------ inputs

def _rope_tables(n_pos, rot, dev):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    a = torch.arange(n_pos, dtype=torch.float64, device=dev)[:, None] * inv
    return torch.cos(a).float(), torch.sin(a).float()


def _cache(g, n_seq, n_kv, cap, d, dev, length=None):
    """Codes and (step, base) of keys and values: heads of unlike size, some slots much larger than the rest, as caches
    are. What lies behind a sequence's length is left over from before: any bits, NaN among them."""
    out = {}
    for x in ("k", "v"):
        out[x] = torch.randint(0, 256, (n_seq, n_kv, cap, d // 2), generator=g, device=dev, dtype=torch.uint8)
        step = 0.27 * torch.exp(0.5 * torch.randn((n_seq, n_kv, cap, 1), generator=g, device=dev))
        step = step * (0.7 + 0.6 * torch.rand((n_seq, n_kv, cap, d // GROUP), generator=g, device=dev))
        mid = 0.2 * torch.randn((n_seq, n_kv, cap, d // GROUP), generator=g, device=dev)
        sb = torch.empty((n_seq, n_kv, cap, d // GROUP, 2), dtype=torch.float16, device=dev)
        sb[..., 0] = step
        sb[..., 1] = mid - 23.5 * step
        if length is not None:
            sb.masked_fill_((torch.arange(cap, device=dev) >= length[:, None])[:, None, :, None, None], float("nan"))
        out[x + "s"] = sb
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    n_seq, n_kv, d = case["n_seq"], case["n_kv"], case["d"]
    s = dict(case=case, dev=dev)
    if case["op"] in ("rope", "append"):
        tokens, n_q = n_seq * case["m"], case["n_q"]
        # q, k and v as one projection's output: rows of all heads, the three parts side by side
        width = (n_q + 2 * n_kv) * d
        x = torch.randn((tokens, width), generator=g, device=dev)
        x *= torch.exp(0.7 * torch.randn((width,), generator=g, device=dev))
        s["q"], s["k"], s["v"] = x[:, :n_q * d], x[:, n_q * d:(n_q + n_kv) * d], x[:, (n_q + n_kv) * d:]
        s["gq"] = 0.8 + 0.4 * torch.rand((d,), generator=g, device=dev)
        s["gk"] = 0.8 + 0.4 * torch.rand((d,), generator=g, device=dev)
        n_pos = 16384
        s["cos"], s["sin"] = _rope_tables(n_pos, case["rot"], dev)
        room = (case["cap"] if case["op"] == "append" else n_pos) - case["m"]
        start = torch.randint(0, room + 1, (n_seq,), generator=g, device=dev, dtype=torch.int32)
        s["start"] = start
        s["pos"] = (start[:, None] + torch.arange(case["m"], device=dev, dtype=torch.int32)).reshape(-1).contiguous()
        s["qo"] = torch.empty((tokens, n_q * d), device=dev)
        if case["op"] == "rope":
            s["ko"] = torch.empty((tokens, n_kv * d), device=dev)
        else:
            s["cache"] = _cache(g, n_seq, n_kv, case["cap"], d, dev, start)
            s["end"] = start + case["m"]
            s["kr"] = torch.empty((n_seq, n_kv, case["m"], d), dtype=torch.float16, device=dev)
            s["vr"] = torch.empty_like(s["kr"])
    else:
        cap = case["cap"]
        s["len"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
        s["cache"] = _cache(g, n_seq, n_kv, cap, d, dev, s["len"])
        # accumulated weight: heavy-tailed, many slots that never received any, and equal ones
        w = torch.exp(2.0 * torch.randn((n_seq, n_kv, cap), generator=g, device=dev))
        w = torch.where(torch.rand(w.shape, generator=g, device=dev) < 0.2, torch.zeros_like(w), w)
        s["w"] = torch.where(w > 1.0, w, torch.floor(w * 64) / 64)
        if case["op"] == "attn":
            s["q"] = torch.randn((n_seq * case["m"], case["n_q"] * d), generator=g, device=dev)
            s["out"] = torch.empty_like(s["q"])
            s["w_out"] = torch.zeros_like(s["w"])
        else:
            keep = case["keep"]
            s["dst"] = _cache(g, n_seq, n_kv, keep, d, dev)
            s["idx"] = torch.empty((n_seq, n_kv, keep), dtype=torch.int32, device=dev)
            s["w_kept"] = torch.empty((n_seq, n_kv, keep), device=dev)
            s["len_out"] = torch.empty((n_seq,), dtype=torch.int32, device=dev)
            s["zero"] = torch.zeros((n_seq,), dtype=torch.int32, device=dev)
            s["kr"] = torch.empty((n_seq, n_kv, keep, d), dtype=torch.float16, device=dev)
            s["vr"] = torch.empty_like(s["kr"])
    if own:
        import sparrow_b200.kernels as K
        K.init(0)
        s["K"] = K
        s["stream"] = torch.cuda.current_stream()
        for name in ("cache", "dst"):
            if name in s:
                c = s[name]
                s[name + "_h"] = K.Kv4Cache(c["k"], c["v"], c["ks"], c["vs"])
        if "cos" in s:
            s["rope"] = K.Rope(s["cos"], s["sin"], s["pos"], interleaved=case["inter"])
    return s


# --------------------------------------------------------- the package's calls

def _run_own(s):
    c, K, st = s["case"], s["K"], s["stream"]
    if c["op"] == "rope":
        K.qk_norm_rope_dev(s["q"], s["k"], s["gq"], s["gk"], EPS, s["rope"], s["qo"], s["ko"], c["n_seq"] * c["m"],
                           c["n_q"], c["n_kv"], c["d"], stream=st)
        return {"q": s["qo"], "k": s["ko"]}
    if c["op"] == "append":
        K.kv4_append_dev(s["cache_h"], s["k"], s["v"], s["start"], c["m"], q=s["q"], qo=s["qo"], n_q=c["n_q"],
                         gq=s["gq"], gk=s["gk"], eps=EPS, rope=s["rope"], stream=st)
        K.kv4_read_dev(s["cache_h"], s["start"], s["end"], c["m"], s["kr"], s["vr"], stream=st)
        return {"q": s["qo"], "k": s["kr"], "v": s["vr"]}
    if c["op"] == "attn":
        if c["weights"]:
            K.kv4_attn_dev(s["cache_h"], s["q"], s["len"], s["out"], c["m"], c["n_q"], 1.0 / math.sqrt(c["d"]),
                           w_in=s["w"], w_out=s["w_out"], stream=st)
            return {"out": s["out"], "w": s["w_out"]}
        K.kv4_attn_dev(s["cache_h"], s["q"], s["len"], s["out"], c["m"], c["n_q"], 1.0 / math.sqrt(c["d"]), stream=st)
        return {"out": s["out"]}
    K.kv4_evict_dev(s["cache_h"], s["dst_h"], s["w"], s["len"], c["keep"], c["first"], c["recent"], s["idx"],
                    s["w_kept"], s["len_out"], stream=st)
    K.kv4_read_dev(s["dst_h"], s["zero"], s["len_out"], c["keep"], s["kr"], s["vr"], stream=st)
    return {"idx": s["idx"], "w": s["w_kept"], "len": s["len_out"], "k": s["kr"], "v": s["vr"]}


# ------------------------------------------------------------- the plain form

def _norm_rope(x, gain, cos, sin, rot, inter):
    """x [tokens, heads, d]: RMSNorm of each head, then the rotation of its first `rot` columns."""
    sq = x * x
    while sq.shape[-1] > 1:  # the sum of squares: halves added until one value is left
        h = sq.shape[-1] // 2
        sq = sq[..., :h] + sq[..., h:]
    y = x * (1.0 / torch.sqrt(sq / x.shape[-1] + EPS)) * gain
    c, s = cos[:, None, :], sin[:, None, :]
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if inter else (y[..., :rot // 2], y[..., rot // 2:rot])
    ra, rb = a * c - b * s, b * c + a * s
    turned = torch.stack((ra, rb), -1).reshape(*x.shape[:-1], rot) if inter else torch.cat((ra, rb), -1)
    return torch.cat((turned, y[..., rot:]), -1)


def _through_4_bits(x):
    """The values that x [..., d] stands for once it is held in 4 bits."""
    g = x.reshape(*x.shape[:-1], -1, GROUP).clamp(-CLAMP, CLAMP)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = ((hi - lo) / 15.0).half().float()
    base = (lo - 16.0 * step).half().float()
    inv = torch.where(step > 0, 1.0 / step, torch.zeros_like(step))
    code = (torch.round((g - base) * inv) - 16.0).clamp(0.0, 15.0)
    return (step * (16.0 + code) + base).half().reshape(x.shape)


def _values(codes, sb):
    """f32 values of 4-bit rows: codes [..., d/2], sb [..., d/32, 2]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    c = c.reshape(*sb.shape[:-1], GROUP)
    sb = sb.float()
    return (sb[..., :1] * (16.0 + c) + sb[..., 1:]).half().float().flatten(-2)


def _run_plain(s):
    c = s["case"]
    n_seq, n_kv, d = c["n_seq"], c["n_kv"], c["d"]
    if c["op"] in ("rope", "append"):
        tokens, n_q, m = n_seq * c["m"], c["n_q"], c["m"]
        at = s["pos"].long()
        cos, sin = s["cos"][at], s["sin"][at]
        q = _norm_rope(s["q"].reshape(tokens, n_q, d), s["gq"], cos, sin, c["rot"], c["inter"])
        k = _norm_rope(s["k"].reshape(tokens, n_kv, d), s["gk"], cos, sin, c["rot"], c["inter"])
        if c["op"] == "rope":
            return {"q": q.reshape(tokens, -1), "k": k.reshape(tokens, -1)}
        k = k.reshape(n_seq, m, n_kv, d).transpose(1, 2)
        v = s["v"].reshape(n_seq, m, n_kv, d).transpose(1, 2)
        return {"q": q.reshape(tokens, -1), "k": _through_4_bits(k), "v": _through_4_bits(v)}
    cap, kv = c["cap"], s["cache"]
    slot = torch.arange(cap, device=s["dev"])
    if c["op"] == "attn":
        m, group = c["m"], c["n_q"] // n_kv
        used = (slot < s["len"][:, None])[:, None, :, None]
        k = torch.where(used, _values(kv["k"], kv["ks"]), torch.zeros((), device=s["dev"]))
        v = torch.where(used, _values(kv["v"], kv["vs"]), torch.zeros((), device=s["dev"]))
        q = s["q"].reshape(n_seq, m, n_kv, group, d).permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, m * group, d)
        score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
        seen = s["len"][:, None] - (m - 1 - torch.arange(m, device=s["dev"]))
        mask = (slot < seen[:, :, None])[:, None, :, None, :]
        score = score.reshape(n_seq, n_kv, m, group, cap).masked_fill_(~mask, float("-inf"))
        top = score.amax(-1, keepdim=True)
        p = torch.exp(score - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
        out = torch.matmul(p.reshape(n_seq, n_kv, m * group, cap), v)
        out = out.reshape(n_seq, n_kv, m, group, d).permute(0, 2, 1, 3, 4).reshape(n_seq * m, -1)
        if not c["weights"]:
            return {"out": out}
        old = torch.where(slot < s["len"][:, None] - m, 1.0, 0.0)[:, None, :]
        w = torch.where((slot < s["len"][:, None])[:, None, :], s["w"] * old + p.sum((2, 3)), s["w_out"])
        return {"out": out, "w": w}
    keep, n = c["keep"], s["len"].long()[:, None, None]
    w = s["w"]
    kept_always = (slot < c["first"]) | (slot >= n - c["recent"])
    key = torch.where(kept_always, torch.full_like(w, float("inf")), w)
    key = torch.where(slot < n, key, torch.full_like(w, float("-inf")))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    some = torch.arange(keep, device=s["dev"]) < n  # a shorter sequence keeps all it has
    idx = torch.where(some, order, torch.full_like(order, cap)).sort(-1).values
    at = torch.where(some, idx, torch.zeros_like(idx))
    out = {"idx": torch.where(some, idx, torch.full_like(idx, -1)).int(),
           "w": torch.where(some, torch.gather(w, 2, at), torch.zeros((), device=s["dev"])),
           "len": torch.clamp(s["len"], max=keep)}
    for x in ("k", "v"):
        codes = torch.gather(kv[x], 2, at[..., None].expand(-1, -1, -1, d // 2))
        sb = torch.gather(kv[x + "s"], 2, at[..., None, None].expand(-1, -1, -1, d // GROUP, 2))
        out[x] = torch.where(some[..., None], _values(codes, sb), torch.zeros((), device=s["dev"])).half()
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------- the definitions in f64

def _exact_norm_rope(x, gain, cos, sin, rot, inter):
    x = x.astype(np.float64)
    y = x / np.sqrt(np.mean(x ** 2, axis=-1, keepdims=True) + EPS) * gain.astype(np.float64)
    z = y[..., :rot:2] + 1j * y[..., 1:rot:2] if inter else y[..., :rot // 2] + 1j * y[..., rot // 2:rot]
    z = z * (cos.astype(np.float64) + 1j * sin.astype(np.float64))[:, None, :]
    if inter:
        y[..., :rot:2], y[..., 1:rot:2] = z.real, z.imag
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    return y


def _exact_4_bits(x):
    g = np.clip(x.astype(np.float64), -CLAMP, CLAMP).reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    step = ((hi - lo) / 15).astype(np.float16).astype(np.float64)
    base = (lo - 16 * step).astype(np.float16).astype(np.float64)
    code = np.clip(np.rint((g - base) / np.where(step > 0, step, 1)) - 16, 0, 15) * (step > 0)
    return (step * (16 + code) + base).astype(np.float16).astype(np.float64).reshape(x.shape)


def _exact_values(codes, sb):
    """f64 values of 4-bit rows on the GPU: codes [n, d/2], sb [n, d/32, 2]."""
    c = torch.empty((codes.shape[0], codes.shape[1] * 2), dtype=torch.float64, device=codes.device)
    c[:, 0::2], c[:, 1::2] = (codes % 16).double(), (codes // 16).double()
    step, base = (sb[..., i].double().repeat_interleave(GROUP, -1) for i in (0, 1))
    return (step * (16 + c) + base).half().double()


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    n_seq, n_kv, d = case["n_seq"], case["n_kv"], case["d"]
    if case["op"] in ("rope", "append"):
        host = {k: s[k].cpu().numpy() for k in ("q", "k", "v", "gq", "gk", "pos", "cos", "sin")}
        tokens, m = n_seq * case["m"], case["m"]
        cos, sin = host["cos"][host["pos"]], host["sin"][host["pos"]]
        q, k = (_exact_norm_rope(host[x].reshape(tokens, -1, d), host["g" + x], cos, sin, case["rot"], case["inter"])
                for x in ("q", "k"))
        if case["op"] == "rope":
            return {"q": q.reshape(tokens, -1), "k": k.reshape(tokens, -1)}
        v = host["v"].reshape(tokens, n_kv, d)
        turn = lambda x: _exact_4_bits(x).reshape(n_seq, m, n_kv, d).transpose(0, 2, 1, 3)  # noqa: E731
        return {"q": q.reshape(tokens, -1), "k": turn(k), "v": turn(v)}
    lens, kv = _lengths(case), s["cache"]
    if case["op"] == "attn":
        m, n_q = case["m"], case["n_q"]
        group = n_q // n_kv
        q = s["q"].double().reshape(n_seq, m, n_q, d)
        out = torch.zeros_like(q)
        w = s["w_out"].double()
        for b, n in enumerate(lens):
            for h in range(n_kv):
                if n < 1:
                    continue
                k = _exact_values(kv["k"][b, h, :n], kv["ks"][b, h, :n])
                v = _exact_values(kv["v"][b, h, :n], kv["vs"][b, h, :n])
                z = q[b, :, h * group:(h + 1) * group] @ k.T / math.sqrt(d)
                late = torch.arange(n, device=z.device)[None, :] > n - m + torch.arange(m, device=z.device)[:, None]
                p = torch.softmax(z.masked_fill(late[:, None, :], float("-inf")), -1)
                p = torch.nan_to_num(p, nan=0.0)  # a token before the first slot sees nothing
                out[b, :, h * group:(h + 1) * group] = p @ v
                w[b, h, :n] = p.sum((0, 1))
                w[b, h, :max(0, n - m)] += s["w"][b, h, :max(0, n - m)].double()
        out = out.reshape(n_seq * m, -1)
        return {"out": out, "w": w} if case["weights"] else {"out": out}
    keep = case["keep"]
    idx = np.full((n_seq, n_kv, keep), -1, np.int64)
    w = np.zeros((n_seq, n_kv, keep))
    out = {x: torch.zeros((n_seq, n_kv, keep, d), dtype=torch.float64, device=s["dev"]) for x in ("k", "v")}
    scores = s["w"].cpu().numpy()
    for b, n in enumerate(lens):
        for h in range(n_kv):
            x = scores[b, h, :n].astype(np.float64)
            if n <= keep:
                at = np.arange(n)
            else:
                must = np.union1d(np.arange(min(case["first"], n)), np.arange(max(0, n - case["recent"]), n))
                rest = np.setdiff1d(np.arange(n), must)
                best = rest[np.lexsort((rest, -x[rest]))][:keep - len(must)]
                at = np.sort(np.concatenate((must, best)))
            idx[b, h, :len(at)], w[b, h, :len(at)] = at, x[at]
            t = torch.from_numpy(at).to(s["dev"])
            for y in ("k", "v"):
                out[y][b, h, :len(at)] = _exact_values(kv[y][b, h][t], kv[y + "s"][b, h][t])
    return {"idx": idx.astype(np.int32), "w": w, "len": np.minimum(np.array(lens), keep).astype(np.int32), **out}
