"""Decode with a 4-bit key/value cache: one attention block of a 2304-wide decoder (36 heads of 64), run the way an engine
would run it on this library.

    x -> Q8 q, k, v projections           vmlm_gemm_nt_int8_batch_dev
      -> norm, rotation, append           vmlm_kv4_append_dev (queries rotated in the same pass)
      -> attention over the cache         vmlm_kv4_attn_dev   (and the weight each slot received)
      -> Q8 output projection, residual   vmlm_gemm_nt_int8_dev
    when the cache is full: the slots with the most weight stay, moved to the other of two caches (vmlm_kv4_evict_dev).

A prompt goes in first, then tokens one by one. `python examples/kv4_decode.py --check` also computes every step's attention
in f32 over the same slots without the 4-bit rounding and prints how far the block is from it.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import sparrow_b200.kernels as K  # noqa: E402

HIDDEN, HEADS, D, EPS = 2304, 36, 64, 1e-5


def q8(n, k, gen):
    """A projection as the Q8 path keeps it: int8 rows, one scale a row."""
    w = torch.randn((n, k), generator=gen, device="cuda") * 0.02
    scale = w.abs().amax(1) / 127
    return torch.clamp(torch.round(w / scale[:, None]), -127, 127).to(torch.int8), scale.contiguous()


class Block:
    """The weights, two caches (one in use, one to evict into) and the buffers of one attention block."""

    def __init__(self, n_seq, cap, max_tokens, seed=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.n_seq, self.cap = n_seq, cap
        self.wq, self.wk, self.wv, self.wo = (q8(HIDDEN, HIDDEN, gen) for _ in range(4))
        self.gq, self.gk = (0.8 + 0.4 * torch.rand(D, generator=gen, device="cuda") for _ in range(2))
        a = torch.arange(max_tokens, device="cuda", dtype=torch.float64)[:, None]
        a = a * 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        self.cos, self.sin = torch.cos(a).float().contiguous(), torch.sin(a).float().contiguous()
        self.cache, self.other = (K.Kv4Cache.empty(n_seq, HEADS, cap, D) for _ in range(2))
        self.weight = torch.zeros((n_seq, HEADS, cap), device="cuda")
        self.length = torch.zeros(n_seq, dtype=torch.int32, device="cuda")  # slots in use
        self.seen = torch.zeros(n_seq, dtype=torch.int32, device="cuda")    # tokens so far: the next position
        self.used = 0  # the same count as in `length`, for the host
        self.stream = torch.cuda.current_stream()

    def evict(self, keep, first, recent):
        """Keep the slots that received the most weight; returns which (per sequence and head, in order)."""
        idx = torch.empty((self.n_seq, HEADS, keep), dtype=torch.int32, device="cuda")
        kept = torch.empty((self.n_seq, HEADS, keep), device="cuda")
        now = torch.empty_like(self.length)
        K.kv4_evict_dev(self.cache, self.other, self.weight, self.length, keep, first, recent, idx, kept, now,
                        stream=self.stream)
        self.cache, self.other = self.other, self.cache
        self.weight[:, :, :keep] = kept
        self.length, self.used = now, min(self.used, keep)
        return idx

    def step(self, x, m):
        """m new tokens of every sequence, x [n_seq * m, HIDDEN]: the block's output and what --check compares."""
        rows = self.n_seq * m
        q, k, v, qr, att, y = (torch.empty((rows, HIDDEN), device="cuda") for _ in range(6))
        K.gemm_nt_int8_batch_dev([(x, w, s, o, rows, HIDDEN, HIDDEN) for (w, s), o in
                                  ((self.wq, q), (self.wk, k), (self.wv, v))], stream=self.stream)
        pos = (self.seen[:, None] + torch.arange(m, device="cuda", dtype=torch.int32)).reshape(-1).contiguous()
        rope = K.Rope(self.cos, self.sin, pos)
        K.kv4_append_dev(self.cache, k, v, self.length, m, q=q, qo=qr, n_q=HEADS, gq=self.gq, gk=self.gk, eps=EPS,
                         rope=rope, stream=self.stream)
        self.length, self.seen, self.used = self.length + m, self.seen + m, self.used + m
        K.kv4_attn_dev(self.cache, qr, self.length, att, m, HEADS, D ** -0.5, w_in=self.weight, w_out=self.weight,
                       stream=self.stream)
        K.gemm_nt_int8_dev(att, *self.wo, y, rows, HIDDEN, HIDDEN, stream=self.stream)
        return x + y, (qr, k, v, rope, att)


def run(prompt=200, tokens=64, n_seq=2, cap=224, keep=128, first=4, recent=32, check=False, seed=0):
    """Returns {"evictions", "us_per_token", "error"}: error is the largest relative difference (2-norm) of a step's
    attention from f32 attention over the same slots without the 4-bit rounding, 0 without `check`; the time a token is that of
    the tokens behind the prompt, with the check if there is one."""
    if not (tokens > 0 and 0 < prompt <= cap and keep < cap):
        raise ValueError("the prompt has to fit the cache, an eviction to leave room in it, and a token to follow")
    torch.cuda.set_device(0)
    K.init(0)
    block = Block(n_seq, cap, prompt + tokens, seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed + 1)
    evictions, worst, kf, vf = 0, 0.0, None, None
    x = torch.randn((n_seq * prompt, HIDDEN), generator=gen, device="cuda")
    for t in range(tokens + 1):
        m = prompt if t == 0 else 1
        if t == 1:
            K.sync(block.stream)
            began = time.perf_counter()
        if block.used + m > cap:
            idx = block.evict(keep, first, recent)
            evictions += 1
            if check:
                at = idx.long()[..., None].expand(-1, -1, -1, D)
                kf, vf = torch.gather(kf, 2, at), torch.gather(vf, 2, at)
        y, (q, k, v, rope, att) = block.step(x, m)
        if check:
            kr = torch.empty_like(k)
            K.qk_norm_rope_dev(None, k, None, block.gk, EPS, rope, None, kr, n_seq * m, 0, HEADS, D, stream=block.stream)
            heads = lambda z: z.reshape(n_seq, m, HEADS, D).transpose(1, 2)  # noqa: E731
            kf = heads(kr) if kf is None else torch.cat((kf, heads(kr)), 2)
            vf = heads(v) if vf is None else torch.cat((vf, heads(v)), 2)
            s = heads(q) @ kf.transpose(2, 3) * D ** -0.5
            n = kf.shape[2]
            late = torch.arange(n, device="cuda")[None] > n - m + torch.arange(m, device="cuda")[:, None]
            ref = (torch.softmax(s.masked_fill(late, float("-inf")), -1) @ vf).transpose(1, 2).reshape(n_seq * m, -1)
            worst = max(worst, ((att - ref).norm() / ref.norm()).item())
        x = y.reshape(n_seq, m, HIDDEN)[:, -1].contiguous()
        x = x / x.norm(dim=1, keepdim=True) * HIDDEN ** 0.5  # stands in for the rest of the layer
    K.sync(block.stream)
    return {"evictions": evictions, "us_per_token": (time.perf_counter() - began) / tokens * 1e6, "error": worst}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("prompt", 200), ("tokens", 64), ("n-seq", 2), ("cap", 224), ("keep", 128)):
        ap.add_argument("--" + name, type=int, default=default)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    got = run(a.prompt, a.tokens, a.n_seq, a.cap, a.keep, check=a.check)
    print(f"{a.tokens} tokens of {a.n_seq} sequences behind a prompt of {a.prompt}: {got['us_per_token']:.0f} us a token, "
          f"{got['evictions']} evictions" + (f", attention {got['error']:.3f} from f32" if a.check else ""))
