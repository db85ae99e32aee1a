"""Plain 64-bit forms of the paged 8-bit KV cache, on the CPU, and the makers of its test inputs."""
import math

import torch

TYPES = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}


def rope_tables(rows, dim, base=10000.0):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def rotate(x, cos, sin, dim, halves):
    """x [rows, heads, hd] (f64), cos / sin [rows, dim / 2]."""
    y = x.clone()
    a, b = (slice(0, dim // 2), slice(dim // 2, dim)) if halves else (slice(0, dim, 2), slice(1, dim, 2))
    c, s = cos.double()[:, None], sin.double()[:, None]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


class Cache:
    """Codes, scales and a shuffled page table for sequences with room for `room[b]` positions."""

    def __init__(self, room, page, n_kv, hd, seed, extra=2, max_pages=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-r // page) for r in room]
        self.page, self.n_kv, self.hd, self.n_seq = page, n_kv, hd, len(room)
        self.n_pages, self.max_pages = sum(need) + extra, max_pages or max(max(need), 1)
        order = torch.randperm(self.n_pages, generator=g).int()
        self.table = torch.full((len(room), self.max_pages), -7, dtype=torch.int32)  # unused entries are no pages
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = order[at:at + m]
            at += m
        shape = (self.n_pages, n_kv, page, hd)
        self.k, self.v = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in "kv")
        self.ks, self.vs = (0.002 + 0.02 * torch.rand(shape[:2], generator=g) for _ in "kv")

    def to(self, dev):
        from tpt_spark_b200 import kernels as K

        self.dev = {n: getattr(self, n).clone().to(dev) for n in ("k", "v", "ks", "vs", "table")}
        self.dev["status"] = torch.zeros(1, dtype=torch.int32, device=dev)
        d = self.dev
        return K.Kv8Cache(d["k"], d["v"], d["ks"], d["vs"], d["table"], d["status"], self.n_pages, self.page, self.n_kv,
                          self.hd, self.n_seq, self.max_pages)

    def values(self, b, n, first=0):
        """K and V of positions first .. first + n of sequence b as [n, heads, hd] in f64."""
        pos = torch.arange(first, first + n)
        at, off = self.table[b].long()[pos // self.page], pos % self.page
        return [(c[at, :, off].double() * s[at][..., None].double()) for c, s in ((self.k, self.ks), (self.v, self.vs))]


def attend(q, k, v, limit):
    """Causal attention in f64: q [lq, H, hd], k / v [lk, n_kv, hd]; row i sees limit[i] keys (none: zeros)."""
    H, G = q.shape[1], q.shape[1] // k.shape[1]
    out = torch.zeros_like(q)
    seen = torch.arange(k.shape[0])[None] < limit[:, None]
    some = limit > 0
    for h in range(H):
        s = q[:, h] @ k[:, h // G].T / math.sqrt(q.shape[2])
        p = torch.softmax(s.masked_fill(~seen, -math.inf)[some], 1)
        out[some, h] = p @ v[:, h // G]
    return out
