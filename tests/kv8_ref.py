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


def attend_and_noise(q, k, v, limit, drop=None):
    """attend(), and for each (row, head) sum p_j^2 |v_j|^2, what independent errors of the weights act on.
    drop: a slice of keys that is left out of the sums, as a kernel that lost them would."""
    H, G = q.shape[1], q.shape[1] // k.shape[1]
    out, noise = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=q.dtype)
    seen = torch.arange(k.shape[0])[None] < limit[:, None]
    if drop is not None:
        seen[:, drop] = False
    for h in range(H):
        s = (q[:, h] @ k[:, h // G].T / math.sqrt(q.shape[2])).masked_fill(~seen, -math.inf)
        p = torch.softmax(s, 1).nan_to_num(0.0)
        out[:, h], noise[:, h] = p @ v[:, h // G], p ** 2 @ (v[:, h // G] ** 2).sum(1)
    return out, noise


def norm_bound(want, noise, weight, result):
    """How far a (row, head) of attention may lie from `want`, as a norm over head_dim: the weights carry independent
    roundings of up to `weight` relative (their mean square is at most a third of its square) and the output's
    elements of up to `result`; three times the root of the two together, as the sum of two or more roundings stays
    below sqrt(6) of it and that of many has nearly its mean.  f32 sums, exponentials and scores: 2^-16 of the same sizes."""
    size = want.norm(dim=-1)
    return 3 * ((weight ** 2 * noise + result ** 2 * size ** 2) / 3).sqrt() + 2.0 ** -16 * (size + noise.sqrt()) + 1e-9


def whole_inputs(case, dtype):
    """Cache and queries (scores within a few units) for the cases that look for lost keys."""
    n_heads, n_kv, hd, page, lens = case
    c = Cache(lens, page, n_kv, hd, 23)
    q = (0.7 * torch.randn(len(lens), n_heads, hd, generator=torch.Generator().manual_seed(24))).to(dtype)
    return c, q


def roundings(dtype):
    """Of the weights and of the result in decode attention: 16-bit queries take fp16 weights, f32 ones two fp16 parts
    (scores of up to 2^5 carry 2^-22 each: 2^-17)."""
    if dtype == torch.float32:
        return 2.0 ** -17, 2.0 ** -24
    return 2.0 ** -11, torch.finfo(dtype).eps / 2
