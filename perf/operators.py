"""Measured cases of the batched-serving operators: the paged 8-bit KV cache (append with the position
rotation, read back, decode attention), causal attention over packed prompts, and log probabilities.

``own`` selects between the plain torch form of each operator and the library's kernels.  Head
layouts and vocabularies are those of the benchmark configurations (32 query heads on 8 or 32 kv
heads, head_dim 64 / 96 / 128, vocabularies of 32000 to 128256 tokens)."""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = float(np.finfo(np.float32).tiny)


# ---------------------------------------------------------------- cases


def listed():
    return [
        # one decode step of a 64-sequence batch: a token each, in the middle of half-filled pages
        dict(name="append_decode_64", op="append", n_seq=64, lo=1, hi=1, start=2000, page=16, n_heads=32, n_kv=8, hd=128,
             rot=128, halves=False, type="f16", ragged=1),
        # eight ragged prompts entering an empty cache, rotation over half of each head
        dict(name="append_prompts_8", op="append", n_seq=8, lo=500, hi=1800, start=0, page=64, n_heads=32, n_kv=8, hd=128,
             rot=64, halves=True, type="bf16", ragged=2),
        # a short cached prefix of one sequence (a system prompt) read back for its continuation
        dict(name="read_prefix_1", op="read", n_seq=1, lo=300, hi=300, page=16, n_kv=8, hd=128, type="bf16", ragged=3),
        # the cached turns of a batch read back
        dict(name="read_prefix_6", op="read", n_seq=6, lo=2000, hi=6000, page=32, n_kv=8, hd=128, type="f16", ragged=4),
        # one chat, one token: the smallest call, latency counts
        dict(name="decode_1x777", op="decode", n_seq=1, lo=777, hi=777, page=16, n_heads=32, n_kv=8, hd=128, type="f32",
             ragged=5),
        # a ragged batch in service
        dict(name="decode_32_ragged", op="decode", n_seq=32, lo=40, hi=8000, page=32, n_heads=32, n_kv=8, hd=128,
             type="f16", ragged=6),
        # long contexts
        dict(name="decode_8x32k", op="decode", n_seq=8, lo=31001, hi=32768, page=64, n_heads=32, n_kv=8, hd=128,
             type="bf16", ragged=7),
        # one short prompt
        dict(name="prompt_1x301", op="prompt", n_seq=1, lo=301, hi=301, n_heads=32, n_kv=8, hd=128, type="f16", ragged=8),
        # a batch of ragged prompts, 64-wide heads
        dict(name="prompt_12_ragged", op="prompt", n_seq=12, lo=60, hi=2100, n_heads=32, n_kv=8, hd=64, type="bf16",
             ragged=9),
        # one long prompt
        dict(name="prompt_1x8192", op="prompt", n_seq=1, lo=8192, hi=8192, n_heads=32, n_kv=8, hd=128, type="bf16",
             ragged=10),
        # log probabilities beside one sampled token
        dict(name="logprobs_1", op="logprobs", rows=1, vocab=128256, n_top=20, type="f32", ragged=11),
        # scoring a prompt
        dict(name="logprobs_1500", op="logprobs", rows=1500, vocab=128256, n_top=5, type="bf16", ragged=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "prompt", "logprobs"])
    c = dict(op=op, type=rng.choice(["f16", "bf16"]), ragged=rng.randrange(1 << 20))
    if op == "logprobs":
        c.update(rows=_log_int(rng, 1, 700), vocab=_log_int(rng, 32000, 130000), n_top=rng.randint(1, 32),
                 type=rng.choice(["f32", "f16", "bf16"]))
        return c
    hd = rng.choice([64, 96, 128, 128])
    n_kv, group = rng.choice([(8, 4), (8, 4), (32, 1), (4, 3), (1, 8), (4, 7), (2, 16)])
    c.update(hd=hd, n_kv=n_kv)
    if op != "read":
        c.update(n_heads=n_kv * group)
    if op != "prompt":
        c.update(page=rng.choice([16, 32, 64]))
    if op == "append":
        n = _log_int(rng, 1, 64)
        if rng.random() < 0.4:
            c.update(n_seq=n, lo=1, hi=1, start=_log_int(rng, 1, 4000))
        else:
            hi = _log_int(rng, 2, max(2, 8000 // n))
            c.update(n_seq=n, lo=max(1, hi // 4), hi=hi, start=rng.choice([0, 0, _log_int(rng, 1, 500)]))
        c.update(rot=rng.choice([hd, hd // 2]), halves=rng.random() < 0.5, type=rng.choice(["f32", "f16", "bf16"]))
    elif op == "read":
        n = _log_int(rng, 1, 32)
        hi = _log_int(rng, 2, 24000 // n)
        c.update(n_seq=n, lo=max(1, hi // 5), hi=hi)
    elif op == "decode":
        n = _log_int(rng, 1, 96)
        hi = _log_int(rng, 2, min(32768, 200000 // n))
        c.update(n_seq=n, lo=max(1, hi // 20), hi=hi, type=rng.choice(["f32", "f16", "bf16"]))
        if n * hi * n_kv > 1500000:  # the cost of the largest listed case
            c["hi"] = max(2, 1500000 // (n * n_kv))
            c["lo"] = max(1, c["hi"] // 20)
    else:
        n = _log_int(rng, 1, 24)
        hi = _log_int(rng, 2, int(6000 / math.sqrt(n)))
        c.update(n_seq=n, lo=max(1, hi // 8), hi=hi)
    return c


def _lengths(c):
    r = random.Random(c["ragged"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["n_seq"])]


def _starts(c):
    r = random.Random(c["ragged"] + 1)
    return [r.randint(c["start"] // 2, c["start"]) for _ in range(c["n_seq"])]


def work(c):
    e = TYPES[c["type"]].itemsize
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * e + c["rows"] * (12 + 8 * c["n_top"]), "flops": 4 * n}
    n, hd, kv = _lengths(c), c["hd"], c["n_kv"]
    if c["op"] == "append":
        t, back = sum(n), sum(a + s % c["page"] for a, s in zip(n, _starts(c)))
        ev = 2 if c["type"] == "f32" else e
        moved = 2 * t * (c["n_heads"] + kv) * hd * e + t * kv * hd * e  # q and k in and out, v in
        return {"bytes": moved + 2 * t * kv * hd + 2 * back * kv * hd * (1 + ev), "flops": 3 * t * (c["n_heads"] + kv) * c["rot"]}
    if c["op"] == "read":
        return {"bytes": 2 * sum(n) * kv * hd * (1 + e), "flops": 2 * sum(n) * kv * hd}
    if c["op"] == "decode":
        return {"bytes": 2 * sum(n) * kv * hd + 2 * len(n) * c["n_heads"] * hd * e, "flops": 4 * sum(n) * c["n_heads"] * hd}
    return {"bytes": 2 * sum(n) * (c["n_heads"] + kv) * hd * e,
            "flops": 4 * hd * c["n_heads"] * sum(a * (a + 1) // 2 for a in n)}


# ---------------------------------------------------------------- inputs


def _cu(n):
    return torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device=DEV)


def _quantise(x):
    """A page's rows as codes with one scale for each (page, head): [pages, heads, rows, hd]."""
    s = x.abs().amax((2, 3)) / 127
    return (x / s[..., None, None]).round().clamp(-127, 127).to(torch.int8), s


def _cache(c, total, g):
    """A cache whose pages lie in a shuffled order, with room for total[b] positions of sequence b."""
    page, kv, hd = c["page"], c["n_kv"], c["hd"]
    need = [-(-t // page) for t in total]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device=DEV)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    s = dict(table=table, n_pages=n_pages, status=torch.zeros(1, dtype=torch.int32, device=DEV))
    for name in "kv":
        x = torch.randn(n_pages, kv, page, hd, generator=g, device=DEV)
        if name == "k":  # keys have channels that stand out
            x *= 1 + 3 * (torch.rand(1, kv, 1, hd, generator=g, device=DEV) < 0.05)
        s[name + "_codes"], s[name + "_scale"] = _quantise(x)
    return s


def _rope_tables(rows, rot):
    inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    a = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * inv
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    c, t = case, TYPES[case["type"]]
    if c["op"] == "logprobs":
        x = 2.5 * torch.randn(c["rows"], c["vocab"], generator=g, device=DEV)
        tokens = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device=DEV, dtype=torch.int32)
        x[torch.arange(c["rows"], device=DEV), tokens.long()] += 8 * torch.rand(c["rows"], generator=g, device=DEV)
        return dict(c=c, logits=x.to(t), tokens=tokens)
    n, kv, hd = _lengths(c), c["n_kv"], c["hd"]
    total = sum(n)

    def rows(heads, count=total):
        return torch.randn(count, heads, hd, generator=g, device=DEV).to(t)

    if c["op"] == "append":
        start = _starts(c)
        s = _cache(c, [a + b for a, b in zip(n, start)], g)
        first = [b - b % c["page"] for b in start]  # positions whose stored values an append can change
        back = [a + b - f for a, b, f in zip(n, start, first)]
        # q, k and v lie side by side, as a fused projection leaves them
        qkv = torch.randn(total, c["n_heads"] + 2 * kv, hd, generator=g, device=DEV).to(t)
        s["cos"], s["sin"] = _rope_tables(max(a + b for a, b in zip(n, start)), c["rot"])
        s.update(qkv=qkv, cu=_cu(n), start=torch.tensor(start, dtype=torch.int32, device=DEV), total=total, most=max(n),
                 back_cu=_cu(back), back_start=torch.tensor(first, dtype=torch.int32, device=DEV), back_total=sum(back),
                 back_most=max(back))
    elif c["op"] == "read":
        s = _cache(c, n, g)
        s.update(cu=_cu(n), start=torch.zeros(len(n), dtype=torch.int32, device=DEV), total=total, most=max(n))
    elif c["op"] == "decode":
        s = _cache(c, n, g)
        s.update(q=rows(c["n_heads"], len(n)), lens=torch.tensor(n, dtype=torch.int32, device=DEV), most=max(n))
    else:
        s = dict(q=rows(c["n_heads"]), k=rows(kv), v=rows(kv), cu=_cu(n), total=total, most=max(n))
    s["c"] = c
    return s


# ---------------------------------------------------------------- plain forms


def _of_tokens(cu, start, total):
    """Sequence and position of each packed row."""
    n = (cu[1:] - cu[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(len(n), device=DEV), n, output_size=total)
    return seq, start.long()[seq] + torch.arange(total, device=DEV) - cu.long()[seq]


def _rotate(x, cos, sin, rot, halves):
    y = x.clone()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if halves else (slice(0, rot, 2), slice(1, rot, 2))
    cos, sin = cos[:, None, :], sin[:, None, :]
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def _store(codes, scale, x, page_of, off, first_page, first_off):
    """x [rows, heads, hd] into pages page_of at rows off; first_page / first_off: where each sequence begins."""
    kv = x.shape[1]
    most = torch.zeros_like(scale).scatter_reduce_(0, page_of[:, None].expand(-1, kv), x.abs().amax(2), "amax")
    old = scale.clone()
    old[page_of[off == 0]] = 0
    new = torch.maximum(old, most / 127)
    new = torch.where(new < TINY, 0, new)
    ratio = torch.where(new > 0, old / new, 0)[first_page][:, :, None, None]
    was = codes[first_page]
    earlier = torch.arange(codes.shape[2], device=DEV)[None, None, :, None] < first_off[:, None, None, None]
    codes[first_page] = torch.where(earlier, (was * ratio).round().to(torch.int8), was)
    inv = torch.where(new > 0, 1 / new, 0)
    q = (x * inv[page_of][..., None]).round().clamp(-127, 127).to(torch.int8)
    codes[page_of[:, None], torch.arange(kv, device=DEV)[None], off[:, None]] = q
    scale[page_of] = new[page_of]


def _values(s, cu, start, total, t):
    seq, pos = _of_tokens(cu, start, total)
    page = s["k_codes"].shape[2]
    at, off = s["table"].long()[seq, pos // page], pos % page
    return [(s[n + "_codes"][at, :, off].float() * s[n + "_scale"][at][..., None]).to(t) for n in "kv"]


def _append(s, read_type):
    c, kv = s["c"], s["c"]["n_kv"]
    seq, pos = _of_tokens(s["cu"], s["start"], s["total"])
    q, k, v = s["qkv"].float().split([c["n_heads"], kv, kv], 1)
    cos, sin = s["cos"][pos], s["sin"][pos]
    q, k = (_rotate(x, cos, sin, c["rot"], c["halves"]) for x in (q, k))
    at, off = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    begin = s["start"].long()
    first_page = s["table"].long().gather(1, (begin // c["page"])[:, None])[:, 0]
    _store(s["k_codes"], s["k_scale"], k, at, off, first_page, begin % c["page"])
    _store(s["v_codes"], s["v_scale"], v, at, off, first_page, begin % c["page"])
    ck, cv = _values(s, s["back_cu"], s["back_start"], s["back_total"], read_type)
    t = s["qkv"].dtype
    return dict(q=q.to(t), k=k.to(t), k_cache=ck, v_cache=cv, k_scale=s["k_scale"], v_scale=s["v_scale"])


def _softmax_product(scores, mask, v):
    scores = scores.masked_fill(~mask, -math.inf)
    e = (scores - scores.amax(-1, keepdim=True)).exp()
    return (e / e.sum(-1, keepdim=True)) @ v


def _decode(s):
    c, q = s["c"], s["q"]
    n, kv, hd = q.shape[0], c["n_kv"], c["hd"]
    at = s["table"].long()
    k, v = ((s[x + "_codes"][at].float() * s[x + "_scale"][at][..., None, None]).transpose(1, 2).reshape(n, kv, -1, hd)
            for x in "kv")
    scores = q.float().view(n, kv, -1, hd) @ k.transpose(2, 3) / math.sqrt(hd)
    mask = torch.arange(k.shape[2], device=DEV) < s["lens"][:, None, None, None]
    return _softmax_product(scores, mask, v).reshape(q.shape).to(q.dtype)


def _prompt(s):
    c, cu, m = s["c"], s["cu"].long(), s["most"]
    kv, hd, group = c["n_kv"], c["hd"], c["n_heads"] // c["n_kv"]
    n, i = cu[1:] - cu[:-1], torch.arange(m, device=DEV)
    at = (cu[:-1, None] + i).clamp(max=s["total"] - 1)
    q = s["q"][at].float().view(-1, m, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(-1, kv, group * m, hd)
    k, v = (s[x][at].float().transpose(1, 2) for x in "kv")
    scores = (q @ k.transpose(2, 3) / math.sqrt(hd)).view(-1, kv, group, m, m)
    v = torch.where((i < n[:, None])[:, None, :, None], v, 0)
    out = _softmax_product(scores, i[None, :] <= i[:, None], v[:, :, None])
    out = out.permute(0, 3, 1, 2, 4).reshape(-1, m, c["n_heads"], hd)
    return out[i < n[:, None]].to(s["q"].dtype)


def _logprobs(s):
    x, rows = s["logits"].float(), torch.arange(s["c"]["rows"], device=DEV)
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    z = e.sum(1, dtype=torch.float64)
    log_z = z.log()
    order = x.sort(dim=1, descending=True, stable=True)[1][:, :s["c"]["n_top"]]  # ties: lowest index first
    return dict(logprob=(d[rows, s["tokens"].long()].double() - log_z).float(),
                entropy=(log_z - (e * d).sum(1, dtype=torch.float64) / z).float(),
                top_ids=order.to(torch.int32), top_logprobs=(d.gather(1, order).double() - log_z[:, None]).float())


# ---------------------------------------------------------------- one pass


def _handle(s, K):
    """The cache's descriptor, made once beside the cache it describes."""
    if "handle" not in s:
        c = s["c"]
        s["handle"] = K.Kv8Cache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], s["table"], s["status"], s["n_pages"],
                                 c["page"], c["n_kv"], c["hd"], s["table"].shape[0], s["table"].shape[1])
    return s["handle"]


def _own(s):
    from tpt_spark_b200 import kernels as K

    c = s["c"]
    kind = {"f32": K.F32, "f16": K.F16, "bf16": K.BF16}[c["type"]]
    t = TYPES[c["type"]]
    st = torch.cuda.current_stream().cuda_stream  # the one that the inputs and the outputs belong to
    if c["op"] == "logprobs":
        r, n = c["rows"], c["n_top"]
        logprob, entropy = torch.empty(2, r, device=DEV).unbind(0)
        top_lp, top_ids = torch.empty(r, n, device=DEV), torch.empty(r, n, dtype=torch.int32, device=DEV)
        K.logprobs(s["logits"], kind, r, c["vocab"], c["vocab"], s["tokens"], logprob, entropy, n, top_ids, top_lp, stream=st)
        return dict(logprob=logprob, entropy=entropy, top_ids=top_ids, top_logprobs=top_lp)
    kv, hd = c["n_kv"], c["hd"]
    if c["op"] == "prompt":
        h, out = c["n_heads"], torch.empty_like(s["q"])
        K.attn_packed(s["q"], s["k"], s["v"], out, kind, h * hd, kv * hd, kv * hd, s["cu"], s["cu"], c["n_seq"], s["total"],
                      s["total"], s["most"], h, kv, hd, stream=st)
        return out
    cache = _handle(s, K)
    if c["op"] == "decode":
        h, out = c["n_heads"], torch.empty_like(s["q"])
        if "work" not in s:
            s["work"] = torch.zeros(cache.attn_workspace_bytes(h), dtype=torch.uint8, device=DEV)
        cache.attn(s["q"], h * hd, kind, s["lens"], h, out, s["work"], s["work"].numel(), stream=st)
        return out

    def read(cu, start, total, most, kind, t):
        k, v = torch.empty(2, total, kv, hd, dtype=t, device=DEV).unbind(0)
        cache.read(cu, start, total, most, kind, k, v, stream=st)
        return k, v

    if c["op"] == "read":
        return read(s["cu"], s["start"], s["total"], s["most"], kind, t)
    h, width = c["n_heads"], (c["n_heads"] + 2 * kv) * hd
    if "rope" not in s:
        s["rope"] = K.Rope(s["cos"], s["sin"], s["cos"].shape[0], c["rot"], c["halves"])
    q = torch.empty(s["total"], h, hd, dtype=t, device=DEV)
    k = torch.empty(s["total"], kv, hd, dtype=t, device=DEV)
    qkv, e = s["qkv"].data_ptr(), s["qkv"].element_size() * hd
    cache.append(s["rope"], kind, qkv, width, qkv + h * e, width, qkv + (h + kv) * e, width, h, q, k, s["cu"], s["start"],
                 s["total"], s["most"], stream=st)
    if c["type"] == "f32":
        kind, t = K.F16, torch.float16
    ck, cv = read(s["back_cu"], s["back_start"], s["back_total"], s["back_most"], kind, t)
    return dict(q=q, k=k, k_cache=ck, v_cache=cv, k_scale=s["k_scale"], v_scale=s["v_scale"])


def run(s):
    if own:
        return _own(s)
    c = s["c"]
    t = torch.float16 if c["type"] == "f32" else TYPES[c["type"]]  # the type of values read back
    if c["op"] == "append":
        return _append(s, t)
    if c["op"] == "read":
        return tuple(_values(s, s["cu"], s["start"], s["total"], TYPES[c["type"]]))
    return {"decode": _decode, "prompt": _prompt, "logprobs": _logprobs}[c["op"]](s)


# ---------------------------------------------------------------- 64 bits


def _attend64(q, k, v, limit):
    """Rows q [r, hd] over keys [m, hd]; row i sees the first limit[i] keys."""
    p = q @ k.T / math.sqrt(q.shape[1])
    p = torch.softmax(p.masked_fill(torch.arange(k.shape[0], device=DEV)[None] >= limit[:, None], -math.inf), 1)
    return p @ v


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "logprobs":
        lp, h, ids, top = [], [], [], []
        for i in range(0, c["rows"], 256):
            y = torch.log_softmax(s["logits"][i:i + 256].double(), 1)
            lp.append(y.gather(1, s["tokens"][i:i + 256, None].long())[:, 0])
            h.append(-(y.exp() * y).sum(1))
            o = s["logits"][i:i + 256].double().sort(dim=1, descending=True, stable=True)[1][:, :c["n_top"]]
            ids.append(o.int())
            top.append(y.gather(1, o))
        return dict(logprob=torch.cat(lp), entropy=torch.cat(h), top_ids=torch.cat(ids), top_logprobs=torch.cat(top))
    n, kv, hd, page = _lengths(c), c["n_kv"], c["hd"], c.get("page")
    if c["op"] == "prompt":
        group, out, at = c["n_heads"] // kv, [], 0
        for m in n:
            limit = torch.arange(1, m + 1, device=DEV)
            q, k, v = (s[x][at:at + m].double() for x in ("q", "k", "v"))
            out.append(torch.stack([_attend64(q[:, h], k[:, h // group], v[:, h // group], limit)
                                    for h in range(c["n_heads"])], 1))
            at += m
        return torch.cat(out)

    def stored(name, b, m):
        """The first m positions of sequence b as [heads, m, hd]."""
        at = s["table"][b, :-(-m // page)].long()
        x = s[name + "_codes"][at].double() * s[name + "_scale"][at].double()[..., None, None]
        return x.transpose(0, 1).reshape(kv, -1, hd)[:, :m]

    if c["op"] == "decode":
        group, out = c["n_heads"] // kv, []
        for b, m in enumerate(n):
            k, v, q = stored("k", b, m), stored("v", b, m), s["q"][b].double()
            limit = torch.full((group,), m, device=DEV)
            out.append(torch.cat([_attend64(q[h * group:(h + 1) * group], k[h], v[h], limit) for h in range(kv)]))
        return torch.stack(out)
    if c["op"] == "read":
        return tuple(torch.cat([stored(x, b, m).transpose(0, 1) for b, m in enumerate(n)]) for x in "kv")
    # append, sequence by sequence and page by page
    h, rot, start = c["n_heads"], c["rot"], _starts(c)
    x = s["qkv"].double()
    pos = torch.cat([torch.arange(b, b + m, device=DEV) for b, m in zip(start, n)])
    cos, sin = s["cos"].double()[pos][:, None], s["sin"].double()[pos][:, None]
    turned = x[:, :h + kv].clone()
    if c["halves"]:
        lo, hi = x[:, :h + kv, :rot // 2], x[:, :h + kv, rot // 2:rot]
        turned[..., :rot] = torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1)
    else:
        z = torch.view_as_complex(x[:, :h + kv, :rot].reshape(len(x), h + kv, rot // 2, 2).contiguous())
        turned[..., :rot] = torch.view_as_real(z * torch.complex(cos, sin)).flatten(-2)
    got = {}
    for name, rows in (("k", turned[:, h:]), ("v", x[:, h + kv:])):
        scale, back, at = s[name + "_scale"].double(), [], 0
        for b, m in enumerate(n):
            done = 0
            while done < m:
                p, off = divmod(start[b] + done, page)
                take = min(page - off, m - done)
                new, where = rows[at + done:at + done + take], int(s["table"][b, p])
                top = new.abs().amax((0, 2)) / 127
                if off:
                    was = scale[where].clone()
                    scale[where] = torch.maximum(was, top)
                    old = s[name + "_codes"][where, :, :off].double()
                    back.append((torch.round(old * (was / scale[where])[:, None, None]) * scale[where][:, None, None]).transpose(0, 1))
                else:
                    scale[where] = top
                step = scale[where][None, :, None]
                back.append(torch.round(new / step) * step)
                done += take
            at += m
        got[name + "_cache"], got[name + "_scale"] = torch.cat(back), scale
    return dict(q=turned[:, :h], k=turned[:, h:], **got)
