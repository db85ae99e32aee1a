"""A batch served end to end with the batched operators: prompts of different lengths enter the paged 8-bit
cache, are attended packed, and tokens follow one by one with the log probability of each choice -- held
against the same steps in 64 bits on the same cache contents."""
import pytest

torch = pytest.importorskip("torch")

from kv8_ref import Cache, attend, rope_tables, rotate  # noqa: E402
from tpt_spark_b200 import kernels as K  # noqa: E402

pytestmark = pytest.mark.gpu

H, KV, HD, PAGE, VOCAB = 8, 2, 64, 16, 700
PROMPTS, STEPS = [70, 1, 33, 16], 6


def stored(c, b, n):
    """What the cache on the device stands for: positions 0 .. n of sequence b in f64."""
    pos = torch.arange(n)
    at, off = c.table[b].long()[pos // PAGE], pos % PAGE
    return [c.dev[x].cpu()[at, :, off].double() * c.dev[x + "s"].cpu()[at][..., None].double() for x in "kv"]


def test_prompts_then_tokens(cuda_device):
    dev, n_seq = cuda_device, len(PROMPTS)
    g = torch.Generator().manual_seed(0)
    c = Cache([n + STEPS for n in PROMPTS], PAGE, KV, HD, seed=1)
    cache = c.to(dev)
    cos, sin = rope_tables(max(PROMPTS) + STEPS, HD)
    rope = K.Rope(cos.to(dev), sin.to(dev), len(cos), HD, True)
    head = 0.2 * torch.randn(VOCAB, H * HD, generator=g)  # attention output -> logits
    table = torch.randn(VOCAB, (H + 2 * KV) * HD, generator=g).half()  # a token's q | k | v
    tokens = [torch.randint(0, VOCAB, (n,), generator=g) for n in PROMPTS]
    width = (H + 2 * KV) * HD
    work = torch.zeros(cache.attn_workspace_bytes(H), dtype=torch.uint8, device=dev)

    # the prompts
    total, most = sum(PROMPTS), max(PROMPTS)
    qkv = table[torch.cat(tokens)].to(dev)
    cu = torch.tensor([0] + PROMPTS).cumsum(0).int().to(dev)
    q, k = (torch.empty(total, h, HD, dtype=torch.float16, device=dev) for h in (H, KV))
    zero = torch.zeros(n_seq, dtype=torch.int32, device=dev)
    at, e = qkv.data_ptr(), 2 * HD
    cache.append(rope, K.F16, at, width, at + H * e, width, at + (H + KV) * e, width, H, q, k, cu, zero, total, most)
    out = torch.empty_like(q)
    K.attn_packed(q, k, at + (H + KV) * e, out, K.F16, H * HD, KV * HD, width, cu, cu, n_seq, total, total, most, H, KV, HD)
    x = table[torch.cat(tokens)].double().view(total, -1, HD)
    first = 0
    for n in PROMPTS:
        rows, pos = slice(first, first + n), torch.arange(n)
        rq, rk = (rotate(y[rows], cos[pos], sin[pos], HD, True) for y in (x[:, :H], x[:, H:H + KV]))
        want = attend(rq, rk, x[rows, H + KV:], pos + 1)
        # q, k and the weights are fp16 (half a step each; |scores| < 2^5 carry the first two), the output as well
        assert ((out[rows].cpu().double() - want).abs() <= 2.0 ** -5 * 4).all()
        assert float((out[rows].cpu().double() - want).norm() / want.norm()) < 2.0 ** -7
        first += n

    # a prompt continued from the cache instead: its last tokens against the positions read back
    b, tail = 0, 20
    n = PROMPTS[b]
    kk, vv = (torch.empty(n, KV, HD, dtype=torch.float16, device=dev) for _ in "kv")
    one = torch.tensor([0, n] + [n] * (n_seq - 1), dtype=torch.int32, device=dev)
    cache.read(one, zero, n, n, K.F16, kk, vv)
    cq = torch.tensor([0, tail], dtype=torch.int32, device=dev)
    again = torch.empty(tail, H, HD, dtype=torch.float16, device=dev)
    K.attn_packed(q[n - tail:n], kk, vv, again, K.F16, H * HD, KV * HD, KV * HD, cq, one[:2], 1, tail, n, tail, H, KV, HD)
    sk, sv = stored(c, b, n)
    want = attend(q[n - tail:n].cpu().double(), sk.half().double(), sv.half().double(), torch.arange(n - tail, n) + 1)
    assert float((again.cpu().double() - want).norm() / want.norm()) < 2.0 ** -9

    # tokens one by one
    cur = [int(t[-1]) for t in tokens]
    lens = list(PROMPTS)
    steps = torch.arange(n_seq + 1, dtype=torch.int32, device=dev)
    dhead = head.to(dev)
    for _ in range(STEPS):
        qkv = table[torch.tensor(cur)].to(dev)
        at = qkv.data_ptr()
        q = torch.empty(n_seq, H, HD, dtype=torch.float16, device=dev)
        start = torch.tensor(lens, dtype=torch.int32, device=dev)
        cache.append(rope, K.F16, at, width, at + H * e, width, at + (H + KV) * e, width, H, q, None, steps, start, n_seq, 1)
        lens = [n + 1 for n in lens]
        out = torch.empty_like(q)
        cache.attn(q, H * HD, K.F16, torch.tensor(lens, dtype=torch.int32, device=dev), H, out, work, work.numel())
        logits = out.float().view(n_seq, -1) @ dhead.T
        ids, top = torch.empty(n_seq, 3, dtype=torch.int32, device=dev), torch.empty(n_seq, 3, device=dev)
        K.logprobs(logits, K.F32, n_seq, VOCAB, VOCAB, None, None, None, 3, ids, top)
        torch.cuda.synchronize()
        for b in range(n_seq):
            sk, sv = stored(c, b, lens[b])
            want = attend(q[b:b + 1].cpu().double(), sk, sv, torch.tensor([lens[b]]))[0]
            # weights in fp16 and the output's rounding, as in the operator's own tests
            big = 127 * float(c.dev["vs"].cpu()[c.table[b, :-(-lens[b] // PAGE)].long()].max())
            assert ((out[b].cpu().double() - want).abs() <= (2.0 ** -10 + 2.0 ** -11) * big + 2.0 ** -11 * want.abs()).all()
            y = torch.log_softmax(logits[b].cpu().double(), 0)
            assert int(ids[b, 0]) == int(y.argmax()) and abs(float(top[b, 0]) - float(y.max())) < 1e-5
        cur = ids[:, 0].tolist()
    assert int(c.dev["status"]) == 0
