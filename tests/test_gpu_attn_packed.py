"""Causal attention over packed prompts (tptc_attn_packed) against a 64-bit form."""
import pytest

torch = pytest.importorskip("torch")

from kv8_ref import TYPES, attend, attend_and_noise, norm_bound  # noqa: E402
from tpt_spark_b200 import kernels as K  # noqa: E402

pytestmark = pytest.mark.gpu


def limits(lq, lk):
    return (torch.arange(lq) + lk - lq + 1).clamp(min=0)


def run(q, k, v, kind, lq, lk, dev, lead=0, cu_q=None, cu_k=None, most=None, status=None, stream=None):
    """q, k, v: [rows, heads, hd] views (any row stride) on the device."""
    H, hd = q.shape[1:]
    out = torch.full((q.shape[0], H, hd), 7.0, dtype=q.dtype, device=dev)
    cu = [torch.tensor([0] + x).cumsum(0).int() + lead if c is None else torch.tensor(c, dtype=torch.int32)
          for x, c in ((lq, cu_q), (lk, cu_k))]
    K.attn_packed(q, k, v, out, kind, q.stride(0), k.stride(0), v.stride(0), cu[0].to(dev), cu[1].to(dev), len(lq), q.shape[0],
                  k.shape[0], max(lq) if most is None else most, H, k.shape[1], hd, status, stream)
    torch.cuda.synchronize()
    return out


def reference(q, k, v, lq, lk, lead=0):
    out, a, b = [], lead, lead
    for n, m in zip(lq, lk):
        out.append(attend(q[a:a + n].double().cpu(), k[b:b + m].double().cpu(), v[b:b + m].double().cpu(), limits(n, m)))
        a, b = a + n, b + m
    return torch.cat(out)


def check(got, want, v, kind):
    """Weights are rounded to the type (half a step eps / 2 relative, or 2^-25 of 2^-8 and more below
    fp16's normal range), the sum that divides them is not: eps / 2 of sum p |v| <= max |v|, with f32
    sums and the exponential well below a quarter of that; then the output's own rounding."""
    eps = torch.finfo(TYPES[kind]).eps / 2
    top = v.double().abs().max().cpu()
    err = (got.cpu().double() - want).abs()
    assert (err <= 1.25 * eps * top + eps * want.abs() + 2.0 ** -25).all(), float(err.max())


CASES = [
    # n_heads, n_kv, hd, query lengths, key lengths
    (4, 1, 128, [1], [1]),
    (4, 1, 128, [300], [300]),
    (32, 8, 128, [5, 128, 1, 129, 64, 33], None),
    (8, 8, 128, [127, 257, 700], None),                 # one query head per kv head
    (14, 2, 128, [300, 18, 37], None),                  # seven: 18 tokens to a tile
    (6, 2, 64, [85, 86, 400], None),                    # three: 42 tokens
    (16, 1, 64, [1000, 9], None),
    (12, 12, 96, [200, 140], None),
    (12, 4, 96, [1, 2, 3, 500], None),
    (128, 1, 64, [5, 3], None),                         # one token to a tile
    (100, 1, 128, [4], None),
    (8, 2, 128, [10, 100, 1, 64], [500, 228, 129, 64]),  # prompts that continue a prefix
    (8, 2, 64, [10, 100, 40, 3], [4, 0, 33, 3]),         # fewer keys than queries: rows that see none
    (4, 4, 128, [0, 77, 0], [5, 77, 0]),
]


@pytest.mark.parametrize("kind", [K.F16, K.BF16])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention(cuda_device, case, kind):
    H, n_kv, hd, lq, lk = case
    lk, lead, tail, t = lk or lq, 3, 2, TYPES[kind]
    g = torch.Generator().manual_seed(len(lq) + hd)
    # q, k and v with gaps between rows; what is outside the sequences is NaN
    def rows(n, heads):
        x = torch.full((lead + n + tail, heads * hd + 24), float("nan"))
        x[lead:lead + n, :heads * hd] = torch.randn(n, heads * hd, generator=g)
        return x.to(t).to(cuda_device)[:, :heads * hd].unflatten(1, (heads, hd))

    q, k, v = rows(sum(lq), H), rows(sum(lk), n_kv), rows(sum(lk), n_kv)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    got = run(q, k, v, kind, lq, lk, cuda_device, lead=lead, status=status)
    assert int(status) == 0
    assert (got[:lead] == 7).all() and (got[lead + sum(lq):] == 7).all()
    check(got[lead:lead + sum(lq)], reference(q, k, v, lq, lk, lead), torch.nan_to_num(v, 0.0), kind)


@pytest.mark.parametrize("kind", [K.F16, K.BF16])
def test_a_long_prompt(cuda_device, kind):
    n, hd = 5000, 128
    g = torch.Generator(cuda_device).manual_seed(3)
    q, k, v = (torch.randn(n, h, hd, generator=g, device=cuda_device).to(TYPES[kind]) for h in (4, 1, 1))
    check(run(q, k, v, kind, [n], [n], cuda_device), reference(q, k, v, [n], [n]), v, kind)


def test_scores_that_climb_and_fall(cuda_device):
    """A reference maximum that moves in every tile, or never again after the first."""
    n, hd = 900, 64
    g = torch.Generator().manual_seed(4)
    v = torch.randn(n, 1, hd, generator=g).half()
    for slope in (0.2, -0.2):
        q, k = torch.zeros(n, 2, hd), torch.zeros(n, 1, hd)
        q[..., 0], k[:, 0, 0] = 8.0, torch.arange(n) * slope  # scores up to 180 apart
        q, k = q.half(), k.half()
        got = run(q.to(cuda_device), k.to(cuda_device), v.to(cuda_device), K.F16, [n], [n], cuda_device)
        check(got, reference(q, k, v, [n], [n]), v, K.F16)


@pytest.mark.parametrize("n", [40, 300, 2500])
def test_many_short_prompts_beside_long_ones(cuda_device, n):
    """Tokens to decode and prompts of every length in one batch, in an order that is not sorted."""
    hd, lq = 64, [1 + (i * 7919 % 5) * (i % 3 == 0) for i in range(n)]
    for at, long in ((n // 3, 700), (n // 2, 300), (n - 1, 699), (7, 0)):
        lq[at] = long
    lk = [m + i % 4 * 5 for i, m in enumerate(lq)]
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(m, h, hd, generator=g).half() for m, h in ((sum(lq), 2), (sum(lk), 1), (sum(lk), 1)))
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    got = run(q.to(cuda_device), k.to(cuda_device), v.to(cuda_device), K.F16, lq, lk, cuda_device, status=status)
    assert int(status) == 0
    check(got, reference(q, k, v, lq, lk), v, K.F16)


def test_as_many_sequences_as_a_grid_has_rows(cuda_device):
    """70000 tokens that see one key each: the output is that key's value."""
    n, hd, dev = 70000, 64, cuda_device
    q, k, v = (torch.randn(n, h, hd, device=dev).bfloat16() for h in (2, 1, 1))
    cu, out = torch.arange(n + 1, dtype=torch.int32, device=dev), torch.zeros_like(q)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    K.attn_packed(q, k, v, out, K.BF16, 2 * hd, hd, hd, cu, cu, n, n, n, 1, 2, 1, hd, status)
    torch.cuda.synchronize()
    assert int(status) == 0 and torch.equal(out, v.expand(-1, 2, -1))


def test_results_do_not_depend_on_the_batch(cuda_device):
    """A prompt alone, among others, and continued from a prefix: the same bits."""
    dev, hd = cuda_device, 128
    lens = [300, 41, 700, 128]
    q, k, v = (torch.randn(sum(lens), h, hd, device=dev).bfloat16() for h in (8, 2, 2))
    both = run(q, k, v, K.BF16, lens, lens, dev)
    at = 0
    for n in lens:
        one = [x[at:at + n] for x in (q, k, v)]
        assert torch.equal(run(*one, K.BF16, [n], [n], dev), both[at:at + n])
        at += n
    # the last 64 tokens of the 700: their tiles hold the same rows (64 tokens to a pair)
    tail = run(q[341 + 636:341 + 700], k[341:1041], v[341:1041], K.BF16, [64], [700], dev)
    want = reference(q[341 + 636:341 + 700], k[341:1041], v[341:1041], [64], [700])
    check(tail, want, v, K.BF16)
    for _ in range(3):
        assert torch.equal(run(q, k, v, K.BF16, lens, lens, dev), both)


BAD = {"offsets past the rows": dict(cu_q=[0, 10, 400]), "keys past the rows": dict(cu_k=[0, 10, 400]),
       "offsets that descend": dict(cu_k=[0, 10, 4]), "negative offset": dict(cu_k=[0, 10, -4]),
       "longer than said": dict(most=10), "queries that descend": dict(cu_q=[0, 10, 3])}


@pytest.mark.parametrize("what", BAD)
def test_bad_offsets_are_flagged(cuda_device, what):
    dev = cuda_device
    q, k, v = (torch.randn(50, h, 64, device=dev).half() for h in (4, 2, 2))
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    want = run(q, k, v, K.F16, [10, 40], [10, 40], dev)
    got = run(q, k, v, K.F16, [10, 40], [10, 40], dev, status=status, **BAD[what])
    assert int(status) == -1 and torch.equal(got[:10], want[:10]) and (got[10:] == 7).all()


def test_no_keys_at_all(cuda_device):
    q = torch.randn(5, 4, 64, device=cuda_device).half()
    k = torch.empty(0, 2, 64, device=cuda_device, dtype=torch.float16)
    out = torch.full_like(q, 7)
    cu = torch.tensor([0, 5], dtype=torch.int32, device=cuda_device)
    K.attn_packed(q, q, q, out, K.F16, 256, 128, 128, cu, torch.zeros_like(cu), 1, 5, 0, 5, 4, 2, 64)
    assert (out == 0).all() and k.numel() == 0


def test_in_a_graph_on_another_stream(cuda_device):
    dev, lens = cuda_device, [200, 30]
    q, k, v = (torch.randn(230, h, 96, device=dev).half() for h in (6, 3, 3))
    want = run(q, k, v, K.F16, lens, lens, dev)
    src, out = torch.zeros_like(q), torch.zeros_like(q)
    cu = torch.tensor([0, 200, 230], dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.attn_packed(src, k, v, out, K.F16, 6 * 96, 3 * 96, 3 * 96, cu, cu, 2, 230, 230, 200, 6, 3, 96,
                      stream=torch.cuda.current_stream().cuda_stream)
    src.copy_(q)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# scores as q . k, their first two dims: (the queries' values, the keys' values by index)
FAR = {
    "alike": lambda i, big: ((big, 0), (i * 0 + big, i * 0)),
    "alike below zero": lambda i, big: ((big, 0), (i * 0 - big, i * 0)),
    "climbing": lambda i, big: ((big, 0), (big / 2 + i % 900 * (big / 2048), i * 0)),
    "falling": lambda i, big: ((big, 0), (big - i % 900 * (big / 2048), i * 0)),
    "apart by f32 steps": lambda i, big: ((60000, 1), (i * 0 + 60000, i * 7919 % 4 * 256)),
    "apart by little": lambda i, big: ((2048, 1), (i * 0 + 4096, i * 7919 % 9)),
}


@pytest.mark.parametrize("what", FAR)
@pytest.mark.parametrize("kind,big", [(K.F16, 32768), (K.F16, 60000), (K.BF16, 57344), (K.BF16, 2.0 ** 60)])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_scores_far_from_zero(cuda_device, hd, kind, big, what):
    """Finite inputs whose scores times log2 e / sqrt(hd) have f32 steps far above 1; the scores themselves are exact."""
    n = 700
    (qa, qb), (ka, kb) = FAR[what](torch.arange(n, dtype=torch.float64), big)
    g = torch.Generator().manual_seed(5)
    q, k, v = torch.zeros(n, 2, hd), torch.zeros(n, 1, hd), torch.randn(n, 1, hd, generator=g).to(TYPES[kind])
    q[..., 0], q[..., 1], k[:, 0, 0], k[:, 0, 1] = qa, qb, ka, kb
    q, k = q.to(TYPES[kind]), k.to(TYPES[kind])
    got = run(q.to(cuda_device), k.to(cuda_device), v.to(cuda_device), kind, [n], [n], cuda_device)
    check(got, reference(q, k, v, [n], [n]), v, kind)


@pytest.mark.parametrize("kind", [K.F16, K.BF16])
@pytest.mark.parametrize("H,n_kv,hd,lq,lk", [(4, 1, 128, 3000, 3000), (3, 1, 64, 400, 5000), (2, 2, 96, 1500, 1500)])
def test_no_key_is_lost(cuda_device, kind, H, n_kv, hd, lq, lk):
    """Each row's output by its norm, which a few missing keys would exceed (shown in test_serve_bounds.py)."""
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(n, h, hd, generator=g).to(TYPES[kind]) for n, h in ((lq, H), (lk, n_kv), (lk, n_kv)))
    got = run(q.to(cuda_device), k.to(cuda_device), v.to(cuda_device), kind, [lq], [lk], cuda_device)
    want, noise = attend_and_noise(q.double(), k.double(), v.double(), limits(lq, lk))
    eps = torch.finfo(TYPES[kind]).eps / 2
    err = (got.cpu().double() - want).norm(dim=-1)
    bound = norm_bound(want, noise, eps, eps)
    assert (err <= bound).all(), (int((err / bound).max(1)[0].argmax()), float((err / bound).max()))
