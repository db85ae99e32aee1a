"""Decode attention over the paged 8-bit cache (tptc_kv8_attn) against a 64-bit form."""
import pytest

torch = pytest.importorskip("torch")

from kv8_ref import TYPES, Cache, attend, attend_and_noise, norm_bound, roundings, whole_inputs  # noqa: E402
from tpt_spark_b200 import kernels as K  # noqa: E402
from tpt_spark_b200._lib import EngineError  # noqa: E402

pytestmark = pytest.mark.gpu


def run(c, q, kind, lens, dev, work=None, stride=None, stream=None):
    """c: a Cache moved to dev by its to()."""
    H, hd = q.shape[1], q.shape[2]
    out = torch.full((len(lens), H, hd), float("nan"), dtype=TYPES[kind], device=dev)
    if work is None:
        work = torch.zeros(c.handle.attn_workspace_bytes(H), dtype=torch.uint8, device=dev)
    c.handle.attn(q, stride or H * hd, kind, torch.tensor(lens, dtype=torch.int32, device=dev), H, out, work, work.numel(), stream)
    torch.cuda.synchronize()
    return out


def make(lens, page, n_kv, hd, seed, dev, **kw):
    c = Cache(lens, page, n_kv, hd, seed, **kw)
    c.handle = c.to(dev)
    return c


def reference(c, q, lens):
    out = []
    for b, n in enumerate(lens):
        k, v = c.values(b, n)
        out.append(attend(q[b:b + 1].double().cpu(), k, v, torch.tensor([n])))
    return torch.cat(out)


def check(got, want, c, lens, kind):
    """With V codes up to 127 steps of the largest scale (big = 127 max vs over the sequence's pages):
    f32 -- scores carry |s| 2^-22 (a 22-bit query, f32 sums of up to 128 products), |s| < 2^5 here, so weights are
    off by 2^-17 relative at most, f16 pairs by 2^-22, the exponential by 2^-22: 2^-16 big;
    f16, bf16 -- the same, and each weight rounded to fp16 (2^-11, or 2^-25 of the largest
    where it is subnormal): 2^-10.5 of sum p |v| <= big; then the output's own rounding."""
    kind = kind if isinstance(kind, int) else K.F32
    rel = 2.0 ** -16 if kind == K.F32 else 2.0 ** -16 + 2.0 ** -10.5
    eps = 0 if kind == K.F32 else torch.finfo(TYPES[kind]).eps / 2
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        big = 127 * float(c.vs[c.table[b, :-(-n // c.page)].long()].max())
        err = (got[b].cpu().double() - want[b]).abs()
        assert (err <= rel * big + eps * want[b].abs() + 2.0 ** -25).all(), (b, n, float(err.max()), rel * big)


CASES = [
    # n_heads, n_kv, hd, page, lens
    (32, 8, 128, 16, [1]),
    (32, 8, 128, 32, [777]),
    (32, 8, 128, 64, [16, 0, 17, 15, 64, 1000, 1, 33, 0]),
    (8, 1, 64, 16, [5000, 3]),
    (7, 1, 64, 64, [129, 2000, 31]),
    (4, 4, 64, 32, [300, 1]),
    (12, 4, 96, 16, [47, 0, 1025]),
    (32, 32, 96, 32, [100, 4, 65]),
    (28, 4, 128, 16, [259, 1, 512]),
    (16, 1, 128, 64, [700, 63]),      # two passes of eight heads
    (44, 4, 64, 16, [33, 480]),       # eleven heads per kv head: eight and three
    (2, 1, 128, 16, [40000]),         # one pair over many CTAs
    (4, 2, 64, 16, [1 + (7 * i) % 90 for i in range(300)]),  # more sequences than threads
]


@pytest.mark.parametrize("kind", [K.F32, K.F16, K.BF16])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention(cuda_device, case, kind):
    n_heads, n_kv, hd, page, lens = case
    c = make(lens, page, n_kv, hd, 11, cuda_device)
    g = torch.Generator().manual_seed(12)
    q = (0.7 * torch.randn(len(lens), n_heads, hd, generator=g)).to(TYPES[kind])
    got = run(c, q.to(cuda_device), kind, lens, cuda_device)
    check(got, reference(c, q, lens), c, lens, kind)
    assert int(c.dev["status"]) == 0


def test_calls_repeat_and_share_a_workspace(cuda_device):
    """The same bits every time, whatever ran on the workspace before, and with strided queries."""
    lens = [3000, 10, 0, 511, 7000]
    c = make(lens, 16, 2, 128, 13, cuda_device)
    q = torch.randn(5, 8, 128, device=cuda_device).half()
    wide = torch.zeros(5, 12, 128, dtype=torch.float16, device=cuda_device)
    wide[:, :8] = q
    work = torch.zeros(c.handle.attn_workspace_bytes(8), dtype=torch.uint8, device=cuda_device)
    first = run(c, q, K.F16, lens, cuda_device, work)
    for other in ([10, 10, 0, 500, 10], [2999, 1, 0, 1, 6999]):
        run(c, q, K.F16, other, cuda_device, work)
        assert torch.equal(run(c, q, K.F16, lens, cuda_device, work), first)
    out = torch.empty_like(first)
    c.handle.attn(wide, 12 * 128, K.F16, torch.tensor(lens, dtype=torch.int32, device=cuda_device), 8, out, work, work.numel())
    assert torch.equal(out, first)


def test_one_workspace_for_batches_of_any_shape(cuda_device):
    """A batch that grows and shrinks, other heads and widths: one workspace serves them all."""
    shapes = [(3, 8, 2, 64, 900), (60, 32, 8, 128, 700), (2, 16, 1, 96, 3000), (60, 32, 8, 64, 300), (3, 8, 2, 64, 900)]
    caches = []
    for i, (n, H, n_kv, hd, most) in enumerate(shapes):
        lens = [1 + (most * (7 * b + 3 * i + 1)) // 997 % most for b in range(n)]
        c = make(lens, 16, n_kv, hd, 30 + i, cuda_device)
        q = torch.randn(n, H, hd, device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(i)).half()
        caches.append((c, q, lens, run(c, q, K.F16, lens, cuda_device)))
    work = torch.zeros(max(c.handle.attn_workspace_bytes(q.shape[1]) for c, q, _, _ in caches), dtype=torch.uint8,
                       device=cuda_device)
    for c, q, lens, want in caches + caches[::-1]:
        assert torch.equal(run(c, q, K.F16, lens, cuda_device, work), want)


@pytest.mark.parametrize("kind", [K.F16, K.BF16, K.F32])
def test_pages_of_very_different_scales(cuda_device, kind):
    """A page of huge values that nearly no weight falls on, beside small ones that carry the output; a page of zeros."""
    lens, hd = [96], 64
    c = Cache(lens, 16, 1, hd, 14)
    p = c.table[0].long()
    c.k[p] = 0
    c.k[p[3:], :, :, 0] = 1
    c.ks[:] = 1.0
    c.vs[:] = 1e-6
    c.vs[p[0]] = 0.0      # the first page stands for zeros
    c.vs[p[1]] = 1.0      # scores 0: weight e^-40 each against pages 3 ..
    c.handle = c.to(cuda_device)
    q = torch.zeros(1, 1, hd)
    q[0, 0, 0] = 320.0    # score 40 where the key is 1
    q = q.to(TYPES[kind])
    got = run(c, q.to(cuda_device), kind, lens, cuda_device).cpu().double()
    want = reference(c, q, lens)
    # relative to the largest contribution of about 127e-6; an fp16 output has steps of 2^-24 there
    tol = 2.0 ** -10 * 127e-6 + (2.0 ** -25 if kind == K.F16 else 2.0 ** -9 * want.abs())
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("size", [1e-30, 1e-3, 3e4, 1e30])
@pytest.mark.parametrize("kind", [K.F32, K.BF16])
def test_queries_of_any_size(cuda_device, kind, size):
    """Scores stay of order one while q and the key scales go to the ends of the range."""
    lens = [200]
    c = Cache(lens, 32, 2, 64, 15)
    c.ks = c.ks / size
    c.handle = c.to(cuda_device)
    q = (size * torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(1))).to(TYPES[kind])
    got = run(c, q.to(cuda_device), kind, lens, cuda_device)
    check(got, reference(c, q, lens), c, lens, kind)


def test_a_page_marked_as_not_finite_reaches_its_sequence_alone(cuda_device):
    lens = [100, 100, 15]
    c = Cache(lens, 16, 2, 64, 16)
    c.vs[c.table[0, 2].long(), 1] = float("nan")
    c.ks[c.table[1, 6].long(), 0] = float("nan")
    c.handle = c.to(cuda_device)
    q = torch.randn(3, 4, 64, device=cuda_device)
    got = run(c, q, K.F32, lens, cuda_device)
    nan = torch.isnan(got).all(2)
    assert nan.tolist() == [[False, False, True, True], [True, True, False, False], [False] * 4]
    assert not torch.isnan(run(c, q, K.F32, [32, 96, 15], cuda_device)).any()  # before those pages
    assert (torch.isnan(got).any(2) == nan).all()


def test_lengths_and_pages_out_of_range_are_flagged(cuda_device):
    lens = [50, 50, 50, 50]
    c = Cache(lens, 16, 1, 64, 17)
    c.table[2, 1] = c.n_pages
    c.handle = c.to(cuda_device)
    q = torch.randn(4, 2, 64, device=cuda_device)
    got = run(c, q, K.F32, [-1, 65, 50, 50], cuda_device)
    assert int(c.dev["status"]) == -1
    assert (got[:2] == 0).all() and torch.isnan(got[2]).all() and torch.isfinite(got[3]).all()
    assert torch.equal(run(c, q, K.F32, [50, 50, 16, 50], cuda_device)[3], got[3])


def test_workspace_too_small(cuda_device):
    c = make([16], 16, 1, 64, 18, cuda_device)
    q = torch.zeros(1, 1, 64, device=cuda_device)
    with pytest.raises(EngineError, match="needed"):
        run(c, q, K.F32, [16], cuda_device, work=torch.zeros(64, dtype=torch.uint8, device=cuda_device))


def test_offsets_past_32_bits(cuda_device):
    """Pages on both sides of 2^32 bytes of codes."""
    dev, hd, page, n_kv = cuda_device, 128, 64, 8
    n_pages = (1 << 32) // (page * n_kv * hd) + 4
    k, v = (torch.zeros(n_pages, n_kv, page, hd, dtype=torch.int8, device=dev) for _ in "kv")
    ks, vs = torch.zeros(2, n_pages, n_kv, device=dev).unbind(0)
    small = Cache([100], page, n_kv, hd, 19, extra=0)
    small.handle = small.to(dev)
    table = torch.tensor([[n_pages - 1, 1]], dtype=torch.int32, device=dev)
    for i in range(2):
        p = int(small.table[0, i])
        for big, s in ((k, "k"), (v, "v"), (ks, "ks"), (vs, "vs")):
            big[int(table[0, i])] = small.dev[s][p]
    q = torch.randn(1, 16, hd, device=dev).half()
    want = run(small, q, K.F16, [100], dev)
    cache = K.Kv8Cache(k, v, ks, vs, table, None, n_pages, page, n_kv, hd, 1, 2)
    work = torch.zeros(cache.attn_workspace_bytes(16), dtype=torch.uint8, device=dev)
    out = torch.empty_like(want)
    cache.attn(q, 16 * hd, K.F16, torch.tensor([100], dtype=torch.int32, device=dev), 16, out, work, work.numel())
    assert torch.equal(out, want)


def test_two_streams_and_graphs(cuda_device):
    """Two captured graphs with a workspace each, replayed at once on two streams."""
    dev, lens = cuda_device, [4000, 100, 900]
    c = make(lens, 32, 4, 128, 20, dev)
    qs = [torch.randn(3, 16, 128, device=dev).bfloat16() for _ in range(2)]
    want = [run(c, q, K.BF16, lens, dev) for q in qs]
    d_len = torch.tensor(lens, dtype=torch.int32, device=dev)
    streams, graphs, outs, works = [], [], [], []
    for q in qs:
        out, work = torch.zeros_like(want[0]), torch.zeros(c.handle.attn_workspace_bytes(16), dtype=torch.uint8, device=dev)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.handle.attn(q, 16 * 128, K.BF16, d_len, 16, out, work, work.numel(), torch.cuda.current_stream().cuda_stream)
        streams.append(torch.cuda.Stream())
        graphs.append(graph)
        outs.append(out)
        works.append(work)
    for _ in range(20):
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out, w)


@pytest.mark.parametrize("kind", [K.F16, K.BF16, K.F32])
def test_scales_below_the_normal_range(cuda_device, kind):
    """A cache that the caller filled may hold a page whose scale is subnormal: its values are next to nothing."""
    lens, hd = [60, 20], 64
    c = Cache(lens, 16, 2, hd, 21)
    p = c.table[0].long()
    c.vs[p[0]], c.vs[p[2]] = 1e-40, 2.0 ** -149  # the first page, and one behind a normal one
    c.ks[p[2]] = 1e-40
    c.vs[c.table[1, :2].long()] = 1e-40          # a sequence of nothing else
    c.handle = c.to(cuda_device)
    q = (0.7 * torch.randn(2, 4, hd, generator=torch.Generator().manual_seed(22))).to(TYPES[kind])
    got = run(c, q.to(cuda_device), kind, lens, cuda_device)
    check(got, reference(c, q, lens), c, lens, kind)
    # the last is below 127e-40.  fp16: zeros.  bf16, f32: weights as above (2^-10.5 + 2^-16); 2^-126 / l with a sum l of
    # 20 weights of at most 2^8 has steps of 2^-149 (2^-11 relative); the outputs' own steps are 2^-133 and 2^-149
    want = reference(c, q, lens)[1]
    tol = 0 if kind == K.F16 else 2.0 ** -9 * 127e-40 + 2.0 ** -133
    assert ((got[1].cpu().double() - want).abs() <= tol + (kind == K.F16) * want.abs()).all()


WHOLE = [
    # n_heads, n_kv, hd, page, lens
    (2, 1, 128, 16, [40000]),
    (8, 1, 64, 16, [5000, 300]),
    (32, 8, 128, 64, [1000, 2777]),
    (12, 4, 96, 32, [47, 1025]),
]


@pytest.mark.parametrize("kind", [K.F32, K.F16, K.BF16])
@pytest.mark.parametrize("case", WHOLE, ids=[str(i) for i in range(len(WHOLE))])
def test_no_tile_is_lost(cuda_device, case, kind):
    """Each head's output by its norm, which a missing tile of 16 keys or a missing part of a join would exceed (shown for
    the same cases in test_serve_bounds.py)."""
    n_heads, n_kv, hd, page, lens = case
    c, q = whole_inputs(case, TYPES[kind])
    c.handle = c.to(cuda_device)
    got = run(c, q.to(cuda_device), kind, lens, cuda_device)
    for b, n in enumerate(lens):
        k, v = c.values(b, n)
        want, noise = attend_and_noise(q[b:b + 1].double(), k, v, torch.tensor([n]))
        err = (got[b:b + 1].cpu().double() - want).norm(dim=-1)
        assert (err <= norm_bound(want, noise, *roundings(TYPES[kind]))).all(), (b, err)


@pytest.mark.parametrize("size", [1.0, 1e-6, 1e6])
def test_scores_a_step_of_16_apart(cuda_device, size):
    """Scores around 2^27 log2 units, where f32 has steps of 16: the later keys of each sequence lie one step above the earlier
    ones, for sequences whose scores have even and odd last digits."""
    hd, n, first, n_seq = 64, 640, 320, 56
    lens = [n] * n_seq
    c = Cache(lens, 16, 1, hd, 25)
    c.ks[:], c.vs[:] = 1.135e7, size
    c.k[:] = 0
    for b in range(n_seq):
        p = c.table[b].long()
        c.k[p, 0, :, 0] = 127 - b                # 2^27 .. 2^28 units with the first dim of the query
        c.k[p[first // 16:], 0, :, 1] = 64       # and 16 more with its second
        c.v[p[:first // 16]], c.v[p[first // 16:]] = -100, 100
    c.handle = c.to(cuda_device)
    q = torch.zeros(n_seq, 1, hd)
    q[..., 0], q[..., 1] = 1.0, 1.0 / (127 * 65536)  # the smallest step of a query's digits
    got = run(c, q.to(cuda_device), K.F32, lens, cuda_device).cpu() / size
    # a score is rounded to half a step, 8 units: the earlier keys together weigh 2^-(16 - 8) of the later at most
    assert ((got - 100).abs() <= 200 * 2.0 ** -7).all(), got[:, 0, 0]
