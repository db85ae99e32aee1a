"""The paged 8-bit KV cache: tptc_kv8_append and tptc_kv8_read against 64-bit forms."""
import pytest

torch = pytest.importorskip("torch")

from kv8_ref import TYPES, Cache, rope_tables, rotate  # noqa: E402
from tpt_spark_b200 import kernels as K  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of f32, relative


def make_qkv(total, n_heads, n_kv, hd, dtype, seed, pad=16):
    """q, k and v as slices of one fused buffer with a gap behind each row."""
    g = torch.Generator().manual_seed(seed)
    width = (n_heads + 2 * n_kv) * hd + pad
    buf = torch.randn(total, width, generator=g).to(dtype)
    return buf, width


def split(buf, n_heads, n_kv, hd):
    x = buf[:, : (n_heads + 2 * n_kv) * hd].double().view(len(buf), -1, hd)
    return x[:, :n_heads], x[:, n_heads:n_heads + n_kv], x[:, n_heads + n_kv:]


def call(cache, rope, kind, buf, width, n_heads, n_kv, hd, q_out, k_out, cu, start, total, most, stream=None):
    at, e = buf.data_ptr(), buf.element_size() * hd
    cache.append(rope, kind, at if n_heads else None, width, at + n_heads * e, width, at + (n_heads + n_kv) * e, width,
                 n_heads, q_out, k_out, cu, start, total, most, stream)


def check_store(was, codes, scale, new, rows_of):
    """Codes and scales after an append, from what was there and the new f64 rows of each (page, first row)."""
    was_codes, was_scale = was
    touched = torch.zeros(len(codes), dtype=torch.bool)
    for page, off, x in rows_of(new):
        touched[page] = True
        n = len(x)
        top = x.abs().amax((0, 2))
        s = scale[page].double()
        want = torch.maximum(was_scale[page].double(), top / 127) if off else top / 127
        # a: three roundings of the rotation, |x0 c| + |x1 s| <= sqrt(2) a; 1/127 and its product: one each
        assert ((s - want).abs() <= 8 * U * want).all()
        c = codes[page].double()
        # x / s: the errors above against up to 127 steps, then half a step of rounding
        assert ((c[:, off:off + n].transpose(0, 1) - x / s[:, None]).abs() <= 0.5 + 127 * 12 * U).all()
        if off:
            r = was_scale[page].double() / s
            old = was_codes[page, :, :off].double()
            assert ((c[:, :off] - old * r[:, None, None]).abs() <= 0.5 + 127 * 4 * U).all()
            same = was_scale[page] == scale[page]
            assert torch.equal(codes[page, same, :off], was_codes[page, same, :off])
        assert torch.equal(codes[page, :, off + n:], was_codes[page, :, off + n:])  # rows behind: as they were
    assert torch.equal(codes[~touched], was_codes[~touched]) and torch.equal(scale[~touched], was_scale[~touched])


CASES = [
    # n_heads, n_kv, hd, page, type, rot, halves, start, new
    (8, 2, 128, 16, K.F16, 128, False, [0], [1]),
    (8, 2, 128, 16, K.BF16, 128, True, [5, 15, 16, 31, 0], [1, 1, 1, 1, 1]),
    (4, 4, 64, 16, K.F32, 64, False, [3, 0, 40], [30, 0, 17]),
    (4, 4, 64, 32, K.F16, 32, True, [31, 33, 0, 7], [2, 64, 1, 0]),
    (4, 1, 64, 64, K.BF16, 64, True, [10, 64], [200, 65]),
    (12, 4, 96, 16, K.F16, 96, True, [0, 9], [33, 16]),
    (12, 4, 96, 32, K.F32, 48, False, [100, 0], [1, 31]),
    (6, 2, 96, 64, K.BF16, 32, True, [63, 65, 0], [1, 129, 64]),
    (28, 4, 128, 32, K.F32, 128, True, [11, 0], [70, 5]),
    (16, 1, 128, 64, K.F16, 16, False, [17, 0, 300], [129, 63, 1]),
    (2, 2, 128, 64, K.F16, 0, False, [1], [300]),  # no rotation
    (0, 3, 128, 16, K.BF16, 128, False, [0, 21], [40, 3]),  # no queries
    # tokens to decode beside prompts that are far longer
    (2, 1, 64, 16, K.F16, 64, True, [i % 37 for i in range(41)], [400 if i == 17 else i % 3 for i in range(41)]),
    (4, 2, 128, 32, K.BF16, 128, False, [i % 70 for i in range(300)], [600 if i in (0, 299) else 1 for i in range(300)]),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_append(cuda_device, case):
    n_heads, n_kv, hd, page, kind, rot, halves, start, new = case
    dtype, dev, total = TYPES[kind], cuda_device, sum(new)
    c = Cache([s + n for s, n in zip(start, new)], page, n_kv, hd, seed=1)
    cache = c.to(dev)
    lead, tail = 2, 3  # rows of no sequence, before and behind
    buf, width = make_qkv(lead + total + tail, n_heads, n_kv, hd, dtype, seed=2)
    cu = torch.tensor([0] + new).cumsum(0) + lead
    cos, sin = rope_tables(max(s + n for s, n in zip(start, new)), rot) if rot else (None, None)
    rope = K.Rope(cos.to(dev), sin.to(dev), len(cos), rot, halves) if rot else None
    q_out = torch.full((lead + total + tail, n_heads, hd), 7.0, dtype=dtype, device=dev) if n_heads else None
    k_out = torch.full((lead + total + tail, n_kv, hd), 7.0, dtype=dtype, device=dev)
    call(cache, rope, kind, buf.to(dev), width, n_heads, n_kv, hd, q_out, k_out, cu.int().to(dev),
         torch.tensor(start, dtype=torch.int32, device=dev), lead + total + tail, max(new))
    torch.cuda.synchronize()
    assert int(c.dev["status"]) == 0

    pos = torch.cat([torch.arange(s, s + n) for s, n in zip(start, new)])
    rows = slice(lead, lead + total)
    q, k, v = (x[rows] for x in split(buf, n_heads, n_kv, hd))
    if rot:
        size = k.abs().amax((1, 2)) * 0
        q_raw, k_raw = q, k
        q, k = (rotate(x, cos[pos], sin[pos], rot, halves) for x in (q, k))
        # two products and a sum, each rounded: 3 U of |x0 c| + |x1 s|; then the output's rounding
        for got, want, raw in ((q_out, q, q_raw), (k_out, k, k_raw)):
            if got is not None and want.numel():
                eps = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0
                slack = 3 * U * 1.5 * raw.abs().amax((1, 2), keepdim=True)
                assert ((got[rows].cpu().double() - want).abs() <= eps * (want.abs() + slack) + slack + 2.0 ** -25).all()
        del size
    else:
        assert torch.equal(k_out[rows].cpu().double(), k)
        assert torch.equal(q_out[rows].cpu().double(), q)
    for out in (q_out, k_out):
        if out is not None:
            assert (out[:lead] == 7).all() and (out[lead + total:] == 7).all()

    def rows_of(x):
        at = 0
        for b, (s, n) in enumerate(zip(start, new)):
            done = 0
            while done < n:
                p, off = divmod(s + done, page)
                take = min(page - off, n - done)
                yield int(c.table[b, p]), off, x[at + done:at + done + take]
                done += take
            at += n

    check_store((c.k, c.ks), c.dev["k"].cpu(), c.dev["ks"].cpu(), k, rows_of)
    check_store((c.v, c.vs), c.dev["v"].cpu(), c.dev["vs"].cpu(), v, rows_of)


def test_scales_that_grow_and_pages_that_come_back(cuda_device):
    """A larger value rescales the page's earlier rows; a smaller one leaves them; a page that a new
    sequence starts again forgets its old scale."""
    dev, hd, page = cuda_device, 64, 16
    c = Cache([32], page, 1, hd, seed=3)
    cache = c.to(dev)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)

    def put(pos, value):
        x = torch.full((1, 1, hd), value, device=dev)
        cache.append(None, K.F32, None, 0, x, hd, x, hd, 0, None, None, cu,
                     torch.tensor([pos], dtype=torch.int32, device=dev), 1, 1)
        torch.cuda.synchronize()
        p = int(c.table[0, pos // page])
        return c.dev["k"][p, 0].cpu(), float(c.dev["ks"][p, 0])

    codes, s = put(0, 1.0)
    assert (codes[0] == 127).all() and abs(s * 127 - 1) < 4 * U
    codes, s = put(1, 0.5)
    assert (codes[0] == 127).all() and (codes[1] == 64).all()  # 63.5 to even
    codes, s = put(2, -4.0)
    assert (codes[0] == 32).all() and (codes[1] == 16).all() and (codes[2] == -127).all()  # 31.75, 16
    codes, s = put(0, 0.25)
    assert (codes[0] == 127).all() and abs(s * 127 - 0.25) < U


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_that_are_not_finite_mark_their_page(cuda_device, bad):
    dev, hd, page = cuda_device, 128, 16
    c = Cache([32], page, 2, hd, seed=4)
    cache = c.to(dev)
    x = torch.randn(20, 2, hd, device=dev).bfloat16()
    y = x.clone()
    y[3, 1, 100] = bad
    cu = torch.tensor([0, 20], dtype=torch.int32, device=dev)
    start = torch.zeros(1, dtype=torch.int32, device=dev)
    cache.append(None, K.BF16, None, 0, x, 2 * hd, y, 2 * hd, 0, None, None, cu, start, 20, 20)
    one = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    p0, p1 = (int(p) for p in c.table[0, :2])
    assert torch.isnan(c.dev["vs"][p0]).tolist() == [False, True]
    assert not torch.isnan(c.dev["vs"][p1]).any() and not torch.isnan(c.dev["ks"][[p0, p1]]).any()
    # the mark stays while the page's earlier rows do
    cache.append(None, K.BF16, None, 0, x, 2 * hd, x, 2 * hd, 0, None, None, one, start + 5, 20, 1)
    assert torch.isnan(c.dev["vs"][p0]).tolist() == [False, True]
    cache.append(None, K.BF16, None, 0, x, 2 * hd, x, 2 * hd, 0, None, None, one, start, 20, 1)
    assert not torch.isnan(c.dev["vs"][p0]).any()


def test_zeros_and_tiny_values(cuda_device):
    dev, hd = cuda_device, 64
    c = Cache([16], 16, 1, hd, seed=5)
    cache = c.to(dev)
    x = torch.full((2, 1, hd), 1e-40, device=dev)
    cu = torch.tensor([0, 2], dtype=torch.int32, device=dev)
    cache.append(None, K.F32, None, 0, torch.zeros_like(x), hd, x, hd, 0, None, None, cu, cu[:1], 2, 2)
    out = torch.full((2, 2, 1, hd), 3.0, device=dev)
    cache.read(cu, cu[:1], 2, 2, K.F32, out[0], out[1])
    assert (out == 0).all()


def test_rotating_in_place(cuda_device):
    dev, hd, n = cuda_device, 128, 37
    c = Cache([n], 16, 2, hd, seed=6)
    cos, sin = (t.to(dev) for t in rope_tables(n, hd))
    q, k = torch.randn(n, 8, hd, device=dev).half(), torch.randn(n, 2, hd, device=dev).half()
    cu, start = torch.tensor([0, n], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    for halves in (False, True):
        rope = K.Rope(cos, sin, n, hd, halves)
        want_q, want_k = torch.empty_like(q), torch.empty_like(k)
        c.to(dev).append(rope, K.F16, q, 8 * hd, k, 2 * hd, k, 2 * hd, 8, want_q, want_k, cu, start, n, n)
        a, b = q.clone(), k.clone()
        c.to(dev).append(rope, K.F16, a, 8 * hd, b, 2 * hd, k, 2 * hd, 8, a, b, cu, start, n, n)
        assert torch.equal(a, want_q) and torch.equal(b, want_k)


@pytest.mark.parametrize("kind", [K.F32, K.F16, K.BF16])
@pytest.mark.parametrize("hd,page,n_kv", [(64, 16, 5), (96, 32, 3), (128, 64, 9), (128, 16, 1)])
def test_read(cuda_device, kind, hd, page, n_kv):
    dev, start, n = cuda_device, [0, 13, 65, 4, 7], [1, 100, 64, 0, 9]
    c = Cache([a + b for a, b in zip(start, n)], page, n_kv, hd, seed=7)
    cache = c.to(dev)
    total = sum(n)
    cu = torch.tensor([0] + n).cumsum(0).int().to(dev)
    out = torch.full((2, total + 4, n_kv, hd), 9.0, dtype=TYPES[kind], device=dev)
    cache.read(cu, torch.tensor(start, dtype=torch.int32, device=dev), total + 4, 128, kind, out[0], out[1])
    want = [torch.cat(x) for x in zip(*(c.values(b, m, s) for b, (s, m) in enumerate(zip(start, n))))]
    for got, w in zip(out.cpu(), want):
        assert torch.equal(got[:total], w.float().to(TYPES[kind]))  # code * scale is rounded to f32, then to the type
        assert (got[total:] == 9).all()
    only = torch.full_like(out[1], 9.0)
    cache.read(cu, torch.tensor(start, dtype=torch.int32, device=dev), total + 4, 128, kind, None, only)
    assert torch.equal(only, out[1]) and int(c.dev["status"]) == 0


@pytest.mark.parametrize("bad", [None, 0, 150, 299])
def test_read_of_very_different_lengths(cuda_device, bad):
    """One long sequence among 300 short ones; then one of them with positions behind its table."""
    dev, hd, page, n_kv = cuda_device, 64, 16, 2
    n = [900 if i == 70 else i % 4 + (i in (0, 299)) for i in range(300)]
    n[150] = 2
    start = [(i * 13) % 50 for i in range(300)]
    c = Cache([a + b for a, b in zip(start, n)], page, n_kv, hd, seed=17)
    cache, total = c.to(dev), sum(n)
    cu = torch.tensor([0] + n).cumsum(0)
    begin = torch.tensor(start, dtype=torch.int32)
    if bad is not None:
        begin[bad] = c.max_pages * page - 1 + (n[bad] == 1)
    out = torch.full((2, total + 4, n_kv, hd), 9.0, device=dev)
    cache.read(cu.int().to(dev), begin.to(dev), total + 4, 900, K.F32, out[0], out[1])
    torch.cuda.synchronize()
    assert int(c.dev["status"]) == (0 if bad is None else -1)
    want = [torch.cat(x).float() for x in zip(*(c.values(b, m, s) for b, (s, m) in enumerate(zip(start, n))))]
    for got, w in zip(out.cpu(), want):
        if bad is not None:
            w[cu[bad]:cu[bad + 1]] = 9
        assert torch.equal(got[:total], w) and (got[total:] == 9).all()


BAD = {
    "page id": dict(table=10 ** 6), "negative page id": dict(table=-1), "negative start": dict(start=-1),
    "behind the table": dict(start=46), "more rows than said": dict(most=3), "offsets past the rows": dict(cu=99),
    "offsets that descend": dict(cu=-2), "rope rows": dict(rows=4),
}


@pytest.mark.parametrize("what", BAD)
def test_bad_indices_are_flagged_and_touch_nothing(cuda_device, what):
    """One of two sequences is wrong: it is left out and flagged, the other is served."""
    bad, dev, hd, n = BAD[what], cuda_device, 64, 5
    c = Cache([40, 40], 16, 1, hd, seed=8)
    if "table" in bad:
        c.table[1, 0] = bad["table"]
    cache = c.to(dev)
    cu = torch.tensor([0, 3, 8], dtype=torch.int32)
    start = torch.tensor([0, bad.get("start", 0)], dtype=torch.int32)
    if "cu" in bad:
        cu[2] = bad["cu"]
    cos, sin = (t.to(dev) for t in rope_tables(bad.get("rows", 48), hd))
    x = torch.randn(8, 1, hd, device=dev)
    out = torch.full_like(x, 5.0)
    most = bad.get("most", n)
    cache.append(K.Rope(cos, sin, len(cos), hd), K.F32, None, 0, x, hd, x, hd, 0, None, out, cu.to(dev), start.to(dev), 8, most)
    torch.cuda.synchronize()
    assert int(c.dev["status"]) == -1
    good = int(c.table[0, 0])
    others = [p for p in range(c.n_pages) if p != good]
    assert torch.equal(c.dev["k"].cpu()[others], c.k[others]) and torch.equal(c.dev["vs"].cpu()[others], c.vs[others])
    assert not torch.equal(c.dev["k"].cpu()[good, 0, :3], c.k[good, 0, :3])
    if what != "rope rows":
        c.dev["status"].zero_()
        out = torch.full((2, 8, 1, hd), 5.0, device=dev)
        cache.read(cu.to(dev), start.to(dev), 8, most, K.F32, out[0], out[1])
        torch.cuda.synchronize()
        assert int(c.dev["status"]) == -1 and (out[:, 3:] == 5).all() and (out[:, :3] != 5).any()


def test_offsets_past_32_bits(cuda_device):
    """A cache whose codes pass 2^31 bytes: the last page is reached, and nothing near 2^32 wraps."""
    dev, hd, page, n_kv = cuda_device, 128, 64, 8
    n_pages = (1 << 32) // (page * n_kv * hd) + 2
    k = torch.zeros(n_pages * n_kv * page * hd, dtype=torch.int8, device=dev)
    v = torch.zeros_like(k)
    ks, vs = torch.zeros(2, n_pages, n_kv, device=dev).unbind(0)
    table = torch.tensor([[n_pages - 1]], dtype=torch.int32, device=dev)
    cache = K.Kv8Cache(k, v, ks, vs, table, None, n_pages, page, n_kv, hd, 1, 1)
    x = torch.randn(64, n_kv, hd, device=dev)
    cu, start = torch.tensor([0, 64], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    cache.append(None, K.F32, None, 0, x, n_kv * hd, -x, n_kv * hd, 0, None, None, cu, start, 64, 64)
    out = torch.empty(2, 64, n_kv, hd, device=dev)
    cache.read(cu, start, 64, 64, K.F32, out[0], out[1])
    step = x.abs().amax((0, 2)) / 127
    assert ((out[0] - x).abs() <= step[None, :, None] * 0.5001).all()
    assert torch.equal(out[0], -out[1])
    assert not k[: (n_pages - 1) * n_kv * page * hd].any()


def test_on_a_stream_and_in_a_graph(cuda_device):
    dev, hd, n = cuda_device, 128, 50
    c = Cache([n, n], 16, 2, hd, seed=9)
    x = torch.randn(2 * n, 2, hd, device=dev).half()
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=dev)
    start = torch.zeros(2, dtype=torch.int32, device=dev)
    want = c.to(dev)
    want.append(None, K.F16, None, 0, x, 2 * hd, x, 2 * hd, 0, None, None, cu, start, 2 * n, n)
    torch.cuda.synchronize()
    codes, scale = c.dev["k"], c.dev["vs"]
    cache = c.to(dev)
    src, out = torch.zeros_like(x), torch.empty(2, 2 * n, 2, hd, dtype=torch.float16, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        cache.append(None, K.F16, None, 0, src, 2 * hd, src, 2 * hd, 0, None, None, cu, start, 2 * n, n, stream=st)
        cache.read(cu, start, 2 * n, n, K.F16, out[0], out[1], stream=st)
    src.copy_(x)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.dev["k"], codes) and torch.equal(c.dev["vs"], scale) and torch.equal(out[0], out[1])


@pytest.mark.parametrize("kind", [K.F32, K.BF16])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_a_page_that_fills_row_by_row(cuda_device, page, kind):
    """Against the values that went in: a row is rounded when it is stored and again each time the scale grows, by at most
    half of the scale of that moment."""
    dev, hd, n_kv = cuda_device, 128, 4
    c = Cache([2 * page], page, n_kv, hd, seed=40)
    cache = c.to(dev)
    g = torch.Generator().manual_seed(41)
    rows = torch.randn(2 * page, n_kv, hd, generator=g).to(TYPES[kind])
    rows[page:] *= torch.linspace(0.2, 3.0, page)[:, None, None].to(TYPES[kind])  # the second page: it grows and grows
    x, one = rows.to(dev), torch.tensor([0, 1], dtype=torch.int32, device=dev)
    bound = torch.zeros(2 * page, n_kv)
    for i in range(2 * page):
        p = int(c.table[0, i // page])
        before = c.dev["vs"][p].cpu() if i % page else torch.zeros(n_kv)
        cache.append(None, kind, None, 0, x[i], n_kv * hd, x[i], n_kv * hd, 0, None, None, one,
                     torch.tensor([i], dtype=torch.int32, device=dev), 1, 1)
        torch.cuda.synchronize()
        now = c.dev["vs"][p].cpu()
        grown = now > before
        first = i - i % page
        bound[first:i] += torch.where(grown, now, 0.0)  # the earlier rows, rounded again
        bound[i] = now
    # half a step each; the product with 1 / s and the quotient of scales: as for one append, 12 U of up to 127 steps
    bound = bound.double() * (0.5 + 127 * 12 * U)
    stored = [torch.stack([c.dev[n][int(c.table[0, i // page]), :, i % page] * c.dev[n + "s"][int(c.table[0, i // page])][:, None]
                           for i in range(2 * page)]).cpu().double() for n in "kv"]
    for got in stored:
        assert ((got - rows.double()).abs().amax(2) <= bound).all()
    # and with all rows at once half a step of the last scale
    cache.append(None, kind, None, 0, x, n_kv * hd, x, n_kv * hd, 0, None, None, one * 2 * page,
                 torch.zeros(1, dtype=torch.int32, device=dev), 2 * page, 2 * page)
    out = torch.empty(2, 2 * page, n_kv, hd, device=dev)
    cache.read(one * 2 * page, torch.zeros(1, dtype=torch.int32, device=dev), 2 * page, 2 * page, K.F32, out[0], out[1])
    scale = c.dev["vs"][c.table[0, :2].long().to(dev)].repeat_interleave(page, 0).cpu().double()
    for got in out.cpu().double():
        assert ((got - rows.double()).abs().amax(2) <= scale * (0.5 + 127 * 12 * U)).all()
