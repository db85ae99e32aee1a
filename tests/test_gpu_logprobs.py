"""tptc_logprobs against torch in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

from tpt_spark_b200 import kernels as K  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {K.F32: torch.float32, K.F16: torch.float16, K.BF16: torch.bfloat16}


def run(x, kind, tokens, n_top, vocab=None, stride=None, stream=None):
    rows, vocab = x.shape[0], vocab or x.shape[1]
    dev = x.device
    lp, ent = torch.full((rows,), 5.0, device=dev), torch.full((rows,), 5.0, device=dev)
    ids = torch.full((rows, n_top), -9, dtype=torch.int32, device=dev)
    top = torch.full((rows, n_top), 5.0, device=dev)
    K.logprobs(x, kind, rows, vocab, stride or x.stride(0), tokens, lp, ent, n_top, ids, top, stream=stream)
    torch.cuda.synchronize()
    return lp.cpu(), ent.cpu(), ids.cpu(), top.cpu()


def check(x, tokens, got, n_top):
    """x: the logits [rows, vocab] on the CPU, finite or -inf."""
    lp, ent, ids, top = got
    y = torch.log_softmax(x.double(), 1)
    order = x.double().sort(dim=1, descending=True, stable=True)[1][:, :n_top]
    assert torch.equal(ids.long(), order)
    # e^d has a relative error of up to (2 + 1.45 |d|) 2^-23 (the scaled argument's rounding and the
    # exponential's own); a term's weight is e^d, and |d| e^d <= 0.37, so log z is off by at most
    # 4 2^-23 and the sums' roundings (few: a tree of 16-element runs) by as much again; x - m and the
    # final difference round once each, relative to |x - m| and |log p|
    tol = 2.0 ** -20 + 2.0 ** -22 * y.abs().clamp(max=1e30)
    want = y.gather(1, tokens.cpu()[:, None].long())[:, 0]

    def close(a, b, t):
        fine = torch.isfinite(b)
        assert torch.equal(fine, torch.isfinite(a)) and torch.equal(a[~fine].double(), b[~fine])
        assert ((a.double() - b).abs()[fine] <= t[fine]).all(), float((a.double() - b).abs()[fine].max())

    close(lp, want, tol.gather(1, tokens.cpu()[:, None].long())[:, 0])
    close(top, y.gather(1, order), tol.gather(1, order))
    p = y.exp()
    h = -torch.where(p > 0, p * y, 0).sum(1)
    # t / z: the same relative errors on a sum of size sum p |x - m|, and log z as above
    size = torch.where(p > 0, p * (x.double() - x.double().amax(1, keepdim=True)).clamp(min=-1e4).abs(), 0).sum(1)
    assert ((ent.double() - h).abs() <= 2.0 ** -20 + 2.0 ** -19 * size + 2.0 ** -22 * h).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,vocab,n_top", [(1, 128256, 20), (3, 32000, 32), (2, 1, 1), (5, 31, 31), (4, 4097, 1),
                                              (40, 50257, 5), (300, 9000, 7), (1, 262145, 32), (80, 32064, 0)])
def test_logprobs(cuda_device, kind, rows, vocab, n_top):
    g = torch.Generator().manual_seed(vocab + rows)
    x = (3 * torch.randn(rows, vocab, generator=g)).to(TYPES[kind])
    tokens = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    tokens[0] = vocab - 1
    check(x, tokens, run(x.to(cuda_device), kind, tokens.to(cuda_device), n_top), n_top)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("offset", [1, 3, 7])
def test_rows_at_any_alignment(cuda_device, kind, offset):
    rows, vocab, stride = 6, 20001, 20011
    g = torch.Generator().manual_seed(offset)
    buf = torch.full((rows * stride + 16,), float("nan"))
    view = buf[offset:offset + rows * stride].view(rows, stride)
    view[:, :vocab] = 2 * torch.randn(rows, vocab, generator=g)
    buf = buf.to(TYPES[kind])
    x = buf[offset:offset + rows * stride].view(rows, stride)[:, :vocab]
    dev = buf.to(cuda_device)
    tokens = torch.arange(rows, dtype=torch.int32) * 3000
    got = run(dev[offset:offset + rows * stride].view(rows, stride), kind, tokens.to(cuda_device), 9, vocab=vocab)
    check(x, tokens, got, 9)


@pytest.mark.parametrize("shape", ["ascending", "descending", "constant", "few values", "spread", "huge"])
@pytest.mark.parametrize("kind", [K.F32, K.BF16])
def test_orders_and_ties(cuda_device, kind, shape):
    vocab = 70000
    i = torch.arange(vocab, dtype=torch.float64)
    x = {"ascending": i / 7000, "descending": -i / 7000, "constant": i * 0 + 1.5, "few values": (i * 7919 % 5),
         "spread": (i * 7919 % vocab) / 3 - 20000, "huge": (i * 7919 % vocab) * 1e30}[shape]
    x = x.to(TYPES[kind])[None].repeat(2, 1)
    tokens = torch.tensor([0, vocab - 1], dtype=torch.int32)
    check(x, tokens, run(x.to(cuda_device), kind, tokens.to(cuda_device), 32), 32)


@pytest.mark.parametrize("rows", [1, 400])
@pytest.mark.parametrize("kind", list(TYPES))
def test_masked_logits(cuda_device, rows, kind):
    vocab = 33000
    g = torch.Generator().manual_seed(5)
    x = torch.randn(rows, vocab, generator=g).to(TYPES[kind])
    x[:, 100:] = -math.inf
    x[:, 32990] = 0.25
    if rows > 1:
        x[1, :] = torch.finfo(TYPES[kind]).min  # masked by the type's lowest value
        x[1, 77] = 1.0
        x[2, :] = torch.finfo(TYPES[kind]).min
        x[3, 1:] = -math.inf  # one token is left
    tokens = torch.full((rows,), 32990, dtype=torch.int32)
    check(x, tokens, run(x.to(cuda_device), kind, tokens.to(cuda_device), 30), 30)


def test_rows_without_a_distribution(cuda_device):
    vocab = 40000
    x = torch.randn(4, vocab)
    x[0] = -math.inf
    x[1, 500], x[1, 39000] = math.nan, math.nan
    x[2, 700] = math.inf
    tokens = torch.tensor([3, 3, 3, vocab], dtype=torch.int32)
    lp, ent, ids, top = run(x.to(cuda_device), K.F32, tokens.to(cuda_device), 4)
    assert torch.isnan(lp).all() and torch.isnan(ent[:3]).all() and torch.isfinite(ent[3])
    assert torch.isnan(top[:3]).all()
    assert ids[0].tolist() == [0, 1, 2, 3] and ids[1, :2].tolist() == [500, 39000] and ids[2, 0] == 700
    assert ids[3].tolist() == x[3].sort(descending=True, stable=True)[1][:4].tolist()
    x = torch.full((1, vocab), math.nan)
    assert run(x.to(cuda_device), K.F32, tokens[:1].to(cuda_device), 32)[2][0].tolist() == list(range(32))


@pytest.mark.parametrize("rows", [1, 300])
def test_many_nan_and_infinite_logits(cuda_device, rows):
    """NaN, then +inf, then the rest, by lowest index -- also where they fill some warps' lists."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(rows, 60000, generator=g)
    x[:, 5000:5040] = math.nan
    x[:, 40000:40003] = math.inf
    x[:, 59990:] = math.nan
    ids = run(x.to(cuda_device), K.F32, torch.zeros(rows, dtype=torch.int32, device=cuda_device), 32)[2]
    assert (ids == torch.arange(5000, 5032)).all()
    x[:, 5020:5040] = 0.0
    ids = run(x.to(cuda_device), K.F32, torch.zeros(rows, dtype=torch.int32, device=cuda_device), 32)[2]
    assert (ids == torch.tensor(list(range(5000, 5020)) + list(range(59990, 60000)) + [40000, 40001])).all()


def test_parts_and_graph_replay(cuda_device):
    """What is not wanted is left out; a captured call replays on new logits, in any number of CTAs per row."""
    dev = cuda_device
    for rows in (1, 30, 70, 400):
        x = torch.randn(rows, 33333, device=dev)
        tokens = torch.randint(0, 33333, (rows,), device=dev, dtype=torch.int32)
        want = run(x, K.F32, tokens, 6)
        src, lp = torch.zeros_like(x), torch.zeros(rows, device=dev)
        ids, top = torch.zeros(rows, 6, dtype=torch.int32, device=dev), torch.zeros(rows, 6, device=dev)
        ent = torch.zeros(rows, device=dev)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            st = torch.cuda.current_stream().cuda_stream
            K.logprobs(src, K.F32, rows, 33333, 33333, tokens, lp, None, 0, None, None, stream=st)
            K.logprobs(src, K.F32, rows, 33333, 33333, None, None, ent, 6, ids, top, stream=st)
        src.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((lp, ent, ids, top), want):
            assert torch.equal(a.cpu(), b)
