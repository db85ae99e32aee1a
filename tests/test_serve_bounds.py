"""The bounds that the attention operators are held to on the GPU are tight enough to see lost keys: a 64-bit form that
leaves some out, on the same inputs, exceeds them.  CPU only."""
import pytest

torch = pytest.importorskip("torch")

from kv8_ref import attend_and_noise, norm_bound, roundings, whole_inputs  # noqa: E402

WHOLE = [(2, 1, 128, 16, [40000]), (8, 1, 64, 16, [5000, 300]), (32, 8, 128, 64, [1000, 2777]), (12, 4, 96, 32, [47, 1025])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", WHOLE, ids=[str(i) for i in range(len(WHOLE))])
def test_decode(case, dtype):
    c, q = whole_inputs(case, dtype)
    for b, n in enumerate(case[4]):
        k, v = c.values(b, n)
        args = q[b:b + 1].double(), k, v, torch.tensor([n])
        want, noise = attend_and_noise(*args)
        bound = norm_bound(want, noise, *roundings(dtype))
        last = (n - 1) // 16
        # (of 40000 keys a tile moves a bf16 output by less than its own rounding; a CTA's part of the line is 256 keys)
        keys = 96 if dtype == torch.bfloat16 and n > 10000 else 16
        for tile in sorted({0, last // 3, last // 2, last - 1 if last else 0}):
            without = attend_and_noise(*args, drop=slice(16 * tile, 16 * tile + keys))[0]
            assert ((without - want).norm(dim=-1) > bound).any(), (b, tile)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,n_kv,hd,lq,lk", [(4, 1, 128, 3000, 3000), (3, 1, 64, 400, 5000), (2, 2, 96, 1500, 1500)])
def test_prompts(H, n_kv, hd, lq, lk, dtype):
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(n, h, hd, generator=g).to(dtype).double() for n, h in ((lq, H), (lk, n_kv), (lk, n_kv)))
    rows = torch.arange(lq - 64, lq)  # the longest
    q, limit = q[rows], rows + lk - lq + 1
    want, noise = attend_and_noise(q, k, v, limit)
    eps = torch.finfo(dtype).eps / 2
    bound = norm_bound(want, noise, eps, eps)
    for first, n in ((0, 16), (lk // 2, 16), (lk - 100, 16)):
        without = attend_and_noise(q, k, v, limit, drop=slice(first, first + n))[0]
        assert ((without - want).norm(dim=-1) > bound).all(), (first, n)
