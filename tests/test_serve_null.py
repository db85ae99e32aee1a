"""Arrays that a batched serving call does not need may be None in Python, as they may be NULL in C; where it needs
them the library refuses.  CPU only: no call gets as far as a launch, and no address is made up but the cache's,
which no call follows."""
import pytest

from tpt_spark_b200 import kernels as K
from tpt_spark_b200._lib import EngineError

P = 1 << 20


def cache(n_seq, table):
    return K.Kv8Cache(P, P, P, P, table, None, 4, 16, 2, 64, n_seq, 4)


def append(c, n):
    c.append(None, K.F16, None, 256, None, 128, None, 128, 4 if n else 0, None, None, None, None, n, n)


def read(c, n):
    c.read(None, None, n, n, K.F16, P, None)


def attn(c, n):
    c.attn(None, 256, K.F16, None, 4, None, None, 1 << 30)


def packed(n):
    K.attn_packed(None, None, None, None, K.F16, 256, 128, 128, None, None, 1, n, n, n, 4, 2, 64)


def logprobs(n):
    K.logprobs(None, K.F32, n, 100, 100, None, None, None, 0, None, None)


def test_nothing_to_do():
    for call in (append, read, attn):
        call(cache(0, None), 0)
    packed(0)
    logprobs(0)


@pytest.mark.parametrize("call", [append, read, attn])
def test_something_to_do(call):
    with pytest.raises(EngineError, match="null"):
        call(cache(1, P), 4)
    with pytest.raises(EngineError, match="null cache"):
        call(cache(1, None), 4)


def test_rows():
    with pytest.raises(EngineError, match="null"):
        packed(4)
    with pytest.raises(EngineError, match="bad logits"):
        logprobs(4)
