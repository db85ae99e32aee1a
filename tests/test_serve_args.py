"""What the batched serving entry points refuse before anything reaches a GPU.  CPU only: every pointer is
made up, and a call that got as far as a launch would fail with another code."""
import ctypes

import pytest

from tpt_spark_b200 import _lib
from tpt_spark_b200 import kernels as K
from tpt_spark_b200._lib import EngineError

P = 1 << 20  # a 16-byte aligned address that is never read
ARG, UNSUPPORTED = -1, -5


def cache(**kw):
    a = dict(d_k=P, d_v=P, d_k_scale=P, d_v_scale=P, d_table=P, d_status=None, n_pages=4, page=16, n_kv=2, head_dim=64, n_seq=1,
             max_pages=4)
    a.update(kw)
    return K.Kv8Cache(**a)


def rope(**kw):
    a = dict(d_cos=P, d_sin=P, rows=64, dim=64)
    a.update(kw)
    return K.Rope(**a)


def append(c=None, **kw):
    a = dict(rope=rope(), type_=K.F16, d_q=P, q_stride=256, d_k=P, k_stride=128, d_v=P, v_stride=128, n_heads=4, d_q_out=P,
             d_k_out=P, d_cu=P, d_start=P, n_tokens=4, max_new=4)
    a.update(kw)
    (c or cache()).append(**a)


def read(c=None, **kw):
    a = dict(d_cu=P, d_start=P, n_tokens=4, max_rows=4, type_=K.F16, d_k_out=P, d_v_out=P)
    a.update(kw)
    (c or cache()).read(**a)


def refused(code, call, *args, **kw):
    with pytest.raises(EngineError) as e:
        call(*args, **kw)
    assert e.value.code == code and len(str(e.value)) > 8


@pytest.mark.parametrize("call", [append, read])
@pytest.mark.parametrize("code,kw", [
    (UNSUPPORTED, dict(head_dim=80)), (UNSUPPORTED, dict(head_dim=256)), (UNSUPPORTED, dict(page=8)),
    (UNSUPPORTED, dict(page=128)), (ARG, dict(n_pages=0)), (ARG, dict(n_kv=0)), (ARG, dict(max_pages=0)), (ARG, dict(n_seq=-1)),
    (ARG, dict(d_k=0)), (ARG, dict(d_table=0)), (ARG, dict(d_v_scale=0)), (ARG, dict(d_k=P + 8)), (ARG, dict(max_pages=1 << 28))])
def test_caches(call, code, kw):
    refused(code, call, cache(**kw))


@pytest.mark.parametrize("code,kw", [
    (UNSUPPORTED, dict(type_=K.Q8_0)), (ARG, dict(d_k=0)), (ARG, dict(d_cu=0)), (ARG, dict(d_start=0)), (ARG, dict(n_tokens=-1)),
    (ARG, dict(max_new=-1)), (ARG, dict(k_stride=120)), (ARG, dict(v_stride=132)), (ARG, dict(d_v=P + 2)), (ARG, dict(d_q=P + 8)),
    (ARG, dict(q_stride=128)), (ARG, dict(n_heads=3)), (ARG, dict(n_heads=0)), (ARG, dict(d_q=None)), (ARG, dict(d_k_out=P + 4)),
    (ARG, dict(rope=rope(dim=24))), (ARG, dict(rope=rope(dim=80))), (ARG, dict(rope=rope(rows=0))),
    (ARG, dict(rope=rope(d_cos=P + 4))), (ARG, dict(rope=rope(d_sin=0)))])
def test_appends(code, kw):
    refused(code, append, **kw)


@pytest.mark.parametrize("code,kw", [(UNSUPPORTED, dict(type_=2)), (ARG, dict(d_cu=0)), (ARG, dict(n_tokens=-4)),
                                     (ARG, dict(max_rows=-1)), (ARG, dict(d_k_out=P + 8)), (ARG, dict(d_start=0))])
def test_reads(code, kw):
    refused(code, read, **kw)


def attn(c=None, **kw):
    a = dict(d_q=P, q_stride=256, type_=K.F16, d_len=P, n_heads=4, d_out=P, d_workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    (c or cache()).attn(**a)


@pytest.mark.parametrize("code,kw", [
    (UNSUPPORTED, dict(type_=14)), (ARG, dict(d_q=0)), (ARG, dict(d_len=0)), (ARG, dict(d_out=0)), (ARG, dict(d_workspace=0)),
    (ARG, dict(n_heads=3)), (ARG, dict(n_heads=0)), (ARG, dict(q_stride=255)), (ARG, dict(q_stride=260)), (ARG, dict(d_q=P + 8)),
    (ARG, dict(d_out=P + 2)), (ARG, dict(d_workspace=P + 4))])
def test_attentions(code, kw):
    refused(code, attn, **kw)


def test_attention_caches():
    refused(UNSUPPORTED, attn, cache(head_dim=80))
    refused(ARG, attn, cache(n_seq=1 << 30))
    refused(ARG, cache().attn_workspace_bytes, 5)


def packed(**kw):
    a = dict(d_q=P, d_k=P, d_v=P, d_out=P, type_=K.F16, q_stride=256, k_stride=128, v_stride=128, d_cu_q=P, d_cu_k=P, n_seq=1,
             n_q=10, n_k=10, max_q=10, n_heads=4, n_kv=2, head_dim=64)
    a.update(kw)
    K.attn_packed(**a)


@pytest.mark.parametrize("code,kw", [
    (UNSUPPORTED, dict(type_=K.F32)), (UNSUPPORTED, dict(head_dim=256)), (UNSUPPORTED, dict(n_heads=258, q_stride=1 << 20)),
    (ARG, dict(n_heads=3)), (ARG, dict(n_kv=0)), (ARG, dict(n_heads=0)), (ARG, dict(n_seq=-1)), (ARG, dict(n_q=-1)),
    (ARG, dict(n_k=-1)), (ARG, dict(max_q=-1)), (ARG, dict(n_k=2 ** 31 - 100)), (ARG, dict(d_q=0)), (ARG, dict(d_cu_k=0)),
    (ARG, dict(d_out=P + 16)), (ARG, dict(q_stride=248)), (ARG, dict(k_stride=130)), (ARG, dict(d_v=P + 2))])
def test_prompts(code, kw):
    refused(code, packed, **kw)


def test_nothing_to_do_is_no_error():
    packed(n_seq=0)
    packed(n_q=0)
    attn(cache(n_seq=0))
    append(n_tokens=0)
    append(max_new=0)
    append(cache(n_seq=0))
    read(n_tokens=0)
    read(d_k_out=None, d_v_out=None)
    logprobs(rows=0)


def test_empty_arrays_may_be_null():
    append(n_tokens=0, d_q=None, d_k=0, d_v=0, d_q_out=None, d_k_out=None, n_heads=0)
    append(n_tokens=0, d_q=None, d_k=0, d_v=0)
    append(cache(n_seq=0, d_table=0), d_cu=0, d_start=0)
    read(n_tokens=0, d_k_out=None, d_v_out=P)
    attn(cache(n_seq=0, d_table=0), d_q=0, d_len=0, d_out=0, d_workspace=0)
    packed(n_q=0, d_q=0, d_out=0)
    logprobs(rows=0, d_logits=0, d_token=None, d_logprob=P, d_top_id=None)


def logprobs(**kw):
    a = dict(d_logits=P, type_=K.F32, rows=2, vocab=100, row_stride=100, d_token=P, d_logprob=P, d_entropy=P, n_top=5, d_top_id=P,
             d_top_logprob=P)
    a.update(kw)
    K.logprobs(**a)


@pytest.mark.parametrize("code,kw", [
    (UNSUPPORTED, dict(type_=K.Q4_K)), (ARG, dict(d_logits=0)), (ARG, dict(rows=-1)), (ARG, dict(vocab=0)),
    (ARG, dict(row_stride=99)), (ARG, dict(n_top=33)), (ARG, dict(n_top=-1)), (ARG, dict(n_top=5, vocab=4)),
    (ARG, dict(d_top_id=None)), (ARG, dict(d_token=None)), (ARG, dict(d_logprob=None)), (ARG, dict(d_logits=P + 2))])
def test_logprobs(code, kw):
    refused(code, logprobs, **kw)


def test_descriptors_match_the_header_layout():
    assert ctypes.sizeof(_lib.Kv8C) == 6 * 8 + 6 * 4 and ctypes.sizeof(_lib.RopeC) == 32
