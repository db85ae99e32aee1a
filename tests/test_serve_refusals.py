"""Calls of the batched serving entry points that the library refuses because their result would be wrong.
CPU only: every pointer is made up."""
import pytest

from tpt_spark_b200 import kernels as K
from tpt_spark_b200._lib import EngineError

P = 1 << 20
ARG = -1


def cache(**kw):
    a = dict(d_k=P, d_v=P, d_k_scale=P, d_v_scale=P, d_table=P, d_status=None, n_pages=4, page=16, n_kv=2, head_dim=64, n_seq=1,
             max_pages=4)
    a.update(kw)
    return K.Kv8Cache(**a)


def refused(match, call, *args, **kw):
    with pytest.raises(EngineError, match=match) as e:
        call(*args, **kw)
    assert e.value.code == ARG


# queries of 4 heads of 64, keys of 2: without gaps their strides are 256 and 128
@pytest.mark.parametrize("kw", [dict(d_q_out=P, q_stride=512), dict(d_k_out=P, k_stride=512), dict(d_q_out=P, q_stride=264)])
def test_rotation_in_place_of_rows_with_gaps(kw):
    a = dict(rope=None, type_=K.F16, d_q=P, q_stride=256, d_k=P, k_stride=128, d_v=P, v_stride=128, n_heads=4, d_q_out=None,
             d_k_out=None, d_cu=P, d_start=P, n_tokens=4, max_new=4)
    a.update(kw)
    refused("in place", cache().append, **a)


def test_attention_over_more_positions_than_its_sums_hold():
    """A sequence of 2^30 positions is 2^26 tiles of 16 keys; 32 of them pass 31 bits, 31 do not."""
    a = dict(d_q=P, q_stride=256, type_=K.F16, d_len=P, n_heads=4, d_out=P, d_workspace=P, workspace_bytes=1 << 30)
    for c in (cache(n_seq=32, max_pages=1 << 26), cache(n_seq=900, max_pages=1 << 24, page=64), cache(n_seq=16, max_pages=(1 << 27) - 1)):
        refused("positions", c.attn, **a)
        refused("positions", c.attn_workspace_bytes, 4)
    for c in (cache(n_seq=31, max_pages=1 << 26), cache(n_seq=900, max_pages=1 << 25), cache(n_seq=15, max_pages=(1 << 27) - 1)):
        with pytest.raises(EngineError) as e:  # no GPU here: that is as far as an accepted call gets
            c.attn_workspace_bytes(4)
        assert e.value.code != ARG
