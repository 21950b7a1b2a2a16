"""Refusals of the token operators (embedding, dropout, class log-probabilities). The C
entry points check their arguments before they look at the context or touch the GPU, so
these run without one: every call below passes a NULL context, which is the last thing to
be refused."""
import ctypes as C

import pytest

from rustwood_b200 import _native as N

P = 1 << 20  # a well-aligned address that is never read
F32, BF16, I64 = N.RW_F32, N.RW_BF16, N.RW_I64


def embed(**k):
    a = dict(table=P, table_type=F32, vocab=10, ld_table=8, ids=P, id_type=I64, n=4, d=8, scale=1.0,
             out=P, out_type=F32, ld_out=8)
    a.update(k)
    return N.lib.rw_embed_device(None, *a.values(), None)


def embed_grad(**k):
    a = dict(grad=P, grad_type=F32, ld_grad=8, ids=P, id_type=I64, n=4, d=8, vocab=10, scale=1.0,
             accumulate=0, dtable=P, dtable_type=F32, ld_dtable=8, ws=P, ws_bytes=1 << 30)
    a.update(k)
    return N.lib.rw_embed_grad_device(None, *a.values(), None)


def dropout(**k):
    a = dict(x=P, type=F32, rows=2, cols=8, ld_x=8, p=0.5, seed=1, sequence=2, y=P, ld_y=8)
    a.update(k)
    return N.lib.rw_dropout_device(None, *a.values(), None)


def logprobs(**k):
    a = dict(x=P, type=F32, n=2, classes=8, ld_x=8, scale=1.0, targets=P, target_type=I64, top_k=2,
             row_max=P, log_sum=P, lse=P, logp=P, entropy=P, top_logp=P, top_index=P, ws=P,
             ws_bytes=1 << 30)
    a.update(k)
    return N.lib.rw_logprobs_device(None, *a.values(), None)


def logprobs_grad(**k):
    a = dict(x=P, type=F32, n=2, classes=8, ld_x=8, scale=1.0, targets=P, target_type=I64, row_max=P,
             log_sum=P, entropy=P, grad_logp=P, grad_entropy=P, dx=P, ld_dx=8)
    a.update(k)
    return N.lib.rw_logprobs_grad_device(None, *a.values(), None)


NAN, INF = float("nan"), float("inf")
CASES = [
    (embed, dict(table_type=3), "unknown element type"),
    (embed, dict(out_type=-1), "unknown element type"),
    (embed, dict(id_type=2), "unknown id type"),
    (embed, dict(d=1 << 23, ld_table=1 << 23, ld_out=1 << 23), "below 2^23"),
    (embed, dict(table=None), "d_table is NULL"),
    (embed, dict(ids=None), "d_ids is NULL"),
    (embed, dict(out=None), "d_out is NULL"),
    (embed, dict(table=P + 2), "d_table is not aligned"),
    (embed, dict(out=P + 1, out_type=BF16), "d_out is not aligned"),
    (embed, dict(ids=P + 4), "d_ids is not aligned"),
    (embed, dict(ld_table=7), "d_table has a row stride"),
    (embed, dict(ld_out=0), "d_out has a row stride"),
    (embed, dict(n=1 << 40, ld_out=1 << 40), "d_out is too large"),
    (embed_grad, dict(grad_type=9), "unknown element type"),
    (embed_grad, dict(dtable_type=9), "unknown element type"),
    (embed_grad, dict(id_type=-1), "unknown id type"),
    (embed_grad, dict(n=1 << 31), "below 2^31"),
    (embed_grad, dict(vocab=1 << 31), "below 2^31"),
    (embed_grad, dict(d=1 << 23, ld_grad=1 << 23, ld_dtable=1 << 23), "below 2^23"),
    (embed_grad, dict(grad=None), "d_grad is NULL"),
    (embed_grad, dict(ids=None), "d_ids is NULL"),
    (embed_grad, dict(dtable=None), "d_dtable is NULL"),
    (embed_grad, dict(ld_grad=3), "d_grad has a row stride"),
    (embed_grad, dict(ld_dtable=3), "d_dtable has a row stride"),
    (embed_grad, dict(ws=None), "d_workspace is NULL"),
    (embed_grad, dict(ws=P + 128), "not 256-byte aligned"),
    (embed_grad, dict(ws_bytes=8), "8 bytes"),
    (dropout, dict(type=5), "unknown element type"),
    (dropout, dict(p=-0.1), "p is not in"),
    (dropout, dict(p=1.5), "p is not in"),
    (dropout, dict(p=NAN), "p is not in"),
    (dropout, dict(x=None), "d_x is NULL"),
    (dropout, dict(y=None), "d_y is NULL"),
    (dropout, dict(ld_x=4), "d_x has a row stride"),
    (dropout, dict(ld_y=4, y=2 * P), "d_y has a row stride"),
    (dropout, dict(ld_y=16), "in place needs one stride"),
    (logprobs, dict(type=5), "unknown element type"),
    (logprobs, dict(target_type=5), "unknown target type"),
    (logprobs, dict(scale=0.0), "scale"),
    (logprobs, dict(scale=-1.0), "scale"),
    (logprobs, dict(scale=NAN), "scale"),
    (logprobs, dict(scale=INF), "scale"),
    (logprobs, dict(scale=1e-30), "scale"),
    (logprobs, dict(scale=1e30), "scale"),
    (logprobs, dict(classes=1 << 31, ld_x=1 << 31), "below 2^31"),
    (logprobs, dict(top_k=9), "top_k"),
    (logprobs, dict(top_k=33, classes=100, ld_x=100), "top_k"),
    (logprobs, dict(x=None), "d_x is NULL"),
    (logprobs, dict(ld_x=7), "d_x has a row stride"),
    (logprobs, dict(targets=None), "d_targets is NULL"),
    (logprobs, dict(targets=P + 4), "d_targets is not aligned"),
    (logprobs, dict(lse=P + 2), "not aligned"),
    (logprobs, dict(top_index=P + 4), "d_top_index is not aligned"),
    (logprobs_grad, dict(type=5), "unknown element type"),
    (logprobs_grad, dict(target_type=-2), "unknown target type"),
    (logprobs_grad, dict(scale=0.0), "scale"),
    (logprobs_grad, dict(classes=1 << 31), "below 2^31"),
    (logprobs_grad, dict(x=None), "d_x is NULL"),
    (logprobs_grad, dict(dx=None), "d_dx is NULL"),
    (logprobs_grad, dict(ld_x=7), "d_x has a row stride"),
    (logprobs_grad, dict(ld_dx=9), "in place needs one stride"),
    (logprobs_grad, dict(row_max=None), "d_row_max is NULL"),
    (logprobs_grad, dict(log_sum=None), "d_log_sum is NULL"),
    (logprobs_grad, dict(targets=None), "d_targets is NULL"),
    (logprobs_grad, dict(entropy=None), "d_entropy is NULL"),
    (logprobs_grad, dict(grad_logp=P + 2), "not aligned"),
    (embed, dict(), "context is NULL"),
    (embed_grad, dict(), "context is NULL"),
    (dropout, dict(), "context is NULL"),
    (logprobs, dict(), "context is NULL"),
    (logprobs, dict(targets=None, logp=None), "context is NULL"),
    (logprobs, dict(n=0, x=None, targets=None), "context is NULL"),
    (logprobs_grad, dict(), "context is NULL"),
    (logprobs_grad, dict(targets=None, grad_logp=None), "context is NULL"),
    (logprobs_grad, dict(entropy=None, grad_entropy=None), "context is NULL"),
    (logprobs_grad, dict(n=0, x=None, dx=None, row_max=None), "context is NULL"),
    (embed, dict(n=0, ids=None, out=None), "context is NULL"),
    (embed, dict(vocab=0, table=None), "context is NULL"),
    (embed_grad, dict(n=0, ids=None, grad=None), "context is NULL"),
    (dropout, dict(rows=0, x=None, y=None), "context is NULL"),
]


@pytest.mark.parametrize("call,change,message", CASES,
                         ids=lambda v: v.__name__ if callable(v) else None)
def test_bad_arguments_are_refused(call, change, message):
    assert call(**change) == -1
    got = N.lib.rw_last_error(None).decode()
    assert message in got and got.startswith("rw_" + call.__name__ + "_device: "), got


def test_workspace_queries():
    b = C.c_uint64(7)
    assert N.lib.rw_embed_grad_workspace(None, 0, 8, 10, C.byref(b)) == 0 and b.value == 0
    for vocab in (10, 1000):  # summed in tables, and by sorting
        assert N.lib.rw_embed_grad_workspace(None, 10000, 8, vocab, C.byref(b)) == 0 and b.value > 0
    assert N.lib.rw_embed_grad_workspace(None, 1 << 31, 8, 10, C.byref(b)) == -1 and b.value == 0
    assert N.lib.rw_embed_grad_workspace(None, 1, 1, 1, None) == -1
    for bad in ((5, 2, 100), (F32, 33, 100), (F32, 2, 1 << 31)):
        assert N.lib.rw_logprobs_workspace(None, 4, bad[2], bad[0], bad[1], C.byref(b)) == -1
    assert N.lib.rw_logprobs_workspace(None, 4, 100, F32, 2, C.byref(b)) == 0
    assert N.lib.rw_logprobs_workspace(None, 4, 100, F32, 2, None) == -1


class _Ctx:  # what the tensor checks need of a context
    gpu, h = 0, None


def test_tensor_arguments_are_refused():
    import torch

    from rustwood_b200 import tokens
    ids, x = torch.zeros(4, dtype=torch.int64), torch.zeros(4, 8)
    with pytest.raises(ValueError, match="is on cpu"):
        tokens.embed(_Ctx, x, ids)
    with pytest.raises(ValueError, match="not .vocab..d."):
        tokens.embed(_Ctx, torch.zeros(8), ids)
    with pytest.raises(TypeError, match="not a torch tensor"):
        tokens.embed(_Ctx, [[1.0]], ids)
    with pytest.raises(ValueError, match="is on cpu"):
        tokens.embed_grad(_Ctx, x, ids, 10)
    with pytest.raises(ValueError, match="is on cpu"):
        tokens.dropout(_Ctx, x, 0.5, 1)
    with pytest.raises(ValueError, match="is on cpu"):
        tokens.logprobs(_Ctx, x, ids)
    with pytest.raises(ValueError, match="is on cpu"):
        tokens.logprobs_grad(_Ctx, x, ids, x[:, 0], x[:, 0], None, x[:, 0])
