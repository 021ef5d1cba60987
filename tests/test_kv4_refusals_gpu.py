"""Attention over 4-bit pages: calls that are refused before anything is launched."""
import pytest
import torch

from braidinfer_amd import kernels as K
from braidinfer_amd.errors import KernelError
from test_kv4_gpu import PAGE, Cache, dev, step_of

pytestmark = pytest.mark.gpu
NQ, NKV, HD = 4, 2, 64


def calls(n):
    """(output, one token of each of n sequences, n tokens of one sequence), as functions of the queries, their stride and the scale."""
    c = Cache([n], NKV, HD)
    c.fill()
    table, cache = c.tensors
    out = torch.full((n, NQ * HD), 9.0, device="cuda", dtype=torch.bfloat16)

    def one(q, stride, scale=0.1):
        K.attention_decode_kv4(q, stride, out, dev(list(c.slots) * n), dev(c.lens * n), table, cache, n, NQ, NKV, HD, PAGE, None, scale, 1)

    def many(q, stride, scale=0.1):
        K.attention_prefill_kv4(q, stride, out, step_of([n], [0])[2], dev(c.slots), dev(c.lens), table, cache, 1, n, NQ, NKV, HD, PAGE, None,
                                scale, 1)
    return out, one, many


def test_queries_that_are_one_row_said_to_be_many():
    n, width = 70, NQ * HD
    out, *both = calls(n)
    row = torch.randn(1, width, device="cuda").bfloat16()
    for call in both:
        for q in (row.expand(n, width), row[:, :1].expand(n, width)):
            with pytest.raises(KernelError, match="fewer than"):
                call(q, width)
        assert (out == 9).all()
    for call in both:
        call(row.expand(n, width).contiguous(), width)
        assert (out != 9).any()
        out.fill_(9)
