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


@pytest.mark.parametrize("scale", [1e-46, 5e-324, 2.4e38, 1e300, float("inf")])
def test_scales_that_are_none_in_32_bits(scale):
    out, one, many = calls(70)
    q = torch.randn(70, NQ * HD, device="cuda").bfloat16()
    for call in (one, many):
        with pytest.raises(KernelError, match="scale"):
            call(q, NQ * HD, scale)
    assert (out == 9).all()


def test_the_smallest_scale_weighs_all_tokens_alike():
    n = 70
    c = Cache([n], NKV, HD)
    k, v = c.fill()[0]
    table, cache = c.tensors
    q = torch.randn(n, NQ * HD, device="cuda").bfloat16()
    for scale in (1e-45, 1e-40):
        out = torch.full((n, NQ * HD), 9.0, device="cuda", dtype=torch.bfloat16)
        K.attention_prefill_kv4(q, NQ * HD, out, step_of([n], [0])[2], dev(c.slots), dev(c.lens), table, cache, 1, n, NQ, NKV, HD, PAGE, None,
                                scale, 1)
        last = torch.full((1, NQ * HD), 9.0, device="cuda", dtype=torch.bfloat16)
        K.attention_decode_kv4(q, NQ * HD, last, dev(c.slots), dev(c.lens), table, cache, 1, NQ, NKV, HD, PAGE, None, scale, 1)
        for got, rows in ((out, range(n)), (last, [n - 1])):
            got = got.double().cpu().numpy().reshape(-1, NQ, HD)
            for i, t in enumerate(rows):
                # weights of 1 are exact: the sum over t + 1 tokens in float, one rounding to bfloat16
                want, size = (x[:t + 1].mean(0).repeat(NQ // NKV, 0) for x in (v, abs(v)))
                assert (abs(got[i] - want) <= 2.0 ** -8 * abs(want) + (t + 3) * 2.0 ** -24 * size).all()
