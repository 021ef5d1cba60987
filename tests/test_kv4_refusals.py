"""4-bit keys and values, on the CPU: arguments that would have the kernels read what is not there."""
import pytest
import torch

from braidinfer_amd import kernels as K
from braidinfer_amd.errors import KernelError


def test_queries_have_to_lie_in_their_memory():
    bf16, width = torch.bfloat16, 64
    room = torch.zeros(10 * 96, dtype=bf16)
    rows = room.view(10, 96)
    ok = [(rows, 96, 10), (rows[:, :width], 96, 10), (rows[3:], 96, 7), (rows[:, 16:16 + width], 96, 10), (room.view(15, width), width, 15),
          (rows[:1], 96, 10), (rows[:0], 96, 0), (rows[2:, 32:], 96, 8)]
    for q, stride, T in ok:
        K._kv4_queries("q", q, stride, T, width)
    bad = [(rows, 96, 11), (rows[4:], 96, 7), (rows[:, 40:], 96, 10),
           (room[:width].clone().expand(10, width), width, 10),                 # one row, said to be ten
           (room[:1].clone().expand(10, width), width, 10),
           (rows[9:, 32:].expand(10, width), 96, 10),
           (torch.zeros(5, 1, width, dtype=bf16).expand(5, 9, width), width, 45)]
    for q, stride, T in bad:
        with pytest.raises(KernelError, match="fewer than"):
            K._kv4_queries("q", q, stride, T, width)
    for stride in (width - 8, width + 4):
        with pytest.raises(KernelError, match="aligned"):
            K._kv4_queries("q", rows, stride, 2, width)


def test_tables_and_batches_beyond_31_bits():
    def of(*shape):
        return torch.empty(shape, dtype=torch.int32, device="meta")

    assert tuple(K._kv4_table("t", of(3, (1 << 31) - 1))) == (3, (1 << 31) - 1)
    # the entry points take 32-bit sizes: 2^32 + 1 would come through as 1
    for shape in ((1, 1 << 31), (1, (1 << 32) + 1), ((1 << 32) + 2, 1), ((1 << 31), 0)):
        with pytest.raises(KernelError, match="block table"):
            K._kv4_table("t", of(*shape))
    K._kv4_rows("r", of(9), of(9), of((1 << 31) - 1), 9)
    for n in (1 << 31, (1 << 32) + 1):
        with pytest.raises(KernelError, match="slots"):
            K._kv4_rows("r", of(9), of(9), of(n), 9)
