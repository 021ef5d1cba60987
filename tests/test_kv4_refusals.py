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
