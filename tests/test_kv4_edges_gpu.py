"""The cache of 4-bit keys and values on the GPU: batches, lengths and shapes at which its kernels take another way through, against the
same formulas in float64."""
import math

import numpy as np
import pytest
import torch

import plain_kv4 as P
from braidinfer_amd import kernels as K
from braidinfer_amd.errors import KernelError
from test_kv4_gpu import PAGE, bf16, dev, step_of, test_quarter_turns_are_rotated_exactly as quarter_turns, tolerance

pytestmark = pytest.mark.gpu


def held(rows):
    """`plain_kv4.held` of rows without infinities and NaN, on their device."""
    x = rows.double().unflatten(-1, (-1, 32))
    step = torch.exp2((torch.frexp(x.abs().amax(-1, keepdim=True))[1] - 3).clamp(min=-124).double())
    y = (x / step).abs()
    code = (y > 0.25).long() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5)      # ties to the even code
    return (torch.tensor(P.GRID, device=x.device)[code] * step * torch.where(x < 0, -1.0, 1.0)).flatten(-2)


class Written:
    """Sequences of the given lengths in shuffled pages, written by the library's own kernel (checked byte for byte elsewhere);
    `kv`: what the cache holds of each, float64 on the GPU, [tokens, nkv, hd]."""

    def __init__(self, lens, nkv, hd, seed=0, loud=1.0):
        rng = np.random.default_rng(seed)
        self.lens, self.nkv, self.hd = list(lens), nkv, hd
        pages = [-(-n // PAGE) for n in lens]
        n = sum(pages) + 2
        perm, at = rng.permutation(n), 0
        self.slots = rng.permutation(len(lens) + 2)[:len(lens)]
        table = np.full((len(lens) + 2, max(pages + [1])), -1, dtype=np.int32)
        for s, p in zip(self.slots, pages):
            table[s, :p] = perm[at:at + p]
            at += p
        self.table = dev(table)
        self.cache = torch.from_numpy(rng.integers(0, 256, (n, nkv, 68 * hd), dtype=np.uint8)).cuda()
        torch.manual_seed(seed)
        rows = torch.randn(sum(lens), 2 * nkv, hd, device="cuda")
        rows[:, :nkv] *= loud
        rows = rows.bfloat16()
        pos, seq, _ = step_of(lens, [0] * len(lens))
        K.rope_kv4_write(rows.reshape(len(rows), -1), None, None, pos, seq, dev(self.slots), self.table, self.cache, 0, nkv, hd, 0,
                         False, PAGE, True)
        values, cuts = held(rows), np.concatenate([[0], np.cumsum(lens)])
        self.kv = [(values[a:b, :nkv], values[a:b, nkv:]) for a, b in zip(cuts, cuts[1:])]


def attention(q, k, v, scale, first, window=None):
    """`plain_kv4.attention` in float64 on the GPU, of keys and values without NaN."""
    n, nq, hd = q.shape
    G = nq // k.shape[1]
    at, key = torch.arange(first, first + n, device="cuda")[:, None], torch.arange(first + n, device="cuda")[None, :]
    seen = (key <= at) & ((key > at - window) if window is not None else True)
    out, size, most = torch.zeros_like(q), torch.zeros_like(q), 0.0
    for h in range(nq):
        kk, vv = k[:first + n, h // G], v[:first + n, h // G]
        w = torch.softmax((q[:, h] @ kk.T * scale).masked_fill(~seen, float("-inf")), -1)
        out[:, h], size[:, h] = w @ vv, w @ vv.abs()
        most = max(most, float((q[:, h].abs() @ kk.abs().T).max()) * scale)
    return out.cpu().numpy(), size.cpu().numpy(), most


# ---------------------------------------------------------------- rows in and out ----
@pytest.mark.parametrize("hd,rd,adjacent", [(256, 256, False), (128, 128, True), (192, 192, False), (224, 100, True), (64, 12, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_rotations(hd, rd, adjacent, dtype):
    quarter_turns(hd, rd, adjacent, dtype)


def test_more_tokens_than_one_dimension_of_a_grid_holds():
    n, hd = 8 * 32768 + 13, 32
    torch.manual_seed(0)
    rows = torch.randn(n, 2 * hd, device="cuda").bfloat16()
    pages = -(-n // PAGE)
    table = torch.randperm(pages, device="cuda").int().view(1, -1)
    cache = torch.zeros(pages, 1, 68 * hd, dtype=torch.uint8, device="cuda")
    pos, seq, slots = torch.arange(n, device="cuda").int(), torch.zeros(n, device="cuda").int(), dev([0])
    K.rope_kv4_write(rows, None, None, pos, seq, slots, table, cache, 0, 1, hd, 0, False, PAGE, True)
    k, v = (torch.zeros(n, hd, device="cuda") for _ in range(2))
    K.kv4_read(k, v, pos, seq, slots, table, cache, 1, hd, PAGE)
    want = held(rows.view(n, 2, hd))
    assert torch.equal(k.double(), want[:, 0]) and torch.equal(v.double(), want[:, 1])
    np.testing.assert_array_equal(want[:3000].cpu().numpy(), P.held(rows[:3000].float().cpu().numpy().reshape(-1, 2, hd)))


def test_queries_alone_are_rotated_without_a_cache():
    nq, nkv, hd, n = 3, 1, 128, 11
    torch.manual_seed(0)
    qkv = torch.randn(n, (nq + 2 * nkv) * hd, device="cuda").bfloat16()
    cos, sin = torch.zeros(n, hd // 2, device="cuda"), torch.ones(n, hd // 2, device="cuda")
    pos, seq, _ = step_of([n], [0])
    before = qkv.clone().view(n, -1, hd)
    K.rope_kv4_write(qkv, cos, sin, pos, seq, dev([0]), dev([[0]]), None, nq, nkv, hd, hd, False, PAGE, False)
    got = qkv.view(n, -1, hd)
    assert torch.equal(got[:, :nq, :64], -before[:, :nq, 64:]) and torch.equal(got[:, :nq, 64:], before[:, :nq, :64])
    assert torch.equal(got[:, nq:], before[:, nq:])


# ---------------------------------------------------------------- single tokens ----
@pytest.mark.parametrize("hd,nq,nkv", [(128, 8, 2), (64, 7, 1), (128, 12, 1), (96, 40, 2), (256, 4, 2)])
@pytest.mark.parametrize("nsplit,window", [(1, None), (2, None), (7, None), (64, None), (5, 100)])
def test_single_tokens_of_many_sequences(hd, nq, nkv, nsplit, window):
    rng = np.random.default_rng(hd + nq)
    lens = [int(x) for x in rng.choice([0, 1, 30, 64, 65, 200, 900], 150)]
    lens[0], lens[70], lens[149] = 0, 5000, 1300
    c = Written(lens, nkv, hd, seed=nq)
    B, scale = len(lens), 1 / math.sqrt(hd)
    q = torch.randn(B, nq * hd, device="cuda").bfloat16()
    slots = dev(c.slots)
    slots[33] = -1
    out = torch.full((B + 2, nq * hd), 5.0, device="cuda", dtype=torch.bfloat16)
    part = [torch.full((B * nq * nsplit * x,), float("nan"), device="cuda") for x in (hd, 2)] if nsplit > 1 else [None, None]
    K.attention_decode_kv4(q, nq * hd, out, slots, dev(lens), c.table, c.cache, B, nq, nkv, hd, PAGE, window, scale, nsplit, *part)
    assert (out[B:] == 5).all()
    got = out[:B].double().cpu().numpy().reshape(B, nq, hd)
    for b, n in enumerate(lens):
        if n == 0 or b == 33:
            assert (got[b] == 0).all()
            continue
        want, size, most = attention(q[b].double().view(1, nq, hd), *c.kv[b], scale, n - 1, window)
        assert (np.abs(got[b:b + 1] - want) <= tolerance(want, size, most, hd, n)).all(), b


def test_single_tokens_where_nothing_is_there():
    for B, pages in ((3, 0), (70, 0), (70, 4)):
        table, cache = torch.full((80, pages), -1, device="cuda").int(), torch.zeros(1, 1, 68 * 64, device="cuda", dtype=torch.uint8)
        q = torch.randn(B, 128, device="cuda").bfloat16()
        for nsplit in (1, 3):
            out = torch.full((B, 128), 5.0, device="cuda", dtype=torch.bfloat16)
            part = [torch.zeros(B * 2 * nsplit * x, device="cuda") for x in (64, 2)]
            K.attention_decode_kv4(q, 128, out, torch.arange(B, device="cuda").int(), torch.full((B,), 64 * pages, device="cuda").int(), table,
                                   cache, B, 2, 1, 64, PAGE, None, 0.1, nsplit, *part)
            assert (out == 0).all()


def test_shares_that_begin_behind_31_bits():
    # a table of 2.9 million pages, of which two are there: the places that the last workgroups would begin at are beyond 2^31
    hd, pages = 32, 2_900_000
    c = Written([128], 1, hd)
    table = torch.full((1, pages), -1, device="cuda").int()
    table[0, 0], table[0, pages - 1] = c.table[int(c.slots[0]), 0], c.table[int(c.slots[0]), 1]
    q = torch.randn(1, hd, device="cuda").bfloat16()
    out = torch.zeros(1, hd, device="cuda", dtype=torch.bfloat16)
    part = [torch.zeros(2 * x, device="cuda") for x in (hd, 2)]
    K.attention_decode_kv4(q, hd, out, dev([0]), dev([pages * PAGE]), table, c.cache, 1, 1, 1, hd, PAGE, None, 0.2, 2, *part)
    want, size, most = attention(q.double().view(1, 1, hd), *c.kv[0], 0.2, 127)
    assert (np.abs(out.double().cpu().numpy().reshape(1, 1, hd) - want) <= tolerance(want, size, most, hd, 128)).all()


def test_windows_beyond_31_bits_are_none():
    c = Written([300], 1, 64)
    q = torch.randn(300, 64, device="cuda").bfloat16()
    got = []
    for window in (None, 1 << 31, 1 << 33):
        one, many = torch.zeros(1, 64, device="cuda").bfloat16(), torch.zeros(300, 64, device="cuda").bfloat16()
        K.attention_decode_kv4(q, 64, one, dev(c.slots), dev([300]), c.table, c.cache, 1, 1, 1, 64, PAGE, window, 0.1, 1)
        K.attention_prefill_kv4(q, 64, many, dev([0, 300]), dev(c.slots), dev([300]), c.table, c.cache, 1, 300, 1, 1, 64, PAGE, window, 0.1, 1)
        got.append((one, many))
    for one, many in got[1:]:
        assert torch.equal(one, got[0][0]) and torch.equal(many, got[0][1])


# --------------------------------------------------------------------- prompts ----
def prompts(c, q, counts, nq, window, scale, nsplit, max_new=None):
    T, hd = sum(counts), c.hd
    out = torch.full((T + 3, nq * hd), 9.0, device="cuda", dtype=torch.bfloat16)
    part = [torch.full(((T + 3) * nq * nsplit * x,), float("nan"), device="cuda") for x in (hd, 2)] if nsplit > 1 else [None, None]
    K.attention_prefill_kv4(q, nq * hd, out, step_of(counts, [0] * len(counts))[2], dev(c.slots), dev(c.lens), c.table, c.cache, len(counts),
                            max_new or max(counts), nq, c.nkv, hd, PAGE, window, scale, nsplit, *part)
    assert (out[T:] == 9).all()
    return out[:T].double().cpu().numpy().reshape(T, nq, hd)


@pytest.mark.parametrize("hd,nq,nkv", [(32, 35, 7), (64, 32, 8), (96, 32, 8), (128, 32, 8), (128, 20, 20), (256, 16, 8)])
@pytest.mark.parametrize("window,nsplit", [(None, 1), (200, 1), (None, 3)])
def test_prompts_that_fill_the_device(hd, nq, nkv, window, nsplit):
    counts, starts = [700, 0, 650, 3, 65], [0, 20, 300, 20, 1000]
    c = Written([a + b for a, b in zip(counts, starts)], nkv, hd, seed=hd, loud=2.0)
    q = torch.randn(sum(counts) + 3, nq * hd, device="cuda").bfloat16()
    scale, at = 1 / math.sqrt(hd), 0
    got = prompts(c, q, counts, nq, window, scale, nsplit)
    for (k, v), n, s in zip(c.kv, counts, starts):
        if n:
            want, size, most = attention(q[at:at + n].double().view(n, nq, hd), k, v, scale, s, window)
            assert (np.abs(got[at:at + n] - want) <= tolerance(want, size, most, hd, s + n)).all()
        at += n


def test_a_prompt_of_one_row_for_a_long_context():
    # pages beyond the 64 whose numbers a wave holds at a time, and beyond them again
    nq, nkv, hd, n = 4, 1, 128, 9000
    c = Written([n], nkv, hd, loud=2.0)
    for count in (1, 33):
        q = torch.randn(count + 3, nq * hd, device="cuda").bfloat16()
        for nsplit, window in ((1, None), (9, None), (64, None), (1, 5000)):
            got = prompts(c, q, [count], nq, window, 0.1, nsplit, max_new=count)
            want, size, most = attention(q[:count].double().view(count, nq, hd), *c.kv[0], 0.1, n - count, window)
            assert (np.abs(got - want) <= tolerance(want, size, most, hd, n)).all()


def test_the_rule_for_runs_covers_what_the_kernels_take():
    for n_seqs in (1, 7, 64, 500):
        for max_new in (1, 5, 600):
            for nq, nkv, hd in ((32, 8, 128), (1, 1, 32), (71, 1, 256)):
                for max_ctx in (max_new, 700, 40_000, 1 << 21):
                    for window in (None, 1, 4096):
                        assert 1 <= K.attention_kv4_splits(n_seqs, max_new, nq, nkv, hd, max(max_ctx, max_new), window) <= 64


def test_lists_longer_than_the_kernel_counts_are_refused():
    table, cache = torch.full((1, 33_000_000), -1, device="cuda").int(), torch.zeros(1, 1, 68 * 32, device="cuda", dtype=torch.uint8)
    q = torch.zeros(40, 32, device="cuda").bfloat16()
    out = torch.ones(40, 32, device="cuda").bfloat16()
    part = [torch.zeros(40 * 2 * x, device="cuda") for x in (32, 2)]
    with pytest.raises(KernelError):
        K.attention_decode_kv4(q, 32, out, dev([0] * 40), dev([64] * 40), table, cache, 40, 1, 1, 32, PAGE, None, 0.2, 2, *part)
    assert (out == 1).all()


def test_outputs_and_scratch_that_are_not_aligned_or_elsewhere_are_refused():
    c = Written([70], 1, 64)
    q = torch.zeros(4, 64, device="cuda").bfloat16()
    room = torch.ones(4 * 64 + 8, device="cuda").bfloat16()
    good, odd = room[:256].view(4, 64), room[2:258].view(4, 64)
    part = [torch.zeros(4 * 2 * x, device="cuda") for x in (64, 2)]

    def one(out, nsplit=1, part_o=None, part_ml=None, slots=dev(c.slots)):
        K.attention_decode_kv4(q, 64, out, slots, dev([70]), c.table, c.cache, 1, 1, 1, 64, PAGE, None, 0.1, nsplit, part_o, part_ml)

    def many(out, nsplit=1, part_o=None, part_ml=None, cu=dev([0, 4])):
        K.attention_prefill_kv4(q, 64, out, cu, dev(c.slots), dev([70]), c.table, c.cache, 1, 4, 1, 1, 64, PAGE, None, 0.1, nsplit, part_o, part_ml)

    for call in (one, many):
        with pytest.raises(KernelError, match="aligned"):
            call(odd)
        with pytest.raises(KernelError, match="scratch"):
            call(good, 2)
        with pytest.raises(KernelError, match="GPU only"):
            call(good, 2, part[0].cpu(), part[1])
        with pytest.raises(KernelError, match="contiguous"):
            call(good, 2, part[0], torch.zeros(16, 2, device="cuda").t())
        with pytest.raises(KernelError, match="64 runs"):
            call(good, 0)
        with pytest.raises(KernelError, match="GPU only"):
            call(good.cpu())
    with pytest.raises(KernelError, match="GPU only"):
        one(good, slots=dev(c.slots).cpu())
    with pytest.raises(KernelError, match="GPU only"):
        many(good, cu=dev([0, 4]).cpu())
    assert (room == 1).all()
    one(good, 2, *part)
    many(good, 2, *part)
