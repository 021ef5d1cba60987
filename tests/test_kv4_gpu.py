"""The cache of 4-bit keys and values and the attention that reads it, on the GPU, against plain formulas in float64."""
import math

import numpy as np
import pytest
import torch

import plain_kv4 as P
from braidinfer_amd import kernels as K
from braidinfer_amd.errors import KernelError

pytestmark = pytest.mark.gpu
PAGE = 64


def dev(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x), dtype=dtype).cuda()


class Cache:
    """Sequences in shuffled pages of a cache whose other bytes are noise (NaN scales among them)."""

    def __init__(self, lens, nkv, hd, seed=0, spare=3):
        rng = np.random.default_rng(seed)
        self.nkv, self.hd, self.lens = nkv, hd, list(lens)
        pages = [-(-n // PAGE) for n in lens]
        n = sum(pages) + spare
        perm, at = rng.permutation(n), 0
        self.slots = rng.permutation(len(lens) + 2)[:len(lens)]
        self.table = np.full((len(lens) + 2, max(pages + [1])), -1, dtype=np.int32)
        for s, p in zip(self.slots, pages):
            self.table[s, :p] = perm[at:at + p]
            at += p
        self.bytes = rng.integers(0, 256, (n, nkv, 68 * hd), dtype=np.uint8)

    def put(self, b, pos, k, v):
        """Rows k, v [nkv, hd] of position `pos` of sequence b."""
        for h in range(self.nkv):
            P.put(self.bytes[self.table[self.slots[b], pos // PAGE], h], pos % PAGE, k[h], v[h])

    def fill(self, seed=1, loud=1.0):
        """Random rows for all sequences, rounded to bfloat16; returns what the cache holds of them, float64 [tokens, nkv, hd]."""
        rng = np.random.default_rng(seed)
        out = []
        for b, n in enumerate(self.lens):
            k = bf16(rng.standard_normal((n, self.nkv, self.hd)) * loud)
            v = bf16(rng.standard_normal((n, self.nkv, self.hd)))
            for p in range(n):
                self.put(b, p, k[p], v[p])
            out.append([P.held(k), P.held(v)])
        return out

    @property
    def tensors(self):
        return dev(self.table), torch.from_numpy(self.bytes).cuda()


def bf16(x):
    return torch.as_tensor(np.asarray(x, dtype=np.float32)).bfloat16().float().numpy()


def step_of(counts, starts):
    """positions, seq_of_token, cu_seqlens of a step."""
    pos = np.concatenate([np.arange(s, s + n) for s, n in zip(starts, counts)] + [np.zeros(0, int)])
    return dev(pos), dev(np.repeat(np.arange(len(counts)), counts)), dev(np.concatenate([[0], np.cumsum(counts)]))


def tolerance(want, size, most, hd, n):
    """What an element may be off by: the probabilities are rounded to bfloat16 (2^-8 of each, so of the sum with |v|), the result
    is (2^-8 of it); scores are float sums of hd exact products (hd 2^-24 of sum |q k|, as an exponent: that much of each
    probability, in the sum and in the weights' sum), sums over n keys are float, as is the exponential (2^-21)."""
    return 2.0 ** -8 * np.abs(want) + size * (2.0 ** -8 + 2 * hd * 2.0 ** -24 * most + 2 * n * 2.0 ** -24 + 2.0 ** -21) + 1e-30


# ------------------------------------------------------------------------- writing ----
@pytest.mark.parametrize("hd,nq,nkv", [(32, 3, 1), (64, 0, 3), (96, 2, 2), (128, 4, 2), (160, 1, 1), (192, 1, 1), (224, 2, 1), (256, 1, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_go_into_their_pages_byte_for_byte(hd, nq, nkv, dtype):
    counts, starts = [1, 70, 3, 9], [63, 5, 0, 120]
    c = Cache([s + n for s, n in zip(starts, counts)], nkv, hd, seed=hd)
    rng = np.random.default_rng(hd + nq)
    T = sum(counts) + 2                                                    # two rows of padding behind
    rows = (rng.standard_normal((T, nq + 2 * nkv, hd)) * np.exp(3 * rng.standard_normal((T, nq + 2 * nkv, 1)))).astype(np.float32)
    rows[0, nq, :32] = 0.0
    rows[1, nq, 3], rows[2, nq + nkv, 5], rows[3, nq, 31] = np.inf, np.nan, -np.inf
    rows[4, nq] = 3e38 * np.sign(rows[4, nq])
    rows[5, nq + nkv] *= 1e-37
    rows[6, nq, :32] = np.arange(32) / 4                                   # ties
    rows[7, nq + nkv, :32] = -np.arange(32) / 4 * 2.0 ** -60
    rows[8, nq] = -0.0
    t = torch.from_numpy(rows).to(dtype)
    rows = t.float().numpy()
    pos, seq, _ = step_of(counts + [1, 1], starts + [0, 0])
    slots = dev(list(c.slots) + [-1, -1])
    table, cache = c.tensors
    at = 0
    for b, (n, s) in enumerate(zip(counts, starts)):
        for i in range(n):
            c.put(b, s + i, rows[at, nq:nq + nkv], rows[at, nq + nkv:])
            at += 1
    qkv = t.reshape(T, -1).cuda()
    before = qkv.clone()
    K.rope_kv4_write(qkv, None, None, pos, seq, slots, table, cache, nq, nkv, hd, 0, False, PAGE, True)
    got = cache.cpu().numpy()
    want = c.bytes.copy()
    for x in (got, want):                                                  # -0 and 0 are one value: compare the codes as such
        codes = x.reshape(-1, 68 * hd)
        m = hd // 32
        for part in (codes[:, :1024 * m], codes[:, 1088 * m:2112 * m]):
            part[(part & 15) == 8] &= 0xF0
            part[(part >> 4) == 8] &= 0x0F
    assert np.array_equal(got, want)
    assert torch.equal(before.view(torch.int16 if dtype == torch.bfloat16 else torch.int32), qkv.view(torch.int16 if dtype == torch.bfloat16 else torch.int32))
    # and out again, in both types; rows of padding stay
    for out_type in (torch.bfloat16, torch.float32):
        ko, vo = (torch.full((T, nkv * hd), 7.0, dtype=out_type, device="cuda") for _ in range(2))
        K.kv4_read(ko, vo, pos, seq, slots, table, cache, nkv, hd, PAGE)
        for o, first in ((ko, nq), (vo, nq + nkv)):
            want_rows = P.held(rows[:T - 2, first:first + nkv]).reshape(T - 2, -1)
            np.testing.assert_array_equal(o[:T - 2].double().cpu().numpy(), want_rows)
            assert (o[T - 2:] == 7).all()


@pytest.mark.parametrize("hd,rd,adjacent", [(64, 64, False), (64, 64, True), (96, 96, False), (128, 128, False), (128, 32, False), (128, 34, False),
                                            (128, 20, True), (128, 6, True), (160, 160, False), (32, 30, False), (256, 256, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quarter_turns_are_rotated_exactly(hd, rd, adjacent, dtype):
    nq, nkv, n = 3, 2, 21
    c = Cache([n + 50], nkv, hd, seed=rd)
    rng = np.random.default_rng(rd)
    rows = torch.from_numpy(rng.standard_normal((n, nq + 2 * nkv, hd)).astype(np.float32)).to(dtype)
    quarter = rng.integers(0, 4, (n, rd // 2))
    cos, sin = np.array([1, 0, -1, 0])[quarter], np.array([0, 1, 0, -1])[quarter]
    x = rows.float().numpy()
    turned = x.copy()
    i0 = 2 * np.arange(rd // 2) if adjacent else np.arange(rd // 2)
    i1 = i0 + 1 if adjacent else i0 + rd // 2
    for h in range(nq + nkv):
        a, b = x[:, h][:, i0], x[:, h][:, i1]
        turned[:, h, i0], turned[:, h, i1] = a * cos - b * sin, a * sin + b * cos
    pos, seq, _ = step_of([n], [50])
    table, cache = c.tensors
    qkv = rows.reshape(n, -1).cuda()
    K.rope_kv4_write(qkv, dev(cos, torch.float32), dev(sin, torch.float32), pos, seq, dev(c.slots), table, cache, nq, nkv, hd, rd, adjacent,
                     PAGE, True)
    np.testing.assert_array_equal(qkv.float().cpu().numpy().reshape(n, -1, hd)[:, :nq], turned[:, :nq])
    np.testing.assert_array_equal(qkv.float().cpu().numpy().reshape(n, -1, hd)[:, nq:], x[:, nq:])
    ko, vo = (torch.zeros((n, nkv * hd), device="cuda") for _ in range(2))
    K.kv4_read(ko, vo, pos, seq, dev(c.slots), table, cache, nkv, hd, PAGE)
    for o, want in ((ko, turned[:, nq:nq + nkv]), (vo, x[:, nq + nkv:])):
        np.testing.assert_array_equal(o.double().cpu().numpy().reshape(n, nkv, hd), P.held(want))
    # queries alone: nothing of the cache is touched
    kept = cache.clone()
    again = rows.reshape(n, -1).cuda()
    K.rope_kv4_write(again, dev(cos, torch.float32), dev(sin, torch.float32), pos, seq, dev(c.slots), table, None, nq, nkv, hd, rd, adjacent,
                     PAGE, False)
    assert torch.equal(again, qkv) and torch.equal(kept, cache)


@pytest.mark.parametrize("adjacent", [False, True])
def test_any_angle_is_rotated(adjacent):
    nq, nkv, hd, n = 2, 1, 128, 40
    c = Cache([n], nkv, hd)
    rng = np.random.default_rng(5)
    rows = torch.from_numpy(rng.standard_normal((n, nq + 2 * nkv, hd)).astype(np.float32)).bfloat16()
    angle = rng.uniform(-3, 3, (n, hd // 2))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    x = rows.double().numpy()
    i0 = 2 * np.arange(hd // 2) if adjacent else np.arange(hd // 2)
    i1 = i0 + 1 if adjacent else i0 + hd // 2
    turned = x.copy()
    turned[:, :, i0] = x[:, :, i0] * cos[:, None].astype(np.float64) - x[:, :, i1] * sin[:, None].astype(np.float64)
    turned[:, :, i1] = x[:, :, i0] * sin[:, None].astype(np.float64) + x[:, :, i1] * cos[:, None].astype(np.float64)
    pos, seq, _ = step_of([n], [0])
    table, cache = c.tensors
    qkv = rows.reshape(n, -1).cuda()
    K.rope_kv4_write(qkv, dev(cos, torch.float32), dev(sin, torch.float32), pos, seq, dev(c.slots), table, cache, nq, nkv, hd, hd, adjacent,
                     PAGE, True)
    got = qkv.double().cpu().numpy().reshape(n, -1, hd)[:, :nq]
    # rounded to bfloat16 behind two float products of numbers below 8
    assert (np.abs(got - turned[:, :nq]) <= 2.0 ** -8 * np.abs(turned[:, :nq]) + 16 * 2.0 ** -24).all()
    ko, vo = (torch.zeros((n, hd), device="cuda") for _ in range(2))
    K.kv4_read(ko, vo, pos, seq, dev(c.slots), table, cache, nkv, hd, PAGE)
    k = turned[:, nq]
    # The key that is held is off by 2^-8 first, so its block's largest magnitude is off by a factor within 1 +- 2^-7 and its step is the
    # one of either end (a step that is half as large leaves up to 2 of its own beyond 6, more than the larger step's bound).  Of a step,
    # the distance to the nearest value is a quarter below 2, half below 4, 1 up to 7 and less than 2 up to 8.
    most = np.abs(k.reshape(n, -1, 32)).max(-1)
    bound = np.zeros_like(k)
    for off in (1 - 2.0 ** -7, 1 + 2.0 ** -7):
        step = np.repeat(2.0 ** (np.floor(np.log2(most * off)) - 2), 32, -1).reshape(n, hd)
        y = np.abs(k) / step
        bound = np.maximum(bound, step * np.where(y > 5, 2.0, np.where(y > 3.9, 1.0, np.where(y > 1.9, 0.5, 0.25))))
    assert (np.abs(ko.double().cpu().numpy() - k) <= bound + 2.0 ** -8 * np.abs(k) + 16 * 2.0 ** -24).all()


def test_places_that_are_not_there_take_and_give_nothing():
    nkv, hd = 2, 64
    c = Cache([100, 100, 100], nkv, hd)
    n_pages = len(c.bytes)
    c.table[c.slots[1], 0] = n_pages + 7
    c.table[c.slots[2], 0] = -5
    table, cache = c.tensors
    kept = cache.clone()
    # positions beyond the table, below zero, pages outside the cache, slots outside the table, a sequence that is none
    pos = dev([10_000, -3, 5, 6, 7, 8])
    seq = dev([0, 0, 1, 2, 3, 9])
    slots = dev(list(c.slots) + [len(c.table) + 1])
    qkv = torch.randn(6, (1 + 2 * nkv) * hd, device="cuda").bfloat16()
    K.rope_kv4_write(qkv, None, None, pos, seq, slots, table, cache, 1, nkv, hd, 0, False, PAGE, True)
    assert torch.equal(kept, cache)
    ko, vo = (torch.full((6, nkv * hd), 3.0, device="cuda") for _ in range(2))
    K.kv4_read(ko, vo, pos, seq, slots, table, cache, nkv, hd, PAGE)
    assert (ko == 3).all() and (vo == 3).all()


# ---------------------------------------------------------------------- single tokens ----
def decode(c, q, window, scale, nsplit, slots=None, ctx=None, stride=None):
    table, cache = c.tensors
    B, nq, hd = q.shape
    rows = torch.zeros(B, stride or nq * hd, device="cuda", dtype=torch.bfloat16)
    rows[:, :nq * hd] = torch.from_numpy(q).reshape(B, -1).cuda()
    out = torch.full((B, nq * hd), float("nan"), device="cuda", dtype=torch.bfloat16)
    part = torch.full((B * nq * nsplit * hd,), float("nan"), device="cuda"), torch.full((B * nq * nsplit * 2,), float("nan"), device="cuda")
    K.attention_decode_kv4(rows, rows.stride(0), out, dev(c.slots if slots is None else slots), dev(c.lens if ctx is None else ctx), table, cache,
                           B, nq, c.nkv, hd, PAGE, window, scale, nsplit, *(part if nsplit > 1 else (None, None)))
    return out.double().cpu().numpy().reshape(B, nq, hd)


@pytest.mark.parametrize("hd,nq,nkv", [(32, 6, 3), (64, 8, 1), (64, 4, 4), (96, 5, 1), (128, 8, 2), (128, 16, 1), (128, 40, 2), (160, 3, 1), (192, 2, 1), (224, 2, 1),
                                       (256, 4, 1)])
@pytest.mark.parametrize("window,nsplit", [(None, 1), (None, 3), (70, 1), (1, 2), (200, 5)])
def test_single_tokens(hd, nq, nkv, window, nsplit):
    c = Cache([1, 63, 64, 65, 200, 333], nkv, hd, seed=hd + nq)
    kv = c.fill(seed=nq, loud=2.0)
    q = bf16(np.random.default_rng(3).standard_normal((len(c.lens), nq, hd)))
    scale = 1 / math.sqrt(hd)
    got = decode(c, q, window, scale, nsplit, stride=(nq + 2 * nkv) * hd)
    for b, (k, v) in enumerate(kv):
        want, size, most = P.attention(q[b:b + 1].astype(np.float64), k, v, scale, c.lens[b] - 1, window)
        assert (np.abs(got[b:b + 1] - want) <= tolerance(want, size, most, hd, c.lens[b])).all()


def test_padding_empty_sequences_and_missing_pages():
    nq, nkv, hd = 4, 2, 64
    c = Cache([130, 200, 50, 70], nkv, hd)
    kv = c.fill()
    c.table[c.slots[1], 1] = len(c.bytes)              # its second page is not there: attention goes without it
    q = bf16(np.random.default_rng(0).standard_normal((6, nq, hd)))
    slots, ctx = list(c.slots) + [-1, len(c.table)], [130, 200, 0, 70, 40, 40]
    for nsplit in (1, 2, 4):
        got = decode(c, q, None, 0.125, nsplit, slots, ctx)
        assert (got[2] == 0).all() and (got[4:] == 0).all()
        for b in (0, 1, 3):
            k, v = kv[b]
            if b == 1:
                k, v = np.delete(k, slice(64, 128), 0), np.delete(v, slice(64, 128), 0)
            want, size, most = P.attention(q[b:b + 1].astype(np.float64), k, v, 0.125, len(k) - 1)
            assert (np.abs(got[b:b + 1] - want) <= tolerance(want, size, most, hd, 200)).all()


def test_nan_that_a_token_does_not_see_stays_out():
    nq, nkv, hd = 4, 1, 128
    c = Cache([150, 150, 150], nkv, hd)
    kv = c.fill()
    bad = np.full((nkv, hd), np.nan)
    for b in range(3):
        c.put(b, 20, bad, bad)                        # outside the window of 100
    mixed = np.ones((nkv, hd))
    mixed[0, 40] = np.inf                             # a value block that is NaN, inside: its 32 channels and no others
    c.put(1, 130, kv[1][0][130], mixed)
    c.put(2, 131, bad, np.ones((nkv, hd)))            # a key inside: the whole row
    q = bf16(np.random.default_rng(0).standard_normal((3, nq, hd)))
    for nsplit in (1, 3):
        got = decode(c, q, 100, 0.1, nsplit)
        want, size, most = P.attention(q[:1].astype(np.float64), *kv[0], 0.1, 149, 100)
        assert (np.abs(got[:1] - want) <= tolerance(want, size, most, hd, 100)).all()
        assert np.isnan(got[1, :, 32:64]).all() and np.isfinite(got[1, :, :32]).all() and np.isfinite(got[1, :, 64:]).all()
        assert np.isnan(got[2]).all()


# --------------------------------------------------------------------------- prompts ----
def prefill(c, q, counts, window, scale, nsplit, slots=None, behind=0, ctx=None):
    table, cache = c.tensors
    T, nq, hd = q.shape
    out = torch.full((T + behind, nq * hd), 9.0, device="cuda", dtype=torch.bfloat16)
    rows = torch.zeros(T + behind, nq * hd, device="cuda", dtype=torch.bfloat16)
    rows[:T] = torch.from_numpy(q).reshape(T, -1).cuda()
    n = (T + behind) * nq * nsplit
    part = torch.full((n * hd,), float("nan"), device="cuda"), torch.full((n * 2,), float("nan"), device="cuda")
    K.attention_prefill_kv4(rows, nq * hd, out, step_of(counts, [0] * len(counts))[2], dev(c.slots if slots is None else slots),
                            dev(c.lens if ctx is None else ctx), table, cache, len(counts), max(counts), nq, c.nkv, hd, PAGE, window, scale, nsplit,
                            *(part if nsplit > 1 else (None, None)))
    assert (out[T:] == 9).all()
    return out[:T].double().cpu().numpy().reshape(T, nq, hd)


@pytest.mark.parametrize("hd,nq,nkv", [(32, 6, 3), (64, 8, 1), (64, 3, 3), (96, 5, 1), (128, 8, 2), (128, 17, 1), (160, 3, 1), (192, 2, 1), (224, 2, 1), (256, 4, 2)])
@pytest.mark.parametrize("window,nsplit", [(None, 1), (None, 3), (70, 1), (1, 1), (33, 2)])
def test_prompts(hd, nq, nkv, window, nsplit):
    counts, starts = [1, 67, 0, 130, 5], [0, 0, 30, 100, 250]
    c = Cache([a + b for a, b in zip(counts, starts)], nkv, hd, seed=hd + nq)
    kv = c.fill(seed=nq, loud=2.0)
    q = bf16(np.random.default_rng(3).standard_normal((sum(counts), nq, hd)))
    scale = 1 / math.sqrt(hd)
    got = prefill(c, q, counts, window, scale, nsplit, behind=3)
    at = 0
    for (k, v), n, s in zip(kv, counts, starts):
        want, size, most = P.attention(q[at:at + n].astype(np.float64), k, v, scale, s, window)
        assert (np.abs(got[at:at + n] - want) <= tolerance(want, size, most, hd, 300)).all()
        at += n


def test_prompts_of_padding_and_missing_pages():
    nq, nkv, hd = 2, 1, 128
    c = Cache([260, 100], nkv, hd)
    kv = c.fill()
    c.table[c.slots[0], 1] = -1
    c.table[c.slots[0], 4] = len(c.bytes) + 3
    counts = [250, 60, 40, 3]
    q = bf16(np.random.default_rng(0).standard_normal((sum(counts), nq, hd)))
    for nsplit in (1, 2, 7):
        got = prefill(c, q, counts, None, 0.1, nsplit, list(c.slots) + [-1, len(c.table) + 4], ctx=[260, 100, 40, 3])
        assert (got[310:] == 0).all()
        want, size, most = P.attention(q[250:310].astype(np.float64), *kv[1], 0.1, 40)
        assert (np.abs(got[250:310] - want) <= tolerance(want, size, most, hd, 100)).all()
        k, v = kv[0]
        for i in (0, 60, 140, 249):                                        # tokens 10, 70, 150, 259
            seen = [j for j in range(i + 11) if j // 64 not in (1, 4)]
            want, size, most = P.attention(q[i:i + 1].astype(np.float64), k[seen], v[seen], 0.1, len(seen) - 1)
            assert (np.abs(got[i:i + 1] - want) <= tolerance(want, size, most, hd, 260)).all()


@pytest.mark.parametrize("nsplit", [1, 2])
@pytest.mark.parametrize("hd", [64, 128, 160])
def test_nan_reaches_the_rows_that_see_it(hd, nsplit):
    nq, nkv, n = 2, 1, 200
    c = Cache([n], nkv, hd)
    kv = c.fill()
    k, v = kv[0]
    some = np.ones((nkv, hd))
    some[0, 35] = np.nan
    c.put(0, 90, k[90], some)                          # block 1 of token 90's value
    v[90] = P.held(some)
    q = bf16(np.random.default_rng(0).standard_normal((n, nq, hd)))
    got = prefill(c, q, [n], 50, 0.1, nsplit)
    want, size, most = P.attention(q.astype(np.float64), k, v, 0.1, 0, 50)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(want[90:140, :, 32:64]).all() and np.isfinite(want[:90]).all() and np.isfinite(want[140:]).all()
    fine = np.isfinite(want)
    assert (np.abs(got - want) <= tolerance(want, size, most, hd, 64))[fine].all()


# ---------------------------------------------------------------------- used together ----
def test_a_prompt_then_tokens_one_by_one():
    """Rows written, attention over the prompt, then twenty tokens written and attended one at a time, through a page's end."""
    nq, nkv, hd, n = 8, 2, 128, 75
    c = Cache([n + 20], nkv, hd)
    table, cache = c.tensors
    rng = np.random.default_rng(0)
    rows = torch.from_numpy(rng.standard_normal((n + 20, (nq + 2 * nkv) * hd)).astype(np.float32)).bfloat16()
    x = rows.double().numpy().reshape(n + 20, -1, hd)
    k, v = (P.held(z) for z in (x[:, nq:nq + nkv], x[:, nq + nkv:]))
    slots = dev(c.slots)
    out = torch.zeros(n + 20, nq * hd, dtype=torch.bfloat16, device="cuda")
    for first, count in [(0, n)] + [(n + i, 1) for i in range(20)]:
        qkv = rows[first:first + count].cuda()
        pos, seq, cu = step_of([count], [first])
        K.rope_kv4_write(qkv, None, None, pos, seq, slots, table, cache, nq, nkv, hd, 0, False, PAGE, True)
        ctx = dev([first + count])
        o = out[first:first + count]
        nsplit = K.attention_kv4_splits(1, count, nq, nkv, hd, first + count)
        part = [torch.empty(count * nq * nsplit * hd, device="cuda"), torch.empty(count * nq * nsplit * 2, device="cuda")] if nsplit > 1 else [None, None]
        if count > 1:
            K.attention_prefill_kv4(qkv, qkv.stride(0), o, cu, slots, ctx, table, cache, 1, count, nq, nkv, hd, PAGE, None, 0.09, nsplit, *part)
        else:
            K.attention_decode_kv4(qkv, qkv.stride(0), o, slots, ctx, table, cache, 1, nq, nkv, hd, PAGE, None, 0.09, nsplit, *part)
    want, size, most = P.attention(x[:, :nq], k, v, 0.09, 0)
    got = out.double().cpu().numpy().reshape(n + 20, nq, hd)
    assert (np.abs(got - want) <= tolerance(want, size, most, hd, n + 20)).all()


def test_pages_behind_four_gigabytes():
    nq, nkv, hd = 8, 8, 128
    n_pages = (1 << 32) // (nkv * 68 * hd) + 40
    small = Cache([150], nkv, hd)
    kv = small.fill()
    cache = torch.zeros(n_pages, nkv, 68 * hd, dtype=torch.uint8, device="cuda")
    table = np.array([[n_pages - 1, n_pages - 30, n_pages - 2]], dtype=np.int32)
    cache[torch.from_numpy(table[0]).long().cuda()] = torch.from_numpy(small.bytes[small.table[small.slots[0]]]).cuda()
    q = bf16(np.random.default_rng(0).standard_normal((150, nq, hd)))
    want, size, most = P.attention(q.astype(np.float64), *kv[0], 0.1, 0)
    rows = torch.from_numpy(q).reshape(150, -1).bfloat16().cuda()
    out = torch.zeros_like(rows)
    args = (dev([0]), dev([150]), dev(table), cache)
    K.attention_prefill_kv4(rows, nq * hd, out, dev([0, 150]), *args, 1, 150, nq, nkv, hd, PAGE, None, 0.1, 1)
    assert (np.abs(out.double().cpu().numpy().reshape(150, nq, hd) - want) <= tolerance(want, size, most, hd, 150)).all()
    last = torch.zeros(1, nq * hd, dtype=torch.bfloat16, device="cuda")
    K.attention_decode_kv4(rows[149:], nq * hd, last, *args, 1, nq, nkv, hd, PAGE, None, 0.1, 1)
    assert (np.abs(last.double().cpu().numpy().reshape(1, nq, hd) - want[149:]) <= tolerance(want, size, most, hd, 150)[149:]).all()
    qkv = torch.randn(1, (nq + 2 * nkv) * hd, device="cuda")
    K.rope_kv4_write(qkv, None, None, dev([149]), dev([0]), dev([0]), dev(table), cache, nq, nkv, hd, 0, False, PAGE, True)
    ko, vo = torch.zeros(1, nkv * hd, device="cuda"), torch.zeros(1, nkv * hd, device="cuda")
    K.kv4_read(ko, vo, dev([149]), dev([0]), dev([0]), dev(table), cache, nkv, hd, PAGE)
    x = qkv.cpu().numpy().reshape(-1, hd)
    np.testing.assert_array_equal(ko.double().cpu().numpy().reshape(nkv, hd), P.held(x[nq:nq + nkv]))
    np.testing.assert_array_equal(vo.double().cpu().numpy().reshape(nkv, hd), P.held(x[nq + nkv:]))


def test_recorded_steps_and_two_at_a_time():
    """Two steps recorded into graphs with scratch of their own, replayed with eager work between and on two streams at once, give the
    eager results each time; the contexts they read change between replays."""
    nq, nkv, hd = 8, 2, 64
    c = Cache([500, 300], nkv, hd)
    c.fill()
    table, cache = c.tensors
    slots, ctx = dev(c.slots), dev([400, 200])
    pos, seq = dev([399, 199]), dev([0, 1])
    qkv = torch.randn(2, (nq + 2 * nkv) * hd, device="cuda").bfloat16()
    nsplit = 4

    def step(out, part):
        K.rope_kv4_write(qkv, None, None, pos, seq, slots, table, cache, nq, nkv, hd, 0, False, PAGE, True)
        K.attention_decode_kv4(qkv, qkv.stride(0), out, slots, ctx, table, cache, 2, nq, nkv, hd, PAGE, None, 0.1, nsplit, *part)

    outs = [torch.zeros(2, nq * hd, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    parts = [(torch.empty(2 * nq * nsplit * hd, device="cuda"), torch.empty(2 * nq * nsplit * 2, device="cuda")) for _ in range(3)]
    step(outs[2], parts[2])
    graphs = []
    for i in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(outs[i], parts[i])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(6):
        ctx += 1
        pos += 1
        qkv.copy_(torch.randn_like(qkv))
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        if i % 2:
            for g in graphs:
                g.replay()
        else:
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        step(outs[2], parts[2])
        torch.cuda.synchronize()
        assert outs[2].abs().sum() > 0
        for o in outs[:2]:
            assert torch.equal(o, outs[2])


def test_prompts_recorded_and_on_another_stream():
    nq, nkv, hd, n = 4, 1, 128, 100
    c = Cache([700], nkv, hd)
    c.fill()
    table, cache = c.tensors
    rows = torch.randn(n, nq * hd, device="cuda").bfloat16()
    part = torch.empty(n * nq * 3 * hd, device="cuda"), torch.empty(n * nq * 3 * 2, device="cuda")
    args = (dev([0, n]), dev(c.slots), dev([700]), table, cache, 1, n, nq, nkv, hd, PAGE, None, 0.1, 3, *part)
    want = torch.zeros(n, nq * hd, dtype=torch.bfloat16, device="cuda")
    K.attention_prefill_kv4(rows, nq * hd, want, *args)
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        K.attention_prefill_kv4(rows, nq * hd, out, *args)
    s.synchronize()
    assert torch.equal(out, want) and want.abs().sum() > 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.attention_prefill_kv4(rows, nq * hd, out, *args)
    for _ in range(4):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ------------------------------------------------------------------------- refusals ----
def test_refusals():
    nq, nkv, hd, n = 4, 2, 64, 5
    c = Cache([n], nkv, hd)
    table, cache = c.tensors
    pos, seq, cu = step_of([n], [0])
    slots, ctx = dev(c.slots), dev([n])
    qkv = torch.zeros(n, (nq + 2 * nkv) * hd, device="cuda", dtype=torch.bfloat16)
    out = torch.zeros(n, nq * hd, device="cuda", dtype=torch.bfloat16)
    kv = torch.zeros(n, nkv * hd, device="cuda", dtype=torch.bfloat16)
    cs = torch.zeros(n, hd // 2, device="cuda")

    def write(**over):
        a = dict(qkv=qkv, cos=None, sin=None, positions=pos, seq_of_token=seq, slots=slots, block_table=table, cache=cache, nq=nq, nkv=nkv, hd=hd,
                 rotary_dim=0, adjacent=False, page=64, write_cache=True)
        a.update(over)
        K.rope_kv4_write(**a)

    def read(**over):
        a = dict(k_out=kv, v_out=kv.clone(), positions=pos, seq_of_token=seq, slots=slots, block_table=table, cache=cache, nkv=nkv, hd=hd, page=64)
        a.update(over)
        K.kv4_read(**a)

    def one(**over):
        a = dict(q=qkv, q_stride=qkv.stride(0), out=out[:1], slots=slots, ctx_lens=ctx, block_table=table, cache=cache, B=1, nq=nq, nkv=nkv, hd=hd,
                 page=64, window=None, scale=0.1, nsplit=1)
        a.update(over)
        K.attention_decode_kv4(**a)

    def many(**over):
        a = dict(q=qkv, q_stride=qkv.stride(0), out=out, cu_seqlens=cu, slots=slots, ctx_lens=ctx, block_table=table, cache=cache, B=1, max_new=n,
                 nq=nq, nkv=nkv, hd=hd, page=64, window=None, scale=0.1, nsplit=1)
        a.update(over)
        K.attention_prefill_kv4(**a)

    for call in (write, read, one, many):
        call()
        for over in (dict(page=32), dict(cache=cache.view(torch.int8)), dict(cache=cache[:, :1].contiguous()), dict(cache=cache[:, :, :-16]),
                     dict(hd=48), dict(block_table=table.long()), dict(block_table=table.flatten()), dict(slots=slots.long()), dict(slots=slots.cpu())):
            with pytest.raises(KernelError):
                call(**over)
    shifted = torch.zeros(qkv.numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view(qkv.shape)
    for over in (dict(qkv=qkv[:, :-1].contiguous()), dict(qkv=qkv.half()), dict(qkv=shifted), dict(positions=pos[:2]), dict(positions=pos.long()),
                 dict(cos=cs), dict(cos=cs, sin=cs, rotary_dim=hd + 2), dict(cos=cs, sin=cs, rotary_dim=3), dict(cos=cs[:2], sin=cs, rotary_dim=hd),
                 dict(cos=cs.double(), sin=cs.double(), rotary_dim=hd), dict(cache=None)):
        with pytest.raises(KernelError):
            write(**over)
    for over in (dict(k_out=kv[:, :-1].contiguous()), dict(k_out=kv.float()), dict(seq_of_token=seq[:1])):
        with pytest.raises(KernelError):
            read(**over)
    scratch = torch.zeros(10, device="cuda")
    for call in (one, many):
        for over in (dict(q=qkv.float()), dict(out=out.float()), dict(window=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(nsplit=0),
                     dict(nsplit=65), dict(nsplit=2), dict(nsplit=2, part_o=scratch, part_ml=scratch), dict(nq=3), dict(q_stride=nq * hd - 8),
                     dict(q_stride=qkv.stride(0) + 4), dict(q=shifted), dict(ctx_lens=ctx.long())):
            with pytest.raises(KernelError):
                call(**over)
    for over in (dict(B=2), dict(out=out[:0])):
        with pytest.raises(KernelError):
            one(**over)
    for over in (dict(B=2), dict(max_new=n + 1), dict(cu_seqlens=cu[:1]), dict(q=qkv[:3].clone())):
        with pytest.raises(KernelError):
            many(**over)
