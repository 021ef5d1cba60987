"""Into how many runs the pages of 4-bit keys and values are cut, on the CPU: the rule for each of the two kernels."""
import pytest

from braidinfer_amd import kernels as K


@pytest.fixture(autouse=True)
def units(monkeypatch):
    monkeypatch.setattr(K, "device_cus", lambda: 256)


@pytest.mark.parametrize("n_seqs,nq,nkv,hd,ctx,window", [(8, 32, 8, 128, 32768, None), (64, 32, 8, 128, 2048, None), (4, 16, 8, 64, 8000, None),
                                                         (1, 32, 8, 128, 32768, None), (16, 32, 4, 256, 4000, None), (8, 32, 8, 128, 40000, 4096), (300, 8, 8, 32, 900, 1)])
def test_prompts_of_one_token_each_are_cut_as_prompts(n_seqs, nq, nkv, hd, ctx, window):
    one = K.attention_kv4_splits(n_seqs, 1, nq, nkv, hd, ctx, window, False)
    # as many workgroups as fill the device once: a tile a sequence and kv head (two of them a unit for heads of up to 64)
    assert one == 1 or one * n_seqs * nkv <= 256 * (2 if hd <= 64 else 1)
    # as few or as many as of two tokens each, which take the same tiles and pages, but for what the sums of twice the rows cost
    two = K.attention_kv4_splits(n_seqs, 2, nq, nkv, hd, ctx, window)
    assert two <= one <= 2 * two


def test_single_tokens_keep_their_rule():
    for n_seqs in (1, 8, 64):
        for ctx in (64, 1088, 2048, 40000):
            for window in (None, 1, 4096):
                want = K.attention_kv4_splits(n_seqs, 1, 32, 8, 128, ctx, window)
                assert K.attention_kv4_splits(n_seqs, 1, 32, 8, 128, ctx, window, True) == want
                assert K.attention_kv4_splits(n_seqs, 67, 32, 8, 128, ctx + 66, window, False) == K.attention_kv4_splits(n_seqs, 67, 32, 8, 128, ctx + 66, window)
    assert K.attention_kv4_splits(8, 1, 32, 8, 128, 32768) == 64 and K.attention_kv4_splits(8, 1, 32, 8, 128, 32768, None, False) == 4
