"""Whole models whose keys and values are held in 4 bits, against the plain implementation over the rows that the cache holds."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import braidinfer_amd as B
import plain_kv4
import plain_mistral as P
from braidinfer_amd.engine import StepEntry
from braidinfer_amd.errors import CacheError, ConfigError

pytestmark = pytest.mark.gpu

# groups of 2, 4 and 5; windows shorter and longer than a page, on some layers; both pairings; 32 to 128 channels a head
CONFIGS = {
    "window": dict(num_hidden_layers=3, hidden_size=96, num_attention_heads=6, num_key_value_heads=3, head_dim=32, intermediate_size=320,
                   vocab_size=384, rope_theta=1e6, rms_norm_eps=1e-6, sliding_window=8, max_position_embeddings=4096),
    "plain": dict(num_hidden_layers=2, hidden_size=256, num_attention_heads=8, num_key_value_heads=2, head_dim=128, intermediate_size=512,
                  vocab_size=301, rope_theta=1e4, rms_norm_eps=1e-5, max_position_embeddings=4096),
    "mixed": dict(num_hidden_layers=4, hidden_size=160, num_attention_heads=5, num_key_value_heads=1, head_dim=96, intermediate_size=200,
                  vocab_size=256, rope_theta=5e5, rms_norm_eps=3e-6, sliding_window=70, max_position_embeddings=2048, rope_pairing="adjacent",
                  layer_types=["sliding_attention", "full_attention", "sliding_attention", "full_attention"], tie_word_embeddings=True),
}


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    made = {}

    def get(name):
        if name not in made:
            folder = str(tmp_path_factory.mktemp("kv4_" + name))
            B.Engine.write_random_folder(folder, B.MistralConfig.from_dict(CONFIGS[name]), seed=5, std=0.08, vector_jitter=0.3)
            made[name] = (B.Engine.from_folder(folder, max_tokens=4096, kv_cache="mxfp4"), folder, *P.read_folder(folder))
        return made[name]
    return get


def logits_over(eng, slot, cfg, w, tokens, monkeypatch):
    """The plain implementation's logits with keys and values read from the engine's cache, layer by layer; the rows themselves have to be
    the plain ones within the format's steps and the bound of the bfloat16 path (3e-2 of the largest element)."""
    layer = [0]
    plain = P.attention

    def attention(q, k, v, nq, nkv, window=None, scale=None, rnd=P._same):
        first, kk, vv = (x if isinstance(x, int) else x.float().cpu().numpy() for x in eng.cache_rows(slot, layer[0]))
        layer[0] += 1
        T = len(tokens)
        out = []
        for held, own in ((kk, k), (vv, v)):
            own = own.reshape(T, nkv, -1)
            x = np.abs(own).reshape(T, nkv, -1, 32)
            # a value's nearest is within 2 of the block's steps beyond 6, 1 beyond 4, half a step below
            near = 3e-2 * np.abs(own).max()
            step = 2.0 ** (np.floor(np.log2(np.maximum(x.max(-1, keepdims=True) + near, 1e-30))) - 2)
            room = (step * np.where(x + near > 5 * step, 2.0, np.where(x + near > 2 * step, 1.0, 0.5))).reshape(own.shape)
            assert (np.abs(held - own[first:]) <= room[first:] + near).all()
            full = own.copy()
            full[first:] = held
            out.append(full.reshape(k.shape if own is not v else v.shape))
        return plain(q, out[0], out[1], nq, nkv, window, scale, rnd)

    monkeypatch.setattr(P, "attention", attention)
    got = P.forward(cfg, w, tokens, act_dtype="bfloat16")
    monkeypatch.undo()
    return got


def close(got, want):
    for g, w in zip(got, want):
        assert np.abs(g - w).max() <= 3e-2 * np.abs(w).max()
        assert (g * w).sum() / np.sqrt((g * g).sum() * (w * w).sum()) >= 0.999


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_prompts_portions_and_tokens(models, monkeypatch, name):
    eng, _, cfg, w = models(name)
    rng = np.random.default_rng(1)
    tokens = [int(t) for t in rng.integers(0, cfg["vocab_size"], 60)]
    # short enough that nothing of a window has been given back where the comparison wants all rows
    for cuts in ([60], [7, 1, 30, 22], [50] + [1] * 10):
        slot = eng.alloc_slot()
        at, got = 0, []
        for n in cuts:
            got.append(eng.step([StepEntry(slot, tokens[at:at + n], range(n))]).cpu().numpy())
            at += n
        close(np.concatenate(got), logits_over(eng, slot, cfg, w, tokens, monkeypatch))
        eng.free_slot(slot)


def test_unequal_batches_and_pages_used_again(models, monkeypatch):
    eng, _, cfg, w = models("plain")
    rng = np.random.default_rng(2)
    for _ in range(2):
        lens = [1, 65, 130, 300]
        seqs = [[int(t) for t in rng.integers(0, cfg["vocab_size"], n + 5)] for n in lens]
        slots = [eng.alloc_slot() for _ in lens]
        got = [eng.step([StepEntry(s, q[:n], [n - 1]) for s, q, n in zip(slots, seqs, lens)]).cpu().numpy()]
        for i in range(5):                                       # recorded single-token steps
            got.append(eng.step([StepEntry(s, [q[n + i]], [0]) for s, q, n in zip(slots, seqs, lens)]).cpu().numpy())
        for b, (s, q, n) in enumerate(zip(slots, seqs, lens)):
            close([g[b] for g in got], logits_over(eng, s, cfg, w, q, monkeypatch)[n - 1:n + 5])
        # a mixed step: one sequence brings a portion, the others a token each
        more = [int(t) for t in rng.integers(0, cfg["vocab_size"], 40)]
        last = eng.step([StepEntry(slots[0], more, [39])] + [StepEntry(s, [3], [0]) for s in slots[1:]]).cpu().numpy()
        close(last[:1], logits_over(eng, slots[0], cfg, w, seqs[0] + more, monkeypatch)[-1:])
        close(last[3:], logits_over(eng, slots[3], cfg, w, seqs[3] + [3], monkeypatch)[-1:])
        for s in slots:
            eng.free_slot(s)


def test_windows_give_pages_back(models):
    """A long sequence through a window of 8: its pages go back, and the rows of the last ones are what a fresh sequence's would be."""
    eng, _, cfg, _ = models("window")
    rng = np.random.default_rng(3)
    tokens = [int(t) for t in rng.integers(0, cfg["vocab_size"], 400)]
    slot = eng.alloc_slot()
    eng.step([StepEntry(slot, tokens[:300], [])])
    for t in tokens[300:]:
        eng.step([StepEntry(slot, [t], [0])])
    first, k, v = eng.cache_rows(slot, 0)
    assert first == 384 and k.shape == (16, 3, 32)
    other = eng.alloc_slot()
    eng.step([StepEntry(other, tokens, [399])])
    a, b = eng.cache_rows(other, 0)[1], eng.cache_rows(slot, 0)[1]
    # the first layer's rows depend on their own token alone; products of one row and of many round differently
    assert a.shape == b.shape and (a.float() - b.float()).abs().max() <= 0.5 * a.float().abs().max()
    assert (a != b).float().mean() < 0.05
    eng.free_slot(slot)
    eng.free_slot(other)


def test_generation_and_the_command_line(models):
    eng, folder, cfg, _ = models("plain")
    prompts = [[1, 2, 3], [7] * 70]
    out = eng.generate(prompts, max_new_tokens=12, stop_token_ids=[])
    assert [len(o) for o in out] == [12, 12] and out == eng.generate(prompts, max_new_tokens=12, stop_token_ids=[])
    env = dict(os.environ, MODEL=folder, MAX_TOKENS="12")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "bin", "generate"), "--kv-cache", "mxfp4", "--prompt-ids", "1,2,3"], env=env, cwd=root,
                       capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr[-2000:]
    assert len(r.stdout.split()) == 12


def test_what_the_cache_takes_and_what_is_refused(models):
    eng, folder, _, _ = models("plain")
    held = sum(t.numel() * t.element_size() for g in eng.cache.groups for t in g.storage.values())
    wide = B.Engine.from_folder(folder, max_tokens=4096)
    full = sum(t.numel() * t.element_size() for g in wide.cache.groups for t in g.storage.values())
    assert held * 64 == full * 17                                  # 4.25 bits of 16
    with pytest.raises(CacheError):
        wide.cache_rows(wide.alloc_slot())
    with pytest.raises(CacheError):
        eng.cache_rows(eng.cache.n_slots + 5)
    with pytest.raises(ConfigError):
        B.Engine.from_folder(folder, dtype="float32", kv_cache="mxfp4")
    with pytest.raises(ConfigError):
        B.Engine.from_folder(folder, kv_cache="int4")


def test_recorded_steps_over_long_contexts(models, monkeypatch):
    """Contexts long enough that single tokens go over them in shares of one list, from recorded graphs, beside a short one."""
    from braidinfer_amd import kernels as K
    eng, _, cfg, w = models("plain")
    assert K.attention_kv4_splits(2, 1, 8, 2, 128, 1400) > 1
    rng = np.random.default_rng(4)
    lens = [1400, 70]
    seqs = [[int(t) for t in rng.integers(0, cfg["vocab_size"], n + 8)] for n in lens]
    slots = [eng.alloc_slot() for _ in lens]
    got = [eng.step([StepEntry(s, q[:n], [n - 1]) for s, q, n in zip(slots, seqs, lens)]).cpu().numpy()]
    for i in range(8):
        got.append(eng.step([StepEntry(s, [q[n + i]], [0]) for s, q, n in zip(slots, seqs, lens)]).cpu().numpy())
    for b, (s, q, n) in enumerate(zip(slots, seqs, lens)):
        close([g[b] for g in got], logits_over(eng, s, cfg, w, q, monkeypatch)[n - 1:n + 8])
        eng.free_slot(s)
