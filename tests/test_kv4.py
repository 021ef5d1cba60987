"""4-bit keys and values, on the CPU: the number format by its definition, and what the entry points refuse."""
import ctypes

import numpy as np
import pytest
import torch

import plain_kv4 as P
from braidinfer_amd import kernels as K
from braidinfer_amd.errors import KernelError


def test_blocks_by_the_definition():
    x = np.zeros(32, dtype=np.float32)
    x[:12] = [8 - 2 ** -20, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.2500001, 4.999, 5.001, -0.0]
    codes, s = P.block(x)
    assert s == 127
    assert P.value(codes, s)[:12].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -0.5, 4, 6, 0]      # ties to the even code
    assert P.block(np.zeros(32))[1] == 3 and P.block(np.full(32, 1e-45))[1] == 3
    assert P.block(np.full(32, 3.3e38))[1] == 252 and P.block(np.array([np.inf] + [0.0] * 31))[1] == 255
    for e in range(-120, 125, 7):                                                          # the largest element within [4, 8) steps
        codes, s = P.block(np.full(32, 1.999 * 2.0 ** e))
        assert s - 127 == e - 2


@pytest.mark.parametrize("hd", [0, 16, 48, 100, 288, 512])
def test_head_sizes_that_are_refused(hd):
    with pytest.raises(KernelError, match="multiple of 32"):
        K.kv4_head_bytes(hd)


def test_tensors_off_the_gpu_are_refused():
    z = torch.zeros
    i = z(1, dtype=torch.int32)
    cache = z(1, 1, 68 * 32, dtype=torch.uint8)
    table = z(1, 1, dtype=torch.int32)
    row = z(1, 96, dtype=torch.bfloat16)
    out = z(1, 32, dtype=torch.bfloat16)
    with pytest.raises(KernelError, match="GPU only"):
        K.rope_kv4_write(row, None, None, i, i, i, table, cache, 1, 1, 32, 0, False, 64, True)
    with pytest.raises(KernelError, match="GPU only"):
        K.kv4_read(out, out, i, i, i, table, cache, 1, 32, 64)
    with pytest.raises(KernelError, match="GPU only"):
        K.attention_decode_kv4(row, 96, out, i, i, table, cache, 1, 1, 1, 32, 64, None, 1.0, 1)
    with pytest.raises(KernelError, match="GPU only"):
        K.attention_prefill_kv4(row, 96, out, z(2, dtype=torch.int32), i, i, table, cache, 1, 1, 1, 1, 32, 64, None, 1.0, 1)


def _entry(module, name):
    from braidinfer_amd.csrc import build
    return getattr(build.load(module), name)


# sizes that no kernel takes come back as an error before anything is launched (the entry points look at no pointer here)
@pytest.mark.parametrize("hd,nq,nkv,B,nsplit", [(48, 4, 2, 1, 1), (288, 4, 2, 1, 1), (128, 5, 2, 1, 1), (128, 4, 0, 1, 1), (128, 4, 2, 65536, 1),
                                                (128, 4, 2, 1, 0), (128, 4, 2, 1, 65), (128, 4, 2, 1, 2), (128, 4, 2, -1, 1)])
def test_sizes_that_the_attention_entry_points_refuse(hd, nq, nkv, B, nsplit):
    P_, I, Z, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_float
    d = _entry("attention_kv4", "br_attn_decode_kv4")
    d.argtypes = [P_, Z, P_, P_, P_, P_, I, I, P_] + [I] * 6 + [F, I, P_, P_, P_]
    assert d(0, nq * hd, 0, 0, 0, 0, 1, 1, 0, 1, B, nq, nkv, hd, 0, 1.0, nsplit, 0, 0, 0) == 1
    f = _entry("attention_kv4", "br_attn_prefill_kv4")
    f.argtypes = [P_, Z, P_, P_, P_, P_, P_, I, I, P_] + [I] * 8 + [F, I, P_, P_, P_]
    assert f(0, nq * hd, 0, 0, 0, 0, 0, 1, 1, 0, 1, B, 5, 5, nq, nkv, hd, 0, 1.0, nsplit, 0, 0, 0) == 1


def test_sizes_that_the_cache_entry_points_refuse():
    P_, I = ctypes.c_void_p, ctypes.c_int
    w = _entry("kv4_cache", "br_rope_kv4_write")
    w.argtypes = [P_, I, P_, P_, P_, P_, P_, I, P_, I, I, P_] + [I] * 8 + [P_]
    for hd, nkv, rd in [(48, 1, 0), (512, 1, 0), (64, 0, 0), (64, 1, 65), (64, 1, 66), (64, 1, -2)]:
        assert w(0, 1, 0, 0, 0, 0, 0, 1, 0, 1, 1, 0, 1, 4, 1, nkv, hd, rd, 0, 1, 0) == 1
    r = _entry("kv4_cache", "br_kv4_read")
    r.argtypes = [P_, P_, I, P_, P_, P_, I, P_, I, I, P_] + [I] * 4 + [P_]
    assert r(0, 0, 1, 0, 0, 0, 1, 0, 1, 1, 0, 1, 4, 1, 80, 0) == 1
    # no tokens: nothing to do
    assert w(0, 1, 0, 0, 0, 0, 0, 1, 0, 1, 1, 0, 1, 0, 1, 1, 64, 0, 0, 1, 0) == 0
    assert r(0, 0, 1, 0, 0, 0, 1, 0, 1, 1, 0, 1, 0, 1, 64, 0) == 0


def test_models_that_can_hold_keys_and_values_in_4_bits():
    import braidinfer_amd as B
    from braidinfer_amd.config import spec_of, with_kv_cache
    from braidinfer_amd.engine import DecoderModel
    from braidinfer_amd.errors import ConfigError
    spec = spec_of(B.preset("mistral-7b-v0.1", num_hidden_layers=2))
    assert with_kv_cache(spec, None) is spec
    needs = DecoderModel(with_kv_cache(spec, "mxfp4")).cache_needs()
    assert [n.held for n in needs.values()] == ["mxfp4"] * 2 and needs[0].window == 4096
    assert all(n.held is None for n in DecoderModel(spec).cache_needs().values())
    with pytest.raises(ConfigError, match="int8"):
        with_kv_cache(spec, "int8")
    with pytest.raises(ConfigError, match="gqa_attention"):
        with_kv_cache(spec_of(B.any_preset("kesitar-tiny")), "mxfp4")
    with pytest.raises(ConfigError, match="head_dim in steps of 32"):
        DecoderModel(with_kv_cache(spec_of(B.preset("tiny-a")), "mxfp4"))
    from braidinfer_amd.parts.attention import GQAAttention
    from braidinfer_amd.parts import Runtime
    part = GQAAttention(64, 2, 1, 32, kv_cache="mxfp4")
    with pytest.raises(ConfigError, match="bfloat16"):
        part.load({}, "", Runtime(device=torch.device("cpu"), dtype=torch.float32))
    with pytest.raises(ConfigError):
        GQAAttention(64, 2, 1, 32, kv_cache="mxfp8")


def test_mixers_side_by_side_are_both_held_in_4_bits():
    from dataclasses import replace
    import braidinfer_amd as B
    from braidinfer_amd.config import LayerSpec, PartSpec, spec_of, with_kv_cache
    mixer = PartSpec("gqa_attention", {"hidden_size": 64, "num_heads": 2, "num_kv_heads": 1, "head_dim": 32})
    spec = replace(spec_of(B.preset("mistral-7b-v0.1", num_hidden_layers=2)),
                   layers=[LayerSpec(prefix="a."), LayerSpec(prefix="b.", mixer=mixer, more_mixers={"right": mixer})])
    got = with_kv_cache(spec, "mxfp4").layers
    assert got[0].mixer is None and got[1].mixer.params["kv_cache"] == got[1].more_mixers["right"].params["kv_cache"] == "mxfp4"
    assert "kv_cache" not in mixer.params


def test_units_held_in_4_bits():
    from braidinfer_amd.cache import CacheNeed, SequenceCache
    from braidinfer_amd.errors import CacheError
    c = SequenceCache({0: CacheNeed(3, 64, held="mxfp4"), 1: CacheNeed(3, 64), 2: CacheNeed(3, 64, held="mxfp4")}, {}, max_tokens=200,
                      dtype=torch.bfloat16)
    assert len(c.groups) == 2                                             # another form is another group
    g = c.unit_group(0)
    assert g.storage[2].shape == (4, 3, 68 * 64) and g.storage[2].dtype == torch.uint8
    assert c.unit_storage(0) is g.storage[0] and g.keys(0) is None and g.values(0) is None
    assert c.unit_storage(1).shape == (4, 2, 3, 64, 64) and c.unit_group(1).keys(1) is not None
    s = c.alloc_slot()
    c.reserve([s], [130])
    c.commit([s], [130])
    assert [len(x.pages[s]) for x in c.groups] == [3, 3]
    for bad in (CacheNeed(1, 48, held="mxfp4"), CacheNeed(1, 288, held="mxfp4"), CacheNeed(1, 64, value_dim=32, held="mxfp4"), CacheNeed(1, 64, held="fp8"),
                CacheNeed(1, 64, tokens_per_row=2, held="mxfp4")):
        with pytest.raises(CacheError, match="mxfp4"):
            SequenceCache({0: bad}, {}, max_tokens=64, dtype=torch.bfloat16)
    with pytest.raises(CacheError, match="pages of 64"):
        SequenceCache({0: CacheNeed(1, 64, held="mxfp4")}, {}, max_tokens=64, page_tokens=32, dtype=torch.bfloat16)
