"""The cache held in 4 bits, without a GPU: the format itself, sizes, options, and calls that are refused."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import plain_kv4 as P4
from conftest import TINY_A, TINY_B
from cuinfer_b200 import kernels
from cuinfer_b200.cache import CacheGroupSpec, CacheStorage, page_bytes
from cuinfer_b200.config import ConfigError, EngineConfig


@pytest.mark.parametrize("kind", ["normal", "shifted", "positive", "negative", "one large", "zeros", "tiny", "huge", "ties"])
def test_a_group_comes_back_within_half_a_step(kind):
    rng = np.random.default_rng(3)
    for trial in range(50):
        x = rng.standard_normal(32)
        x = {"normal": x, "shifted": x + 7, "positive": np.abs(x), "negative": -np.abs(x), "one large": np.where(np.arange(32) == trial % 32, 900 * x, x),
             "zeros": 0 * x, "tiny": x * 1e-39, "huge": np.clip(x, -3, 3) * 2.0 ** 125, "ties": np.rint(2 * x) / 2}[kind].astype(np.float32)
        codes, word = P4.quantise_group(x)
        step = P4.value(1 + (word & 15), word)
        assert 0 <= min(codes) and max(codes) <= 15 and word >> 15 == 0
        for c, v in zip(codes, x):
            got = P4.value(c, word)
            assert abs(got - float(v)) <= step / 2 * (1 + 2.0 ** -20)
            assert float(torch.tensor(got, dtype=torch.float64).to(torch.bfloat16)) == got          # exact in bfloat16
        if kind != "tiny" and kind != "zeros":
            assert step <= 1.126 * (float(max(0, x.max())) - float(min(0, x.min()))) / 15          # rounded up by at most an eighth


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 2.0 ** 127, -2.0 ** 127])
def test_a_group_with_a_number_that_does_not_fit_reads_as_nan(bad):
    x = np.ones(32, dtype=np.float32)
    x[5] = bad
    codes, word = P4.quantise_group(x)
    assert all(np.isnan(P4.value(c, word)) for c in codes)


@pytest.mark.parametrize("d", [32, 96, 128])
def test_blocks_hold_every_value_once(d):
    rng = np.random.default_rng(d)
    keys, values = (rng.standard_normal((16, d)).astype(np.float32) for _ in range(2))
    block = P4.write_block(keys, values, d)
    for rows, got in zip((keys, values), P4.read_block(block, d)):
        for token in range(16):
            for g in range(d // 32):
                codes, word = P4.quantise_group(rows[token][32 * g:32 * g + 32])
                assert [P4.value(c, word) for c in codes] == got[token][32 * g:32 * g + 32].tolist()


def test_cache_shapes_and_page_bytes():
    assert kernels.kv4_cache_shape(7, 8, 32, 128) == (7, 8, 2, 2304)
    group = CacheGroupSpec((0, 1, 2), 8, 128)
    assert page_bytes(group, 16, torch.bfloat16, True) == 3 * 8 * 2304
    assert page_bytes(group, 16, torch.bfloat16) * 9 == page_bytes(group, 16, torch.bfloat16, True) * 32      # 16 bits against 4.5
    storage = CacheStorage([group], 32, [4], {}, 3, torch.bfloat16, "cpu", kv4=True)
    assert storage.run_cache[1].shape == (4, 8, 2, 2304) and storage.run_cache[1].dtype == torch.uint8
    with pytest.raises(ValueError):
        CacheStorage([CacheGroupSpec((0,), 1, 128, planes=1)], 16, [4], {}, 3, torch.bfloat16, "cpu", kv4=True)
    for d, page in ((48, 16), (0, 16), (288, 16), (128, 8), (128, 24), (128, 0)):
        assert not kernels.kv4_supports(d, page)
        with pytest.raises(kernels.KernelError, match="head size"):
            kernels.kv4_cache_shape(1, 1, page, d)


def test_engine_options():
    assert EngineConfig(kv_cache_dtype="int4", block_size=48).kv_cache_dtype == "int4" and EngineConfig().kv_cache_dtype == "auto"
    with pytest.raises(ConfigError, match="kv_cache_dtype"):
        EngineConfig(kv_cache_dtype="fp8")
    with pytest.raises(ConfigError, match="multiple of 16"):
        EngineConfig(kv_cache_dtype="int4", block_size=24)


def test_which_models_take_it():
    from cuinfer_b200.config.registry import architecture_of
    from cuinfer_b200.parts import DecoderModel

    def mixers(cfg):
        arch = architecture_of(cfg)
        return [b.mixer for b in DecoderModel(arch.spec(arch.parse(cfg)), torch.float32).blocks]

    assert all(m.takes_kv4(32) for m in mixers(TINY_B))                # head size 32
    assert not any(m.takes_kv4(16) for m in mixers(TINY_A))            # head size 16
    assert not any(m.takes_kv4(8) for m in mixers(TINY_B))


def _write_args(T=3, nq=4, nkv=2, d=64, dtype=torch.float32):
    qkv = torch.zeros(T, (nq + 2 * nkv) * d, dtype=dtype)
    return dict(qkv=qkv, positions=torch.zeros(T, dtype=torch.int32), slot_mapping=torch.zeros(T, dtype=torch.int32), q_weight=None, k_weight=None,
                eps=1e-6, rope_table=None, rotary_dim=0, cache=torch.zeros(kernels.kv4_cache_shape(2, nkv, 16, d), dtype=torch.uint8),
                num_q_heads=nq, num_kv_heads=nkv, head_dim=d)


@pytest.mark.parametrize("change, match", [
    (dict(cache=torch.zeros(2, 2, 1, 18 * 64)), "uint8"),
    (dict(cache=torch.zeros(2, 3, 1, 18 * 64, dtype=torch.uint8)), "uint8"),
    (dict(cache=torch.zeros(2, 2, 18 * 64, dtype=torch.uint8)), "uint8"),
    (dict(qkv=torch.zeros(3, 500)), "do not hold"),
    (dict(qkv=torch.zeros(512, 3).T), "dense"),
    (dict(q_out=torch.zeros(3, 255)), "q_out"),
    (dict(q_out=torch.zeros(3, 256, dtype=torch.bfloat16)), "q_out"),
    (dict(positions=torch.zeros(2, dtype=torch.int32)), "each of the 3"),
    (dict(slot_mapping=torch.zeros(2, dtype=torch.int32)), "each of the 3"),
    (dict(q_weight=torch.ones(64)), "both"),
    (dict(k_weight=torch.ones(64)), "both"),
    (dict(q_weight=torch.ones(64), k_weight=torch.ones(64, dtype=torch.bfloat16)), "one dtype"),
    (dict(q_weight=torch.ones(32), k_weight=torch.ones(32)), "64 elements"),
    (dict(rope_table=torch.zeros(9, 32, 2), rotary_dim=32), "rope table"),
])
def test_write_refuses(change, match):
    with pytest.raises(kernels.KernelError, match=match):
        kernels.qk_norm_rope_kv4_write(**{**_write_args(), **change})


@pytest.mark.parametrize("change, match", [
    (dict(keys=torch.zeros(3, 127)), "keys"),
    (dict(values=torch.zeros(2, 128)), "values"),
    (dict(values=torch.zeros(3, 128, dtype=torch.bfloat16)), "values"),
    (dict(cache=torch.zeros(2, 2, 1, 17 * 64, dtype=torch.uint8)), "uint8"),
])
def test_read_refuses(change, match):
    args = dict(cache=torch.zeros(kernels.kv4_cache_shape(2, 2, 16, 64), dtype=torch.uint8), slots=torch.zeros(3, dtype=torch.int32),
                keys=torch.zeros(3, 128), values=torch.zeros(3, 128), num_kv_heads=2, head_dim=64)
    with pytest.raises(kernels.KernelError, match=match):
        kernels.kv4_read(**{**args, **change})


@pytest.mark.parametrize("change, match", [
    (dict(cache=torch.zeros(2, 2, 1, 18 * 64)), "uint8"),
    (dict(num_q_heads=5), "do not share"),
    (dict(q=torch.zeros(3, 255)), "dense"),
    (dict(out=torch.zeros(3, 255)), "dense"),
    (dict(out=torch.zeros(3, 256, dtype=torch.bfloat16)), "out be"),
    (dict(query_start_loc=torch.zeros(2, dtype=torch.int32)), "query_start_loc"),
    (dict(block_table=torch.zeros(1, 1, dtype=torch.int32)), "block_table"),
    (dict(query_lens_host=[3]), "query_lens_host"),
    (dict(window=-1), "window"),
    (dict(max_seq_len=-1), "max_seq_len"),
])
def test_attention_refuses(change, match):
    args = dict(q=torch.zeros(3, 256), out=torch.zeros(3, 256), cache=torch.zeros(kernels.kv4_cache_shape(2, 2, 16, 64), dtype=torch.uint8),
                block_table=torch.zeros(2, 1, dtype=torch.int32), query_start_loc=torch.tensor([0, 1, 3], dtype=torch.int32),
                seq_lens=torch.tensor([1, 2], dtype=torch.int32), query_lens_host=[1, 2], num_q_heads=4, num_kv_heads=2, head_dim=64,
                scale=0.125, max_seq_len=2)
    with pytest.raises(kernels.KernelError, match=match):
        kernels.paged_attention_kv4(**{**args, **change})


def test_tensors_that_are_not_on_the_device_are_refused():
    with pytest.raises(kernels.KernelError, match="CUDA"):
        kernels.qk_norm_rope_kv4_write(**_write_args())


@pytest.mark.parametrize("change, match", [
    (dict(window=1 << 31), "window"),
    (dict(max_seq_len=1 << 32), "max_seq_len"),
    (dict(num_q_heads=0), "do not share"),
    (dict(num_kv_heads=0, cache=torch.zeros(2, 0, 1, 18 * 64, dtype=torch.uint8)), "do not share"),
])
def test_attention_refuses_sizes_out_of_range(change, match):
    test_attention_refuses(change, match)
