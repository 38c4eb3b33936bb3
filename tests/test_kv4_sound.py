"""The cache held in 4 bits, without a GPU: memory that is set aside, and calls that are refused."""
from __future__ import annotations

import random

import pytest
import torch

from conftest import TINY_B, TINY_D
from cuinfer_b200 import kernels
from cuinfer_b200.config import EngineConfig


def runner_without_a_device(cfg, dtype, kv4, **options):
    """A runner that has a model and options and nothing on a device."""
    from cuinfer_b200.config.registry import architecture_of
    from cuinfer_b200.engine.runner import ModelRunner
    from cuinfer_b200.parts import DecoderModel
    arch = architecture_of(cfg)
    runner = object.__new__(ModelRunner)
    runner.model = DecoderModel(arch.spec(arch.parse(cfg)), dtype)
    runner.config = EngineConfig(kv_cache_dtype="int4" if kv4 else "auto", **options)
    runner.kv4, runner.vocab_size = kv4, cfg["vocab_size"]
    return runner


def test_the_scratch_of_the_attention_is_set_aside():
    """Partial results of shared prompts and of single tokens in an even list are no pages: once for steps as they come, once for recorded ones."""
    for graphs, times in ((False, 1), (True, 2)):
        plain, kv4 = (runner_without_a_device(TINY_D, torch.bfloat16, kv, enable_cuda_graph=graphs, max_num_scheduled_tokens=4096)._activation_bytes() for kv in (False, True))
        assert kv4 - plain >= times * 4 * (1 << 24)
    assert (runner_without_a_device(TINY_D, torch.float32, True)._activation_bytes()
            == runner_without_a_device(TINY_D, torch.float32, False)._activation_bytes())
    assert (runner_without_a_device(TINY_B, torch.bfloat16, True)._activation_bytes()         # head size 32: joined in shared memory
            == runner_without_a_device(TINY_B, torch.bfloat16, False)._activation_bytes())


def test_no_launch_needs_more_scratch():
    rng = random.Random(1)
    lib = kernels.library()
    for _ in range(3000):
        d, nkv = rng.choice([64, 128, 256]), rng.choice([1, 2, 8])
        nq, T = nkv * rng.choice([1, 2, 5, 8]), int(2 ** rng.uniform(0, 14))
        g, keys, budget = nq // nkv, int(2 ** rng.uniform(0, 20)), T + rng.randrange(5000)
        used = 0
        cluster, ctas, unit = kernels.kv4_decode_shape(rng.randrange(1, 257) * nkv, keys, lib.cib_attention_kv4_decode_ctas(d))
        if unit:
            used += 4 * lib.cib_attention_kv4_decode_scratch_floats(d, ctas)
        if d < 256:
            shares = kernels.kv4_prompt_shares((-(-T * g // 256)) * nkv, keys, T * nq * d)
            used += 4 * shares * T * nq * (d + 2) if shares > 1 else 0
        assert used <= kernels.kv4_attention_scratch_bytes(budget, nq, d, torch.bfloat16)


# ---- calls that are refused -------------------------------------------------------------------------------------------------------

def attention_args(**change):
    args = dict(q=torch.zeros(3, 256), out=torch.zeros(3, 256), cache=torch.zeros(kernels.kv4_cache_shape(2, 2, 16, 64), dtype=torch.uint8),
                block_table=torch.zeros(2, 1, dtype=torch.int32), query_start_loc=torch.tensor([0, 1, 3], dtype=torch.int32),
                seq_lens=torch.tensor([1, 2], dtype=torch.int32), query_lens_host=[1, 2], num_q_heads=4, num_kv_heads=2, head_dim=64,
                scale=0.125, max_seq_len=2)
    return {**args, **change}


def far_apart(rows, width, stride, dtype=torch.float32):
    return torch.empty_strided((rows, width), (stride, 1), dtype=dtype, device="meta")


@pytest.mark.parametrize("change, match", [
    (dict(out=torch.zeros(1, 256).expand(3, 256)), "apart"),
    (dict(out=torch.zeros(1000).as_strided((3, 256), (255, 1))), "apart"),
    (dict(out=far_apart(3, 256, 1 << 31)), "32-bit strides"),
    (dict(out=far_apart(3, 256, 1 << 33)), "32-bit strides"),
])
def test_attention_refuses_rows_that_overlap_or_lie_too_far_apart(change, match):
    with pytest.raises(kernels.KernelError, match=match):
        kernels.paged_attention_kv4(**attention_args(**change))


def test_strides_of_rows():
    """32 bits of a stride go to the kernels; of a single row nothing does."""
    assert kernels._row_stride(far_apart(2, 64, (1 << 31) - 8)) == (1 << 31) - 8
    assert kernels._row_stride(far_apart(1, 64, 1 << 40)) == 64 and kernels._row_stride(torch.zeros(5, 3, 64)[:, 1]) == 192
    for stride in (1 << 31, (1 << 32) + 64):
        with pytest.raises(kernels.KernelError, match="32-bit strides"):
            kernels._row_stride(far_apart(2, 64, stride))


def test_a_pool_has_no_more_slots_than_32_bits_number(monkeypatch):
    """One key head of 32 in one layer: 180 GB would be some 4e9 slots of 36 bytes."""
    cfg = dict(TINY_B, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1)
    for kv4, block in ((True, 16), (True, 48), (False, 16)):
        runner = runner_without_a_device(cfg, torch.bfloat16, kv4, block_size=block)
        from cuinfer_b200.cache import group_runs
        runner.groups = group_runs(runner.model.cache_needs())
        runner.page_size, runner.dtype, runner.device, runner.max_model_len = block, torch.bfloat16, "cuda:0", 768
        monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (180 << 30, 180 << 30))
        pages = runner._pages_from_memory()
        assert 0 < pages * block < 1 << 31
        if not kv4:
            assert pages * runner.page_bytes() > 140 << 30               # (128 bytes a slot: the memory ends first)
