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
