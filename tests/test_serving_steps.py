"""What the token-by-token path decides on the host before anything reaches a GPU: which device a plan is made
for, steps that do not match the cache.  No GPU is needed; nothing here launches a kernel."""

from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch

from ue5m3_fp4 import _native
from ue5m3_fp4.serving import PagedKVCache, operators


def test_attention_workspace_is_planned_on_the_operands_device(monkeypatch):
    """The plan depends on the device's number of SMs: it is asked for with that device current, and kept apart
    from another device's."""

    current, asked = [0], []

    class Library:
        @staticmethod
        def ue5m3_paged_attention_workspace_bytes(*sizes):
            asked.append(current[0])
            return 1000 * (current[0] + 1) + sizes[0]

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    monkeypatch.setattr(_native, "load", Library)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    operators._workspace_bytes.cache_clear()
    try:
        assert operators._workspace_bytes(0, 5, 1) == 1005
        assert operators._workspace_bytes(1, 5, 1) == 2005
        current[0] = 1
        assert operators._workspace_bytes(0, 5, 1) == 1005 and operators._workspace_bytes(0, 6, 1) == 1006
        assert asked == [0, 1, 0] and current[0] == 1
    finally:
        operators._workspace_bytes.cache_clear()


def test_steps_without_all_their_tokens_are_refused():
    """Fewer ids or query rows than the step has tokens: the last rows of some sequences would be read from
    behind the tensors, and their keys would be missing from the cache."""

    from ue5m3_fp4.integrations.torchtitan.shaped_stack import NemotronHShapedStack, ShapedConfig

    cache = PagedKVCache(layers=1, pages=8, page_size=16, kv_heads=1, head_dim=64, sequences=2, max_length=64, device="cpu")
    assert cache.step_tokens == 0
    cache.begin_step([3, 2])
    assert cache.step_tokens == 5
    rows = torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="5 tokens"):
        cache.attend(0, rows, rows, rows)
    model = NemotronHShapedStack(ShapedConfig(hidden_size=64, intermediate_size=64, mamba_inner=64, mamba_extra=16, attention_heads=1,
                                              kv_heads=1, head_dim=64, vocab_size=10, num_hidden_layers=2,
                                              hybrid_override_pattern="M*"), device="cpu")
    for ids in (torch.zeros(4, dtype=torch.int64), torch.zeros(1, 5, dtype=torch.int64), torch.zeros(0, dtype=torch.int64)):
        with pytest.raises(ValueError, match="5 tokens"):
            model.serve(ids, cache)
    with pytest.raises(RuntimeError, match="begin_step"):
        model.serve(torch.zeros(5, dtype=torch.int64), model.make_cache(sequences=2, max_length=16))
    # refused steps leave the cache as it was; padding behind the step's tokens is taken (and gets as far as the GPU)
    assert cache.lengths == (3, 2)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        cache.attend(0, torch.zeros(7, 1, 64, dtype=torch.bfloat16), rows, rows)


def test_expanded_pages_and_scales_out_of_range_are_refused():
    """Pages that share memory would be written to by several keys at a time; a scale above 2^126 would be infinite
    once log2(e) is in it."""

    pages = torch.zeros(1, 16, 2, 64, dtype=torch.bfloat16)
    assert operators._strides("k_pages", pages) == (2048, 128, 64)
    assert operators._strides("k_pages", torch.zeros(5, 16, 1, 128, dtype=torch.bfloat16)[:, :, :, :64]) == (2048, 128, 64)
    for bad in (pages.expand(4, 16, 2, 64), pages[:, :1].expand(1, 16, 2, 64), pages[:, :, :1].expand(1, 16, 2, 64)):
        with pytest.raises(ValueError, match="expanded"):
            operators._strides("k_pages", bad)
    assert operators._strides("new_k", torch.zeros(3, 1, 64, dtype=torch.bfloat16).expand(3, 4, 64)) == (64, 0)
    library, fake = _native.load(), 0x10000
    cache = _native.PagedCache(fake, fake, 1024, 64, 64, 1024, 64, 64, 4, 16, 1, 64, fake, 1, 2, 2)
    for scale in (2.0 ** 127, 3e38):
        assert library.ue5m3_paged_attention(fake, 128, 64, 1, 2, ctypes.byref(cache), fake, fake, 1, 32, scale, None, 0, 0, None, 0, 0,
                                             fake, 1, None, 0, None, None) == 1
