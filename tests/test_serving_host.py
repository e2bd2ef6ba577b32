"""What the token-by-token path does on the host: refusals, and the bookkeeping of the paged cache.
No GPU is needed; nothing here launches a kernel."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from ue5m3_fp4 import _native, serving
from ue5m3_fp4.nn import PackedFP4Linear, UE5M3Linear, pack_frozen_linears
from ue5m3_fp4.packed import PackedFP4Tensor
from ue5m3_fp4.serving.operators import decode_factor


def packed(rows=8, cols=32, block=16, blocking="row"):
    scale_rows = rows if blocking == "row" else (rows + block - 1) // block
    return PackedFP4Tensor(torch.zeros(rows, (cols + 1) // 2, dtype=torch.uint8),
                           torch.full((scale_rows, (cols + block - 1) // block), 0x78, dtype=torch.uint8), rows, cols, block,
                           blocking, 1.0, 448.0)


def test_operators_have_no_cpu_path():
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        packed().matvec(torch.ones(1, 32))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        PackedFP4Linear(packed())(torch.ones(1, 32))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        serving.sample_tokens(torch.ones(1, 8), torch.zeros(1))
    q, pages = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        serving.paged_attention(q, pages, pages, torch.zeros(1, 1, dtype=torch.int32), one, torch.tensor([0, 1]).int(),
                                max_query_length=1)


def test_decode_factor_follows_the_quantizer():
    assert decode_factor(0.0, 448.0) == 1.0
    assert decode_factor(2688.0, 448.0) == 1.0
    assert decode_factor(1e-38, 448.0) == float(torch.tensor(1.0) / torch.finfo(torch.float32).max)
    amax = torch.tensor(0.11)
    assert decode_factor(0.11, 448.0) == float(1.0 / (torch.tensor(2688.0) / amax))


def test_packed_linear_state_holds_the_tensor_scale():
    saved = PackedFP4Linear(packed(), torch.zeros(8))
    saved.tensor_amax, saved.scale_target = 0.3, 256.0
    loaded = PackedFP4Linear(packed(), torch.ones(8))
    loaded.load_state_dict(saved.state_dict())
    assert (loaded.tensor_amax, loaded.scale_target) == (0.3, 256.0) and not loaded.bias.any()
    without = {name: value for name, value in saved.state_dict().items() if name != "_extra_state"}
    with pytest.raises(RuntimeError, match="_extra_state"):
        loaded.load_state_dict(without)


def test_packed_linear_takes_frozen_weights_only():
    with pytest.raises(TypeError):
        PackedFP4Linear(torch.zeros(4, 4))
    with pytest.raises(ValueError, match="bias"):
        PackedFP4Linear(packed(), torch.zeros(3))
    layer = PackedFP4Linear(packed(), torch.zeros(8))
    assert set(layer.state_dict()) == {"codes", "scales", "bias", "_extra_state"}
    with pytest.raises(ValueError, match="input width"):
        layer(torch.ones(1, 31))
    model = torch.nn.Sequential(UE5M3Linear(64, 64, module_name="a"), torch.nn.Linear(64, 64))
    with pytest.raises(RuntimeError, match="not been frozen"):
        pack_frozen_linears(model)
    assert isinstance(model[0], UE5M3Linear)
    with pytest.raises(ValueError, match="root"):
        pack_frozen_linears(model[0])


def make_cache(**over):
    settings = dict(layers=2, pages=6, page_size=16, kv_heads=1, head_dim=64, sequences=3, max_length=64, device="cpu")
    return serving.PagedKVCache(**{**settings, **over})


@pytest.mark.parametrize("over", [dict(page_size=24), dict(head_dim=96), dict(layers=0), dict(pages=-1), dict(sequences=0),
                                  dict(max_length=0), dict(kv_heads=0), dict(pages=1.5)])
def test_cache_refuses_bad_sizes(over):
    with pytest.raises(ValueError):
        make_cache(**over)


def test_cache_hands_out_and_takes_back_pages():
    cache = make_cache()
    cache.begin_step([16, 17, 0])
    assert cache.lengths == (16, 17, 0) and cache.free_pages == 3
    table = cache.page_table.tolist()
    held = [page for row in table for page in row if page >= 0]
    assert len(set(held)) == 3 and [sum(page >= 0 for page in row) for row in table] == [1, 2, 0]
    assert cache.kv_lengths.tolist() == [16, 17, 0] and cache.query_starts.tolist() == [0, 16, 33, 33]
    assert cache.last_rows.tolist() == [15, 32, 32]
    assert (cache.max_query_length, cache.max_kv_length) == (17, 17)
    address = cache.page_table.data_ptr()
    cache.begin_step([1, 1, 1])
    assert cache.page_table.data_ptr() == address
    assert cache.lengths == (17, 18, 1) and cache.query_starts.tolist() == [0, 1, 2, 3]
    assert [row[:1] for row in cache.page_table.tolist()][:2] == [row[:1] for row in table][:2]
    before = (cache.lengths, cache.free_pages, cache.page_table.clone())
    with pytest.raises(RuntimeError, match="free pages"):
        cache.begin_step([20, 20, 20])
    with pytest.raises(RuntimeError, match="max_length"):
        cache.begin_step([48, 0, 0])
    for wrong in ([1, 1], [0, 0, 0], [1, -1, 1]):
        with pytest.raises(ValueError):
            cache.begin_step(wrong)
    assert (cache.lengths, cache.free_pages) == before[:2] and torch.equal(cache.page_table, before[2])
    cache.release(1)
    assert cache.lengths == (17, 0, 1) and cache.free_pages == 3
    cache.begin_step([0, 40, 0])
    assert cache.lengths == (17, 40, 1) and cache.free_pages == 0
    held = [page for row in cache.page_table.tolist() for page in row if page >= 0]
    assert sorted(held) == list(range(6))
    with pytest.raises(IndexError):
        cache.release(3)
    with pytest.raises(RuntimeError, match="begin_step"):
        make_cache().attend(0, None, None, None)


def test_library_refuses_bad_arguments():
    lib = _native.load()
    fake, odd = 0x10000, 0x10001

    def matvec(**over):
        a = dict(x=fake, x_dtype=0, tokens=1, ldx=64, codes=fake, scales=fake, rows=8, cols=64, block=16, two_d=0, dec=1.0,
                 bias=None, bias_dtype=0, out=fake, out_dtype=0, ldo=8, workspace=None,
                 workspace_bytes=0) | over
        return lib.ue5m3_packed_matvec(*a.values(), None)

    assert matvec(x=None) == matvec(codes=None) == matvec(scales=None) == matvec(out=None) == 1
    assert matvec(tokens=0) == matvec(rows=0) == matvec(cols=0) == matvec(ldx=63) == matvec(ldo=7) == matvec(x_dtype=2) == 1
    assert matvec(block=8) == 2
    assert matvec(x=odd) == matvec(out=odd) == matvec(bias=odd) == 4
    assert matvec(cols=1 << 23, ldx=1 << 23) == 8
    # more than eight tokens take a workspace
    need = lib.ue5m3_packed_matvec_workspace_bytes(0, 9, 64)
    assert need > 0 and lib.ue5m3_packed_matvec_workspace_bytes(0, 8, 64) == 0
    assert lib.ue5m3_packed_matvec_workspace_bytes(1, 9, 64) > need
    assert matvec(tokens=9) == matvec(tokens=9, workspace=fake, workspace_bytes=need - 1) == 7
    assert matvec(tokens=9, workspace=fake + 8, workspace_bytes=need) == 4

    def attention(cache_over=None, **over):
        c = dict(k_pages=fake, v_pages=fake, k_page_stride=1024, k_slot_stride=64, k_head_stride=64, v_page_stride=1024,
                 v_slot_stride=64, v_head_stride=64, pages=4, page_size=16, kv_heads=1, head_dim=64, page_table=fake, sequences=1,
                 table_width=2, table_stride=2) | (cache_over or {})
        a = dict(q=fake, q_token=128, q_head=64, tokens=1, heads=2, cache=ctypes.byref(_native.PagedCache(*c.values())),
                 kv_lengths=fake, query_starts=fake, max_query=1, max_kv=32, scale=0.125, new_k=None, nkt=0, nkh=0, new_v=None,
                 nvt=0, nvh=0, out=fake, zero_tail=1, workspace=None, workspace_bytes=0, status=None) | over
        return lib.ue5m3_paged_attention(*a.values(), None)

    assert attention(q=None) == attention(kv_lengths=None) == attention(query_starts=None) == attention(out=None) == 1
    assert attention({"k_pages": None}) == attention({"v_pages": None}) == attention({"page_table": None}) == 1
    assert attention(new_k=fake) == attention(new_v=fake) == 1
    assert attention(scale=math.nan) == attention(scale=0.0) == attention(scale=-1.0) == attention(scale=math.inf) == 1
    assert attention(heads=3, cache_over={"kv_heads": 2}) == attention({"head_dim": 96}) == attention(tokens=0) == 1
    assert attention(max_query=0) == attention(max_kv=0) == attention({"pages": 0}) == attention({"table_stride": 1}) == 1
    assert attention({"page_size": 48}) == attention({"page_size": 8}) == attention({"page_size": 512}) == 5
    assert attention({"sequences": 70000}) == attention({"table_width": 1 << 28, "table_stride": 1 << 28}) == 8
    assert attention({"k_slot_stride": 68}) == attention(q_token=100) == attention(q=fake + 8) == attention(out=fake + 8) == 4
    assert attention({"v_head_stride": -64}) == 4
    # a long sequence is split: without its workspace the call is refused
    long = dict(pages=4096, table_width=4096, table_stride=4096)
    need = lib.ue5m3_paged_attention_workspace_bytes(1, 1, 2, 1, 64, 1, 65536)
    assert need > 0 and attention(long, max_kv=65536) == 7
    assert attention(long, max_kv=65536, workspace=fake, workspace_bytes=need - 1) == 7
    assert lib.ue5m3_paged_attention_workspace_bytes(1, 1, 2, 1, 64, 1, 64) == 0
    assert lib.ue5m3_paged_attention_workspace_bytes(1, 1, 3, 2, 64, 1, 64) == 0

    def sample(**over):
        a = dict(logits=fake, dtype=1, rows=1, vocabulary=100, ld=100, uniforms=fake, td=None, t=1.0, kd=None, k=0, pd=None,
                 p=1.0, md=None, m=0.0, tokens=fake, logprobs=fake) | over
        return lib.ue5m3_sample_tokens(*a.values(), None)

    assert sample(logits=None) == sample(uniforms=None) == sample(tokens=None) == sample(logprobs=None) == 1
    assert sample(rows=0) == sample(vocabulary=0) == sample(ld=99) == sample(dtype=3) == 1
    assert sample(vocabulary=(1 << 18) + 1, ld=1 << 19) == 8
    assert sample(logits=odd) == 4
