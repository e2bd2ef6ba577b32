"""The token-by-token operators where inputs, sizes and callers are unusual: activations of very different
size side by side, weights of many rows, settings that are not numbers, graphs and streams side by side.

Tolerances count roundings, as in test_gpu_serving.py, whose plain implementations in 64 bits are used here.
"""

from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from test_gpu_serving import DTYPES, check_matvec, check_sample, packed_weight, run_attention, unpack

pytestmark = pytest.mark.gpu


# ---- packed matrix-vector products ----------------------------------------------------------------


def without_columns(codes: torch.Tensor, columns) -> torch.Tensor:
    """The weight with zeros in these columns."""

    codes = codes.clone()
    for column in columns:
        codes[:, column // 2] &= 0x0F if column % 2 else 0xF0
    return codes


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("spread", [30, 33, 40, 60, 100])
@pytest.mark.parametrize("tokens,rows,cols,block,two_d", [(1, 40, 384, 16, False), (8, 33, 1003, 32, False), (3, 150, 4096, 16, True),
                                                          (9, 130, 384, 32, True), (20, 40, 1003, 16, False), (45, 257, 640, 16, True),
                                                          (70, 20, 300, 32, False), (16, 21504, 256, 32, True),
                                                          (8, 30011, 300, 16, False), (2, 20, 140000, 16, False),
                                                          (30, 70, 9000, 32, False)])
def test_matvec_keeps_small_activations_beside_large_ones(tokens, rows, cols, block, two_d, dtype, spread):
    """Elements 2^spread times their neighbours that meet zeros of the weight: what is left is the
    neighbours' sum, to the same tolerance as without them.  Rows without such elements come out bit for
    bit as in a batch that has none."""

    from ue5m3_fp4 import serving

    g = torch.Generator().manual_seed(spread + cols)
    codes, scales = packed_weight(rows, cols, block, two_d, seed=cols)
    large = [5, 130, 131, cols // 2, cols - 1]
    codes = without_columns(codes, large)
    x = torch.randn(tokens, cols, generator=g, dtype=torch.float64)
    plain = x.clone().to(DTYPES[dtype])
    touched = list(range(0, tokens, 3))
    for t in touched:
        x[t, large] *= 2.0 ** (spread if t % 2 else 0)
        if t % 2 == 0:  # ... or the neighbours are small: same ratio
            x[t] *= 2.0 ** -spread
            x[t, large] *= 2.0 ** spread
    x = x.to(DTYPES[dtype])
    got = check_matvec(x, codes, scales, rows, cols, block, two_d, out_dtype=torch.float32, amax=448.0 * 6)
    kw = dict(rows=rows, cols=cols, block_size=block, two_dimensional=two_d, tensor_amax=448.0 * 6, out_dtype=torch.float32)
    without = serving.packed_matvec(plain.cuda(), codes.cuda(), scales.cuda(), **kw)
    others = [t for t in range(tokens) if t not in touched]
    assert torch.equal(got[others], without[others])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("tokens,rows,cols,block,two_d", [(1, 150, 4096, 16, True), (8, 300, 8192, 32, False), (5, 90, 2049, 16, False),
                                                          (64, 520, 4096, 16, True), (20, 129, 6000, 32, False)])
def test_matvec_of_squared_relus(tokens, rows, cols, block, two_d, dtype):
    """Activations as a squared-ReLU MLP makes them: half of them zero, a few very small, here and there alone in the
    columns of the weight that are not zero."""

    g = torch.Generator().manual_seed(cols)
    x = torch.relu(torch.randn(tokens, cols, generator=g)).to(torch.bfloat16).square().to(DTYPES[dtype])
    x[::2, 77::128] = 2.0 ** -40
    codes, scales = packed_weight(rows, cols, block, two_d, seed=cols)
    check_matvec(x, codes, scales, rows, cols, block, two_d)
    codes[:rows // 2] = without_columns(codes[:rows // 2], [j for j in range(cols) if j % 128 != 77])
    check_matvec(x, codes, scales, rows, cols, block, two_d, out_dtype=torch.float32, amax=448.0 * 6)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("tokens", [2, 12])
def test_matvec_of_all_exponents_in_one_chunk(tokens, dtype):
    """Elements from the type's smallest to 2^100 in one row, zeros among them; the weight is zero from 2^-60 up
    in its first half of rows, from 2^40 in the others, so that every size is the largest one somewhere."""

    rows, cols = 64, 256
    codes, scales = packed_weight(rows, cols, 16, False, seed=3)
    exponents = torch.linspace(-140, 100, cols).round()
    g = torch.Generator().manual_seed(4)
    x = (1 + torch.rand(tokens, cols, generator=g, dtype=torch.float64)) * torch.exp2(exponents.double())
    x[:, ::17] = 0
    x = (x * torch.where(torch.rand(tokens, cols, generator=g) < 0.5, -1.0, 1.0)).to(DTYPES[dtype])
    codes[:32] = without_columns(codes[:32], [j for j in range(cols) if exponents[j] >= -60])
    codes[32:] = without_columns(codes[32:], [j for j in range(cols) if exponents[j] >= 40])
    check_matvec(x, codes, scales, rows, cols, 16, False, out_dtype=torch.float32, amax=448.0 * 6)
    x[:, 0], x[0, 255] = 1.0, math.inf  # beside an infinity, in a row of its own
    check_matvec(x[1:], codes, scales, rows, cols, 16, False, out_dtype=torch.float32, amax=448.0 * 6)


@pytest.mark.parametrize("cols", [256, 255])
@pytest.mark.parametrize("block,two_d", [(16, False), (32, True)])
@pytest.mark.parametrize("tokens,rows,dtype", [(16, 21504, "bf16"), (60, 21504, "bf16"), (40, 9601, "bf16"), (16, 12001, "fp32"),
                                               (8, 30011, "bf16"), (8, 30011, "fp32"), (1, 131072, "bf16")])
def test_matvec_of_many_rows(tokens, rows, cols, block, two_d, dtype):
    """Blocks of rows that start at any row, also inside a tile of scales, when they are spread over the SMs' last turn;
    up to eight tokens, more rows to a CTA than one pass over its shared memory takes."""

    g = torch.Generator().manual_seed(rows + cols)
    x = torch.randn(tokens, cols, generator=g).to(DTYPES[dtype])
    codes, scales = packed_weight(rows, cols, block, two_d, seed=cols)
    bias = torch.randn(rows, generator=g) if rows % 2 else None
    check_matvec(x, codes, scales, rows, cols, block, two_d, bias=bias)


@pytest.mark.parametrize("cols", [4096, 4095])
@pytest.mark.parametrize("tokens", [1, 9])
def test_matvec_of_weights_beyond_32_bits(tokens, cols):
    """Codes of more than 2^31 bytes: the last rows, against those rows alone."""

    from ue5m3_fp4 import serving

    rows, last = 1_060_000, 300
    codes = torch.zeros(rows, (cols + 1) // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(rows, (cols + 15) // 16, dtype=torch.uint8, device="cuda")
    assert codes.numel() > 2 ** 31
    some_codes, some_scales = packed_weight(last, cols, 16, False, seed=1)
    codes[-last:], scales[-last:] = some_codes.cuda(), some_scales.cuda()
    x = torch.randn(tokens, cols, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    alone = check_matvec(x, some_codes, some_scales, last, cols, 16, False, out_dtype=torch.float32, amax=448.0 * 6)
    got = serving.packed_matvec(x.cuda(), codes, scales, rows=rows, cols=cols, block_size=16, two_dimensional=False,
                                tensor_amax=448.0 * 6, out_dtype=torch.float32)
    assert not bool(got[:, :-last].any())
    # the reduction axis is shared by other numbers of CTAs: the order of the fp32 sums may differ
    size = x.double().abs() @ unpack(some_codes, some_scales, last, cols, 16, False).T.abs()
    assert bool(((got[:, -last:] - alone).cpu().double().abs() <= size * (16 * 2.0 ** -21 + 60 * 2.0 ** -24)).all())


# ---- sampling ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("vocabulary", [700, 9000, 131072])
@pytest.mark.parametrize("top_p", [0.3, 0.9, 0.999, 1.0])
@pytest.mark.parametrize("top_k", [0, 40, 600])
def test_sample_settings_that_are_not_numbers(vocabulary, top_p, top_k):
    """A NaN among the settings of the rows: every row gets a token, that of the setting that cuts nothing."""

    from ue5m3_fp4 import serving

    g = torch.Generator().manual_seed(vocabulary)
    logits, uniforms = 0.5 * torch.randn(6, vocabulary, generator=g), torch.tensor([0.0, 0.2, 0.5, 0.8, 0.9999, math.nan])
    plain = dict(temperature=torch.full((6,), 0.9), top_k=torch.full((6,), top_k, dtype=torch.int32), top_p=torch.full((6,), top_p),
                 min_p=torch.zeros(6))
    clean = uniforms.nan_to_num()
    expect = check_sample(logits, clean, **plain)

    def run(**over):
        settings = {name: value.cuda() for name, value in {**plain, **over}.items()}
        return serving.sample_tokens(logits.cuda(), uniforms.cuda(), **settings)

    nan = torch.full((6,), math.nan)
    got = run(min_p=nan)
    assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1])
    got = run(top_p=nan)
    assert torch.equal(got[0], check_sample(logits, clean, **{**plain, "top_p": torch.ones(6)})[0])
    got = run(temperature=nan)
    assert torch.equal(got[0].cpu(), logits.argmax(1)) and not bool(got[1].any())


def test_sample_rows_beyond_32_bits():
    """Rows 2^30 elements apart: the third starts 2^31 elements behind the first."""

    from ue5m3_fp4 import serving

    vocabulary, apart = 5000, 2 ** 30
    memory = torch.empty(2 * apart + vocabulary, dtype=torch.bfloat16, device="cuda")
    logits = memory.as_strided((3, vocabulary), (apart, 1))
    logits.copy_(3 * torch.randn(3, vocabulary, generator=torch.Generator().manual_seed(1)))
    uniforms = torch.tensor([0.1, 0.6, 0.9], device="cuda")
    got, expect = (serving.sample_tokens(rows, uniforms, top_p=0.9) for rows in (logits, logits.contiguous()))
    assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1])


# ---- attention over a paged cache -----------------------------------------------------------------


@pytest.mark.parametrize("lengths,queries", [([700, 90], [1, 1]), ([700, 130], [60, 100])])
def test_attention_over_a_cache_beyond_32_bits(lengths, queries):
    """Pages of more than 2^31 elements, used at their end and in the middle: bit for bit as in a small cache with the
    same contents, the new keys and values included."""

    from ue5m3_fp4 import serving

    expect, q, (k, v, table, kv, starts) = run_attention(lengths, queries, page=64, kv_heads=4, group=4, dim=128, seed=2)
    count = k.shape[0]
    pages = 2 ** 31 // (64 * 4 * 128) + 1000
    large_k, large_v = (torch.empty(pages, 64, 4, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    place = torch.arange(count, device="cuda").to(torch.int32)
    place = torch.where(place % 2 == 0, pages - 1 - place, pages // 2 + place)
    large_k[place.long()], large_v[place.long()] = k, v
    moved = torch.where(table >= 0, place[table.clamp(min=0).long()], table)
    new_k, new_v = (torch.randn(sum(queries), 4, 128, device="cuda").to(torch.bfloat16) for _ in range(2))
    for more in ({}, dict(new_k=new_k, new_v=new_v)):
        small = serving.paged_attention(q, k, v, table, kv, starts, max_query_length=max(queries), **more)
        got = serving.paged_attention(q, large_k, large_v, moved, kv, starts, max_query_length=max(queries), **more)
        assert torch.equal(got, small)
    bits = lambda t: t.view(torch.int16)  # noqa: E731
    assert torch.equal(bits(large_k[place.long()]), bits(k)) and torch.equal(bits(large_v[place.long()]), bits(v))


# ---- packed linears ---------------------------------------------------------------------------------


def frozen_linear(weight: torch.Tensor):
    from ue5m3_fp4 import FP4InferenceScalingController
    from ue5m3_fp4.nn import UE5M3Linear

    model = torch.nn.Sequential(UE5M3Linear(weight.shape[1], weight.shape[0], bias=False, module_name="proj", device="cuda",
                                            dtype=torch.bfloat16))
    with torch.no_grad():
        model[0].weight.copy_(weight)
    controller = FP4InferenceScalingController(model.eval(), activation_mode="current_tensor", checkpoint_identity={"name": "none"})
    controller.reset_after_checkpoint_load()
    controller.calibrate_and_freeze_weights()
    return model


def test_packed_linears_take_the_weight_that_was_installed(tmp_path, monkeypatch):
    """A layer whose forward operand came from a file packs and exports that weight, not its parameter; a
    parameter written to afterwards counts again."""

    from ue5m3_fp4.nn import pack_frozen_linears

    monkeypatch.setenv("UE5M3_GEMM_PATH", "fp4")
    g = torch.Generator().manual_seed(1)
    own, other = ((0.02 * torch.randn(192, 256, generator=g)).clamp(-0.05, 0.05).to(torch.bfloat16).cuda() for _ in range(2))
    own[0, 0] = other[0, 0] = 0.06  # the same amax: the file fits the layer
    frozen_linear(other)[0].export_packed_weight(tmp_path / "other")
    model = frozen_linear(own)
    of_parameter = model[0].packed_weight()
    model[0].load_packed_weight(tmp_path / "other")
    expect = frozen_linear(other)[0].packed_weight()
    assert not torch.equal(of_parameter.codes, expect.codes)
    packed = model[0].packed_weight()
    assert torch.equal(packed.codes, expect.codes) and torch.equal(packed.scales, expect.scales)
    model[0].export_packed_weight(tmp_path / "again")
    assert (tmp_path / "again").read_bytes() == (tmp_path / "other").read_bytes()
    written = frozen_linear(own)
    written[0].load_packed_weight(tmp_path / "other")
    with torch.no_grad():
        written[0].weight.mul_(1.0)
    assert torch.equal(written[0].packed_weight().codes, of_parameter.codes)
    pack_frozen_linears(model)
    x = torch.randn(3, 256, device="cuda").to(torch.bfloat16)
    reference = x.double() @ expect.dequantize().double().T
    got = model(x).double()
    assert bool(((got - reference).abs() <= 2.0 ** -8 * reference.abs() + 1e-5).all())


# ---- graphs and streams ------------------------------------------------------------------------------


@pytest.mark.parametrize("cases", [[([5000], [1], 1, 8, 128), ([3001], [2], 2, 3, 64)],
                                   [([4000, 90], [1, 1], 2, 4, 64), ([3500], [40], 1, 8, 64)],
                                   [([2600, 700], [33, 5], 1, 2, 128), ([5000], [300], 1, 1, 128)]])
def test_split_attention_in_two_graphs_and_on_two_streams(cases):
    """Sequences split over CTAs leave partial rows in a workspace: two captured calls with data and lengths of their
    own, replayed side by side on two streams next to eager calls, share none."""

    from ue5m3_fp4 import serving
    from ue5m3_fp4.serving.operators import _workspace_bytes

    calls = []
    for i, (lengths, queries, kv_heads, group, dim) in enumerate(cases):
        expect, q, (k, v, table, kv, starts) = run_attention(lengths, queries, page=32, kv_heads=kv_heads, group=group, dim=dim, seed=i)
        longest = table.shape[1] * 32
        assert _workspace_bytes(q.get_device(), sum(queries), len(lengths), kv_heads * group, kv_heads, dim, max(queries), longest) > 0
        call = lambda q=q, k=k, v=v, table=table, kv=kv, starts=starts, n=max(queries): (  # noqa: E731
            serving.paged_attention(q, k, v, table, kv, starts, max_query_length=n))
        assert torch.equal(call(), expect)
        calls.append((call, expect))
    graphs = []
    for call, _ in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for _, out in graphs:
            out.zero_()
        torch.cuda.synchronize()
        eager = []
        for (graph, _), stream, (call, _) in zip(graphs, streams, reversed(calls)):
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
                    eager.append(call())
        torch.cuda.synchronize()
        assert all(torch.equal(out, expect) for (_, out), (_, expect) in zip(graphs, calls))
        assert all(torch.equal(out, calls[1][1]) for out in eager[:3]) and all(torch.equal(out, calls[0][1]) for out in eager[3:])


FIRST_CALL = """
import sys
sys.path.insert(0, "ue5m3-fp4_b200")
import torch
from ue5m3_fp4 import serving
from ue5m3_fp4.backends import b200

pages = torch.randn(4, 16, 2, 64, device="cuda").to(torch.bfloat16)
q = torch.randn(1, 4, 64, device="cuda").to(torch.bfloat16)
table, kv, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[2, 0, 3]], [40], [0, 1]))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = serving.paged_attention(q, pages, pages, table, kv, starts, max_query_length=1)
words = b200.gemm_status(q.device)
assert words.tolist() == [0, 0, 0, 0]
expect = serving.paged_attention(q, pages, pages, table, kv, starts, max_query_length=1)
assert bool(expect.isfinite().all())
graph.replay()
assert torch.equal(out, expect)
words[0] = 1  # a recorded failure stays until it is cleared
graph.replay()
assert bool(out.isnan().all()) and words.tolist() == [1, 0, 0, 0]
words.zero_()
graph.replay()
assert torch.equal(out, expect)
print("done")
"""


def test_first_call_under_capture_leaves_the_status_words_to_all():
    """A process whose first call of the library is captured: a failure recorded on the device is not cleared by the
    graph's replays, and outputs are NaN until it is."""

    root = Path(__file__).resolve().parent.parent
    done = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "done", done.stderr[-2000:]
