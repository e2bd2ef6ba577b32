"""The operators of the token-by-token path against plain implementations in 64 bits.

Tolerances count roundings: a rounding to a type is off by at most half a step, 2^-8 of the value
for bf16 and 2^-24 for fp32.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- packed matrix-vector products ----------------------------------------------------------------


def unpack(codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int, block: int, two_d: bool) -> torch.Tensor:
    """p * s in 64 bits from packed storage."""

    magnitude = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    codes, scales = codes.cpu().long(), scales.cpu().long()
    nibbles = torch.stack((codes % 16, codes // 16), -1).reshape(rows, -1)[:, :cols]
    values = magnitude[nibbles % 8] * (1 - 2 * (nibbles // 8))
    exponent, mantissa = scales // 8, (scales % 8).double()
    s = torch.where(exponent == 0, mantissa * 2.0 ** -17, (8 + mantissa) * 2.0 ** (exponent - 18).double())
    s = s.repeat_interleave(block, 1)[:, :cols]
    if two_d:
        s = s.repeat_interleave(block, 0)[:rows]
    return values * s


def packed_weight(rows: int, cols: int, block: int, two_d: bool, seed: int, low: int = 96, high: int = 160):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (rows, (cols + 1) // 2), generator=g, dtype=torch.uint8)
    scale_rows = (rows + block - 1) // block if two_d else rows
    scales = torch.randint(low, high, (scale_rows, (cols + block - 1) // block), generator=g, dtype=torch.uint8)
    return codes, scales


def check_matvec(x, codes, scales, rows, cols, block, two_d, *, bias=None, out_dtype=None, amax=0.37, target=448.0,
                 placed=None):
    from ue5m3_fp4 import serving
    from ue5m3_fp4.serving.operators import decode_factor

    got = serving.packed_matvec(x.cuda(), *(placed or (codes.cuda(), scales.cuda())), rows=rows, cols=cols, block_size=block,
                                two_dimensional=two_d, tensor_amax=amax, scale_target=target,
                                bias=None if bias is None else bias.cuda(), out_dtype=out_dtype)
    assert got.shape == (*x.shape[:-1], rows) and got.dtype is (out_dtype or x.dtype)
    weight = unpack(codes, scales, rows, cols, block, two_d) * decode_factor(amax, target)
    flat = x.reshape(-1, cols).double()
    expect, size = flat @ weight.T, flat.abs() @ weight.T.abs()
    if bias is not None:
        expect, size = expect + bias.double(), size + bias.double().abs()
    # 128 products per tensor-core sum in eight steps of at most 2^-21 of the sum of magnitudes each,
    # then one fp32 addition per further chunk and warp (16 warps share the axis up to eight tokens, at
    # least two above), factor and bias
    additions = math.ceil(cols / (2048 if flat.shape[0] <= 8 else 256)) + 20
    tolerance = size * (8 * 2.0 ** -21 + additions * 2.0 ** -24)
    tolerance = tolerance + expect.abs() * (2.0 ** -8 if got.dtype is torch.bfloat16 else 2.0 ** -24) + 1e-38
    error = (got.cpu().double().reshape(-1, rows) - expect).abs()
    assert bool((error <= tolerance).all()), float((error / tolerance).max())
    return got


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("block,two_d", [(16, True), (16, False), (32, True), (32, False)])
@pytest.mark.parametrize("tokens,rows,cols", [(1, 512, 4096), (1, 1, 32), (3, 17, 33), (8, 150, 2048), (2, 149, 96),
                                              (9, 31, 160), (5, 777, 1003), (17, 300, 4128), (64, 130, 640)])
def test_matvec_matches_the_definition(tokens, rows, cols, block, two_d, dtype):
    g = torch.Generator().manual_seed(tokens * 1000 + rows)
    x = torch.randn(tokens, cols, generator=g).to(DTYPES[dtype])
    codes, scales = packed_weight(rows, cols, block, two_d, seed=cols)
    bias = torch.randn(rows, generator=g).to(DTYPES[dtype]) if rows % 2 else None
    check_matvec(x, codes, scales, rows, cols, block, two_d, bias=bias)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("block,two_d", [(16, True), (32, False)])
@pytest.mark.parametrize("tokens,rows,cols", [(9, 128, 128), (12, 1, 33), (16, 129, 256), (33, 257, 1152), (32, 1000, 1003),
                                              (65, 64, 2560), (130, 40, 4224), (100, 300, 77), (40, 515, 20096)])
def test_matvec_of_many_tokens(tokens, rows, cols, block, two_d, dtype):
    """Token tiles, blocks of 128 rows, and reduction axes shared by one to eight CTAs."""

    g = torch.Generator().manual_seed(tokens + cols)
    wide = torch.randn(tokens, cols + 5, generator=g).to(DTYPES[dtype])
    codes, scales = packed_weight(rows, cols, block, two_d, seed=cols)
    bias = torch.randn(rows, generator=g) if rows % 2 else None
    for x in (wide[:, :cols].contiguous(), wide[:, 1:cols + 1]):  # rows on 16-byte boundaries, and not
        got = check_matvec(x, codes, scales, rows, cols, block, two_d, bias=bias)
        assert torch.equal(got, check_matvec(x, codes, scales, rows, cols, block, two_d, bias=bias))


@pytest.mark.parametrize("block,two_d", [(16, False), (16, True), (32, False), (32, True)])
@pytest.mark.parametrize("tokens", [1, 8, 20, 70])
def test_matvec_of_weights_that_start_anywhere(tokens, block, two_d):
    """The first and last bytes of codes and scales, at every place in the aligned pieces they are read by."""

    for shift in (0, 1, 5, 15):
        for rows, cols in ((1, 1), (2, 3), (17, 9), (40, 33), (33, 130), (5, 2049)):
            codes, scales = packed_weight(rows, cols, block, two_d, seed=shift + cols)
            placed = []
            for part in (codes, scales):
                buffer = torch.full((part.numel() + 48,), 0xFF, dtype=torch.uint8, device="cuda")
                view = buffer[shift:shift + part.numel()].view(part.shape)
                view.copy_(part)
                placed.append(view)
            x = torch.randn(tokens, cols, generator=torch.Generator().manual_seed(cols)).to(torch.bfloat16)
            check_matvec(x, codes, scales, rows, cols, block, two_d, placed=placed)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_matvec_of_many_tokens_keeps_rows_apart(dtype):
    """A row's infinities, NaN and magnitudes are its own; the others are as they are without them."""

    from ue5m3_fp4 import serving

    rows, cols = 150, 700
    codes, scales = packed_weight(rows, cols, 16, False, seed=6)
    x = torch.randn(45, cols, generator=torch.Generator().manual_seed(8)).to(DTYPES[dtype])
    kw = dict(rows=rows, cols=cols, block_size=16, two_dimensional=False, tensor_amax=1.0)
    plain = serving.packed_matvec(x.cuda(), codes.cuda(), scales.cuda(), **kw)
    mixed = x.clone()
    mixed[3, 17], mixed[9], mixed[20, 699], mixed[44] = math.inf, x[9] * 2.0 ** 90, math.nan, x[44] * 2.0 ** -90
    got = serving.packed_matvec(mixed.cuda(), codes.cuda(), scales.cuda(), **kw)
    same = [t for t in range(45) if t not in (3, 9, 20, 44)]
    assert torch.equal(got[same], plain[same])
    assert not bool(got[3].isfinite().any()) and bool(got[20].isnan().all())
    assert torch.equal(got[9], plain[9] * 2.0 ** 90) and torch.equal(got[44], plain[44] * 2.0 ** -90)


def test_matvec_of_many_tokens_in_two_graphs_and_on_two_streams():
    from ue5m3_fp4 import serving

    rows, cols = 300, 2048
    codes, scales = (t.cuda() for t in packed_weight(rows, cols, 32, False, seed=7))
    kw = dict(rows=rows, cols=cols, block_size=32, two_dimensional=False, tensor_amax=1.0)
    inputs = [torch.randn(tokens, cols, device="cuda", dtype=torch.bfloat16) for tokens in (20, 60)]
    expect = [serving.packed_matvec(x, codes, scales, **kw) for x in inputs]
    graphs, outs = [], []
    for x in inputs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(serving.packed_matvec(x, codes, scales, **kw))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        eager = []
        for graph, stream, x in zip(graphs, streams, reversed(inputs)):
            with torch.cuda.stream(stream):
                graph.replay()
                eager.append(serving.packed_matvec(x, codes, scales, **kw))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, expect))
        assert all(torch.equal(a, b) for a, b in zip(eager, reversed(expect)))


def test_matvec_takes_every_scale_byte_and_code():
    """Scale bytes 0..255 (subnormal ones, and those above the quantizer's largest) times all 16 codes."""

    rows, cols = 256, 64
    codes = torch.arange(32, dtype=torch.uint8).repeat(rows, 1) * 8 + torch.arange(32, dtype=torch.uint8) % 8
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 4)
    x = torch.randn(2, cols, generator=torch.Generator().manual_seed(3))
    check_matvec(x, codes, scales, rows, cols, 16, False)
    check_matvec(x.to(torch.bfloat16), codes, scales, rows, cols, 16, False, out_dtype=torch.float32)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_matvec_activation_range(dtype):
    """Rows of tiny (subnormal), huge and widely spread activations."""

    rows, cols = 40, 384
    codes, scales = packed_weight(rows, cols, 16, False, seed=1)
    g = torch.Generator().manual_seed(2)
    base = torch.randn(4, cols, generator=g, dtype=torch.float64)
    base[0] *= 2.0 ** -128
    base[1] *= 2.0 ** 110
    base[2] *= torch.exp2(torch.randint(-14, 15, (cols,), generator=g).double())
    check_matvec(base.to(DTYPES[dtype]), codes, scales, rows, cols, 16, False, out_dtype=torch.float32, amax=448.0 * 6)


def test_matvec_infinities_and_nans_stay_in_their_row():
    from ue5m3_fp4 import serving

    rows, cols = 48, 300
    codes, scales = packed_weight(rows, cols, 16, False, seed=5)
    for dtype in DTYPES.values():
        x = torch.randn(4, cols, generator=torch.Generator().manual_seed(1)).to(dtype)
        x[1, 7] = math.inf
        x[3, 299] = math.nan
        got = serving.packed_matvec(x.cuda(), codes.cuda(), scales.cuda(), rows=rows, cols=cols, block_size=16,
                                    two_dimensional=False, tensor_amax=1.0).cpu()
        weight = unpack(codes, scales, rows, cols, 16, False)
        expect = (x.double().nan_to_num(nan=math.nan, posinf=math.inf)[:, None, :] * weight[None]).sum(-1)
        assert torch.equal(got[1].isnan(), expect[1].isnan())
        assert torch.equal(got[1][~got[1].isnan()].sign().double(), expect[1][~expect[1].isnan()].sign())
        assert bool(got[1][~got[1].isnan()].isinf().all()) and bool(got[3].isnan().all())
        assert bool(got[0].isfinite().all()) and bool(got[2].isfinite().all())


def test_matvec_strides_offsets_and_repeatability():
    from ue5m3_fp4 import serving

    rows, cols = 100, 480
    codes, scales = packed_weight(rows, cols, 32, True, seed=9)
    wide = torch.randn(6, cols + 7, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    view = wide[::2, 3:3 + cols]
    kw = dict(rows=rows, cols=cols, block_size=32, two_dimensional=True, tensor_amax=1.0)
    got = serving.packed_matvec(view, codes.cuda(), scales.cuda(), **kw)
    assert torch.equal(got, serving.packed_matvec(view.contiguous(), codes.cuda(), scales.cuda(), **kw))
    buffer = torch.zeros(codes.numel() + 5, dtype=torch.uint8, device="cuda")
    shifted = buffer[5:].view(codes.shape)  # code rows off their 16-byte boundaries
    shifted.copy_(codes)
    assert torch.equal(got, serving.packed_matvec(view, shifted, scales.cuda(), **kw))
    assert serving.packed_matvec(view[:0], codes.cuda(), scales.cuda(), **kw).shape == (0, rows)
    cube = view.contiguous().view(3, 1, cols)
    assert torch.equal(serving.packed_matvec(cube, codes.cuda(), scales.cuda(), **kw).view(3, rows), got)


def test_matvec_agrees_with_dequantize_on_a_quantized_weight():
    from ue5m3_fp4.packed import PackedFP4Tensor

    weight = (0.02 * torch.randn(192, 320, generator=torch.Generator().manual_seed(8))).to(torch.bfloat16).cuda()
    for two_d in (False, True):
        packed = PackedFP4Tensor.quantize(weight, block_size=16, two_dimensional=two_d, tensor_amax=weight.abs().max().float())
        x = torch.randn(4, 320, device="cuda")
        expect = x.double() @ packed.dequantize().double().T
        got = packed.matvec(x).double()
        assert float((got - expect).norm() / expect.norm()) < 1e-6


# ---- attention over a paged cache -----------------------------------------------------------------


def build_cache(lengths, page, kv_heads, dim, seed, spare=3, layout="plain"):
    """Pages in random order, unset table entries -1, and NaN wherever no key belongs."""

    g = torch.Generator().manual_seed(seed)
    counts = [(length + page - 1) // page for length in lengths]
    total, width = sum(counts) + spare, max(max(counts), 1)
    shape = (total, page, kv_heads, dim)
    if layout == "heads_first":
        k = torch.randn(total, kv_heads, page, dim, generator=g).to(torch.bfloat16).cuda().transpose(1, 2)
        v = torch.randn(total, kv_heads, page, dim, generator=g).to(torch.bfloat16).cuda().transpose(1, 2)
    elif layout == "interleaved":
        both = torch.randn(total, 2, page, kv_heads, dim, generator=g).to(torch.bfloat16).cuda()
        k, v = both[:, 0], both[:, 1]
    else:
        k = torch.randn(shape, generator=g).to(torch.bfloat16).cuda()
        v = torch.randn(shape, generator=g).to(torch.bfloat16).cuda()
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    used = torch.zeros(total, page, dtype=torch.bool)
    at = 0
    for b, (length, count) in enumerate(zip(lengths, counts)):
        table[b, :count] = order[at:at + count]
        for j in range(count):
            used[order[at + j], :min(page, length - j * page)] = True
        at += count
    k[~used.cuda()] = math.nan
    v[~used.cuda()] = math.nan
    return k, v, table.cuda()


def reference_attention(q, k_pages, v_pages, table, lengths, queries, scale):
    """Output and, per output, the largest error that rounding the probabilities to bf16 may cause."""

    q, k_pages, v_pages, table = q.cpu().double(), k_pages.cpu().double(), v_pages.cpu().double(), table.cpu().long()
    tokens, heads, dim = q.shape
    kv_heads, page = k_pages.shape[2], k_pages.shape[1]
    out, spread = torch.zeros(tokens, heads, dim, dtype=torch.float64), torch.zeros(tokens, heads, dim, dtype=torch.float64)
    row = 0
    for b, (length, n) in enumerate(zip(lengths, queries)):
        for i in range(n):
            seen = length - n + i + 1
            if seen > 0:
                pages = table[b, :(seen + page - 1) // page]
                k = k_pages[pages].reshape(-1, kv_heads, dim)[:seen].repeat_interleave(heads // kv_heads, 1)
                v = v_pages[pages].reshape(-1, kv_heads, dim)[:seen].repeat_interleave(heads // kv_heads, 1)
                p = torch.softmax(torch.einsum("hd,khd->hk", q[row], k) * scale, -1)
                out[row] = torch.einsum("hk,khd->hd", p, v)
                spread[row] = torch.einsum("hk,khd->hd", p, v.abs())
            row += 1
    return out, spread


def run_attention(lengths, queries, *, page, kv_heads, group, dim, seed=0, append=True, layout="plain", tail=0,
                  out=None, **kw):
    from ue5m3_fp4 import serving

    k_pages, v_pages, table = build_cache(lengths, page, kv_heads, dim, seed, layout=layout)
    g = torch.Generator().manual_seed(seed + 1)
    tokens = sum(queries) + tail
    q = (1.5 * torch.randn(tokens, kv_heads * group, dim, generator=g)).to(torch.bfloat16).cuda()
    new_k = torch.randn(tokens, kv_heads, dim, generator=g).to(torch.bfloat16).cuda()
    new_v = torch.randn(tokens, kv_heads, dim, generator=g).to(torch.bfloat16).cuda()
    starts = torch.tensor([0, *np.cumsum(queries)], dtype=torch.int32, device="cuda")
    kv = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    expect_k, expect_v = k_pages.clone(), v_pages.clone()
    if append:
        row = 0
        for b, (length, n) in enumerate(zip(lengths, queries)):
            for i in range(n):
                position = length - n + i
                if position >= 0:
                    at = int(table[b, position // page])
                    expect_k[at, position % page], expect_v[at, position % page] = new_k[row], new_v[row]
                row += 1
    got = serving.paged_attention(q, k_pages, v_pages, table, kv, starts, out=out,
                                  new_k=new_k if append else None, new_v=new_v if append else None,
                                  **{"max_query_length": max(max(queries), 1), **kw})
    bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(bits(k_pages), bits(expect_k)) and torch.equal(bits(v_pages), bits(expect_v))
    expect, spread = reference_attention(q, k_pages, v_pages, table, lengths, queries, kw.get("scale") or dim ** -0.5)
    # the result and every probability are rounded to bf16 once, scores and sums are fp32
    tolerance = 2.0 ** -8 * expect.abs() + (2.0 ** -8 + 2.0 ** -12) * spread + 1e-30
    used = sum(queries)
    error = (got[:used].cpu().double() - expect[:used]).abs()
    assert bool((error <= tolerance[:used]).all()), float((error / tolerance[:used]).max())
    return got, q, (k_pages, v_pages, table, kv, starts)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("lengths,queries", [([1], [1]), ([63], [1]), ([64], [1]), ([65, 1, 300], [1, 1, 1]),
                                             ([5, 200, 17], [5, 1, 9]), ([130], [130]), ([333, 2], [70, 2])])
def test_attention_matches_the_definition(lengths, queries, page, dim):
    run_attention(lengths, queries, page=page, kv_heads=2, group=4, dim=dim, seed=len(lengths) + page)


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (1, 16), (3, 1), (2, 5), (4, 8), (1, 7), (1, 33)])
def test_attention_head_layouts(kv_heads, group):
    run_attention([70, 7], [1, 3], page=16, kv_heads=kv_heads, group=group, dim=64, seed=group)
    run_attention([150, 90], [40, 33], page=32, kv_heads=kv_heads, group=group, dim=128, seed=group + 1)


@pytest.mark.parametrize("layout", ["heads_first", "interleaved"])
def test_attention_strided_pages(layout):
    run_attention([100, 31], [1, 1], page=32, kv_heads=2, group=4, dim=128, layout=layout, seed=3)
    run_attention([100, 61], [50, 33], page=16, kv_heads=2, group=4, dim=64, layout=layout, seed=4)


def test_attention_split_sequences():
    """Long sequences next to short ones: runs of keys on several CTAs, joined by the second launch."""

    run_attention([5000, 1, 700], [1, 1, 1], page=64, kv_heads=1, group=8, dim=128, seed=6)
    run_attention([3001], [2], page=16, kv_heads=2, group=3, dim=64, seed=7)
    run_attention([4097, 64], [4, 1], page=128, kv_heads=1, group=8, dim=128, seed=8)


@pytest.mark.parametrize("append", [True, False])
def test_attention_empty_rows_and_sequences(append):
    """Sequences without keys, without new tokens, and with fewer keys than new tokens: rows that see
    nothing are zero."""

    got, *_ = run_attention([0, 20, 3, 9], [2, 0, 7, 1], page=16, kv_heads=2, group=2, dim=64, append=append)
    assert bool((got[:2] == 0).all()) and bool((got[2:6] == 0).all()) and bool((got[6] != 0).any())
    got, *_ = run_attention([0, 40], [50, 90], page=16, kv_heads=2, group=4, dim=128, append=append)
    assert bool((got[:100] == 0).all()) and bool((got[100] != 0).any())


@pytest.mark.parametrize("queries", [[1, 2], [40, 70]])
def test_attention_padding_rows(queries):
    lengths = [30 + q for q in queries]
    got, q, _ = run_attention(lengths, queries, page=16, kv_heads=2, group=4, dim=64, tail=5)
    assert bool((got[-5:] == 0).all())
    out = torch.full_like(q, 7.0)
    got, *_ = run_attention(lengths, queries, page=16, kv_heads=2, group=4, dim=64, tail=5, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((out[-5:] == 7.0).all())


@pytest.mark.parametrize("lengths,queries", [([700, 300], [1, 1]), ([700, 300], [90, 200]), ([2500], [3])])
def test_attention_bounds_are_hints(lengths, queries):
    """Actual lengths above the bounds of the call come out the same."""

    run_attention(lengths, queries, page=16, kv_heads=2, group=4, dim=128, max_query_length=1, max_kv_length=16)
    run_attention(lengths, queries, page=16, kv_heads=2, group=4, dim=128, max_query_length=512, max_kv_length=1 << 20)


@pytest.mark.parametrize("lengths,queries", [([200, 200], [1, 1]), ([200, 200], [60, 60])])
def test_attention_pages_outside_the_cache(lengths, queries):
    """A table entry that names no page: the rows that need it are NaN, the others and the cache are
    as without it."""

    from ue5m3_fp4 import serving

    _, q, (k, v, table, kv, starts) = run_attention(lengths, queries, page=32, kv_heads=2, group=2, dim=64)
    good = serving.paged_attention(q, k, v, table, kv, starts, max_query_length=queries[0])
    for wrong in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        broken = table.clone()
        broken[1, 2] = wrong
        before = k.clone()
        got = serving.paged_attention(q, k, v, broken, kv, starts, max_query_length=queries[0])
        assert torch.equal(got[:queries[0]], good[:queries[0]]) and bool(got[queries[0]:].isnan().all())
        assert torch.equal(k.nan_to_num(), before.nan_to_num())
    long = kv.clone()
    long[0] = 10 ** 6
    got = serving.paged_attention(q, k, v, table, long, starts, max_query_length=queries[0])
    assert bool(got[:queries[0]].isnan().all()) and torch.equal(got[queries[0]:], good[queries[0]:])


@pytest.mark.parametrize("queries,kv_heads,group,page", [(3, 2, 4, 16), (8, 1, 4, 32), (60, 2, 4, 16), (300, 1, 1, 64), (150, 2, 5, 32)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_values_that_are_not_numbers_stay_with_the_rows_that_see_them(queries, kv_heads, group, page, dim):
    """NaN and infinities in the keys and values of late tokens of a chunk, and of one that all rows see."""

    from ue5m3_fp4 import serving

    old = 70
    length = old + queries
    k_pages, v_pages, table = build_cache([length], page, kv_heads, dim, 1)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(queries, kv_heads * group, dim, generator=g).to(torch.bfloat16).cuda()
    new_k = torch.randn(queries, kv_heads, dim, generator=g).to(torch.bfloat16).cuda()
    new_v = torch.randn(queries, kv_heads, dim, generator=g).to(torch.bfloat16).cuda()
    late = [queries - 1, queries // 2]
    new_v[late[0], 0, 3] = math.nan
    new_v[late[1], 0, 5] = math.inf
    new_v[late[1], kv_heads - 1, dim - 1] = -math.inf
    starts, kv = torch.tensor([0, queries]).int().cuda(), torch.tensor([length]).int().cuda()

    def run():
        return serving.paged_attention(q, k_pages, v_pages, table, kv, starts, max_query_length=queries, new_k=new_k, new_v=new_v)

    got = run().cpu().double()
    expect, _ = reference_attention(q, k_pages, v_pages, table, [length], [queries], dim ** -0.5)
    assert torch.equal(got.isnan(), expect.isnan())
    assert torch.equal(got.isinf(), expect.isinf()) and torch.equal(got[got.isinf()].sign(), expect[expect.isinf()].sign())
    finite = expect.isfinite()
    assert float((got[finite] - expect[finite]).abs().max()) < 0.05
    # a key that is not a number: the rows that see it, all channels of its heads
    new_k[late[1], 0, 0] = math.nan
    got = run().cpu()
    assert bool(got[late[1]:, :group].isnan().all()) and bool(got[:late[1], :, 0].isfinite().all())
    # a value that every row sees
    new_k[late[1], 0, 0] = 0.0
    at = int(table[0, 0])
    v_pages[at, 1, 0, 2] = math.nan
    got = run().cpu()
    assert bool(got[:, :group, 2].isnan().all()) and bool(got[:late[1], :group, 1].isfinite().all())


def test_attention_large_scores_and_scale():
    """Scores of a few hundred (one key takes all), and a scale of its own."""

    run_attention([500], [1], page=16, kv_heads=1, group=4, dim=128, scale=2.0)
    run_attention([400], [60], page=16, kv_heads=1, group=4, dim=128, scale=2.0)
    run_attention([400], [60], page=16, kv_heads=1, group=4, dim=64, scale=1e-4)


# ---- sampling ---------------------------------------------------------------------------------------


def reference_sample(logits, u, temperature, top_k, top_p, min_p):
    """The definition with exact sums: weights in 64 bits, rounded to multiples of 2^-44 (sums of
    doubles would miss borders that u or top_p meet exactly)."""

    from fractions import Fraction

    l = logits.double().cpu().numpy()
    if np.isnan(l).any() or l.max() == -math.inf:
        return -1, math.nan
    if not temperature > 0:
        return int(l.argmax()), 0.0
    with np.errstate(invalid="ignore"):
        z = np.where(l == l.max(), 0.0, (l - l.max()) / temperature)
    w = np.rint(np.where(l == -math.inf, 0.0, np.exp(z)) * 2.0 ** 44).astype(np.int64)
    order = np.argsort(-l, kind="stable")
    kept = np.zeros(len(l), dtype=bool)
    kept[order[:top_k if top_k > 0 else len(l)]] = True
    if top_p < 1:
        ranked = np.where(kept, w, 0)[order]
        before = np.cumsum(ranked) - ranked
        drop = before >= math.ceil(Fraction(top_p) * int(ranked.sum()))
        drop[0] = False
        kept[order[drop]] = False
    kept &= (w >= min_p * 2.0 ** 44) | (l == l.max())
    mass = np.where(kept, w, 0)
    running = np.cumsum(mass)
    if u >= 1:
        token = int(np.nonzero(mass)[0][-1])
    else:
        token = int(np.argmax(running > math.floor(Fraction(max(u, 0.0)) * int(running[-1]))))
    return token, float(z[token] - math.log(int(running[-1]) * 2.0 ** -44))


def check_sample(logits, uniforms, **settings):
    from ue5m3_fp4 import serving

    rows = logits.shape[0]
    tokens, logprobs = serving.sample_tokens(logits.cuda() if not logits.is_cuda else logits, uniforms.cuda(),
                                             **{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in settings.items()})
    assert tokens.dtype is torch.int64 and logprobs.dtype is torch.float32
    for r in range(rows):
        own = {k: float(v[r]) if isinstance(v, torch.Tensor) else v for k, v in settings.items()}
        own = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0} | own
        own = {k: float(np.float32(v)) for k, v in own.items()}
        token, logprob = reference_sample(logits[r], float(uniforms[r]), own["temperature"], int(own["top_k"]), own["top_p"],
                                          own["min_p"])
        assert int(tokens[r]) == token, (r, int(tokens[r]), token)
        got = float(logprobs[r])
        # one rounding to fp32; the weights' sum is exact to 2^-45 of its largest term per term
        assert (math.isnan(got) and math.isnan(logprob)) or abs(got - logprob) <= 2.0 ** -24 * abs(logprob) + 1e-8, (r, got, logprob)
    return tokens, logprobs


SETTINGS = [dict(), dict(top_k=1), dict(top_k=3), dict(top_k=50, top_p=0.9), dict(top_p=0.5), dict(top_p=0.95, min_p=0.02),
            dict(min_p=0.3), dict(temperature=0.0), dict(temperature=0.3, top_k=2000, top_p=0.999), dict(temperature=5.0, top_p=0.7)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,vocabulary", [(1, 1), (3, 2), (5, 37), (2, 4097), (4, 32003), (3, 131072)])
def test_sample_matches_the_definition(rows, vocabulary, dtype):
    g = torch.Generator().manual_seed(vocabulary)
    for i, settings in enumerate(SETTINGS):
        logits = (3.0 * torch.randn(rows, vocabulary, generator=g)).to(DTYPES[dtype])
        uniforms = torch.rand(rows, generator=g)
        uniforms[0] = (0.0, 1.0 - 2.0 ** -24, float(uniforms[0]))[i % 3]
        check_sample(logits, uniforms, **settings)


@pytest.mark.parametrize("vocabulary", [8, 5000, 131072])
def test_sample_ties_go_to_the_lowest_index(vocabulary):
    """All logits equal, two levels, and steps of equal logits: thresholds fall inside ties."""

    uniforms = torch.tensor([0.0, 0.25, 0.5, 0.9999])
    index = torch.arange(vocabulary)
    for logits in (torch.zeros(vocabulary), (index % 2).float(), (index % 7).float(), -(index // 3 % 5).float()):
        rows = logits.repeat(4, 1)
        for settings in (dict(), dict(top_k=3), dict(top_k=vocabulary // 2 + 1), dict(top_p=0.5), dict(top_k=5, top_p=0.6)):
            check_sample(rows, uniforms, **settings)


def test_sample_masked_infinite_and_broken_rows():
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(8, 5001, generator=g)
    logits[0, :] = -math.inf
    logits[1, 17] = math.nan
    logits[2, 1:] = -math.inf
    logits[3, torch.rand(5001, generator=g) < 0.9] = -math.inf
    logits[4, 4000] = math.inf
    logits[5, 10] = math.inf
    logits[5, 4999] = math.inf
    logits[6] = -1e30
    logits[7, 5000] = 3e38
    uniforms = torch.rand(8, generator=g)
    for settings in (dict(), dict(top_k=4), dict(top_p=0.8), dict(top_k=4000, top_p=0.3, min_p=0.1), dict(temperature=0.0),
                     dict(temperature=1e-30, top_p=0.9), dict(temperature=1e30, top_p=0.9)):
        check_sample(logits, uniforms, **settings)


def test_sample_settings_per_row_and_uniform_range():
    g = torch.Generator().manual_seed(2)
    logits = 2 * torch.randn(7, 9000, generator=g)
    uniforms = torch.tensor([0.0, 0.5, 1.0, 2.0, -1.0, 0.999, 1e-30])
    check_sample(logits, uniforms, temperature=torch.tensor([0.0, 1.0, 0.5, 2.0, 1.0, 0.7, 3.0]),
                 top_k=torch.tensor([0, 5, 0, 100, 9000, 1, -3], dtype=torch.int32),
                 top_p=torch.tensor([1.0, 0.9, 0.4, 1.0, 0.0, 0.3, 0.99]), min_p=torch.tensor([0.0, 0.1, 0.0, 0.5, 0.0, 0.0, 0.01]))


@pytest.mark.parametrize("vocabulary", [3000, 131072])
def test_sample_tails_without_weight(vocabulary):
    """A few tokens carry all the weight, thousands none or next to none: the nucleus ends among them."""

    g = torch.Generator().manual_seed(4)
    logits = torch.full((6, vocabulary), -100.0)
    logits[:, ::vocabulary // 900] = 0.0
    logits[1] -= torch.arange(vocabulary) / vocabulary          # all of weight zero, all different
    logits[2, ::7] = -20.0                                      # thousands of equal tiny weights
    logits[3] = -31.0 * torch.rand(vocabulary, generator=g)     # weights down to the last unit
    logits[4] = -16.0 - 16.0 * torch.rand(vocabulary, generator=g)
    logits[4, 5] = 0.0
    logits[5] = -29.0
    logits[5, 11] = 0.0
    uniforms = torch.tensor([0.3, 0.9, 0.99999, 0.5, 1.0 - 2.0 ** -24, 1.0 - 2.0 ** -24])
    for settings in (dict(top_p=0.9999999), dict(top_p=0.999), dict(top_p=1.0 - 2.0 ** -24, min_p=1e-9), dict(top_k=1500, top_p=0.99999),
                     dict(top_k=1000, top_p=0.9999), dict(temperature=0.5, top_p=0.9999999)):
        check_sample(logits, uniforms, **settings)


@pytest.mark.parametrize("vocabulary", [3000, 40000])
@pytest.mark.parametrize("top_k,top_p", [(0, 0.5), (0, 0.999), (700, 0.9), (2500, 0.9), (2500, 1.0)])
def test_sample_subnormal_logits_and_temperature(vocabulary, top_k, top_p):
    # all logits within one of the first bins, most of them without weight
    generator = torch.Generator().manual_seed(vocabulary + top_k)
    steps = torch.randint(0, 400, (2, vocabulary), generator=generator)
    logits = (steps.double() * -2.0 ** -149).float()
    assert logits.unique().numel() == 400
    check_sample(logits, torch.tensor([0.3, 0.97]), temperature=2.0 ** -148, top_k=top_k, top_p=top_p)


def test_sample_strided_rows():
    from ue5m3_fp4 import serving

    wide = torch.randn(6, 1203, device="cuda")
    view = wide[::2, 3:1003]
    uniforms = torch.rand(3, device="cuda")
    got = serving.sample_tokens(view, uniforms, top_p=0.9)
    expect = serving.sample_tokens(view.contiguous(), uniforms, top_p=0.9)
    assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1])
    tokens, logprobs = serving.sample_tokens(view[:0], uniforms[:0])
    assert tokens.shape == (0,) and logprobs.shape == (0,)


# ---- arguments that are refused -----------------------------------------------------------------------


def test_matvec_refusals():
    from ue5m3_fp4 import serving

    codes, scales = (t.cuda() for t in packed_weight(8, 64, 16, False, 0))
    good = dict(rows=8, cols=64, block_size=16, two_dimensional=False, tensor_amax=1.0)
    x = torch.randn(2, 64, device="cuda")
    serving.packed_matvec(x, codes, scales, **good)
    for bad in (dict(block_size=8), dict(rows=9), dict(cols=62), dict(two_dimensional=True), dict(tensor_amax=math.nan),
                dict(tensor_amax=-1.0), dict(scale_target=0.0), dict(bias=torch.zeros(7, device="cuda")), dict(bias=torch.zeros(8))):
        with pytest.raises(ValueError):
            serving.packed_matvec(x, codes, scales, **{**good, **bad})
    with pytest.raises(TypeError):
        serving.packed_matvec(x.half(), codes, scales, **good)
    with pytest.raises(TypeError):
        serving.packed_matvec(x, codes, scales, out_dtype=torch.float16, **good)
    with pytest.raises(ValueError, match="contiguous"):
        serving.packed_matvec(torch.randn(64, 2, device="cuda").T, codes, scales, **good)
    with pytest.raises(ValueError, match="overlap"):
        serving.packed_matvec(x[:1].expand(2, 64), codes, scales, **good)
    with pytest.raises(ValueError):
        serving.packed_matvec(x, codes.cpu(), scales, **good)
    with pytest.raises(RuntimeError, match="no gradients"):
        serving.packed_matvec(x.clone().requires_grad_(True), codes, scales, **good)


def test_attention_refusals():
    from ue5m3_fp4 import serving

    k, v, table = build_cache([20], 16, 2, 64, 0)
    q = torch.randn(1, 4, 64, device="cuda").to(torch.bfloat16)
    kv, starts = torch.tensor([20]).int().cuda(), torch.tensor([0, 1]).int().cuda()

    def call(q=q, k=k, v=v, table=table, kv=kv, starts=starts, max_query_length=1, **kw):
        return serving.paged_attention(q, k, v, table, kv, starts, max_query_length=max_query_length, **kw)

    call()
    new = torch.randn(1, 2, 64, device="cuda").to(torch.bfloat16)
    for bad in (dict(q=q.float()), dict(k=k.float()), dict(q=q[:, :3]), dict(q=q[0]), dict(table=table.long()), dict(kv=kv.long()),
                dict(starts=starts[:1]), dict(max_query_length=0), dict(max_kv_length=0), dict(scale=0.0), dict(scale=math.nan),
                dict(new_k=new), dict(new_k=new, new_v=new[:, :1]), dict(new_k=new.float(), new_v=new), dict(out=q[:, :2]),
                dict(out=q.float()), dict(k=k[:, :12], v=v[:, :12]), dict(v=v[:-1]), dict(q=q.cpu().cuda()[..., :32]),
                dict(table=table.cpu()), dict(q=torch.zeros(1, 4, 66, device="cuda").to(torch.bfloat16)[..., :64])):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(RuntimeError, match="no gradients"):
        call(q=q.clone().requires_grad_(True))
    assert call(q=q[:0], starts=torch.zeros(2).int().cuda()).shape == (0, 4, 64)


def test_sample_refusals():
    from ue5m3_fp4 import serving

    logits, u = torch.randn(2, 50, device="cuda"), torch.rand(2, device="cuda")
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5),
                dict(min_p=-0.1), dict(min_p=2.0), dict(top_k=torch.ones(2, device="cuda")), dict(top_p=torch.ones(3, device="cuda")),
                dict(min_p=torch.ones(2))):
        with pytest.raises(ValueError):
            serving.sample_tokens(logits, u, **bad)
    for args in ((logits[0], u), (logits, u[:1]), (logits, u.double()), (logits.T, torch.rand(50, device="cuda")),
                 (logits[:1].expand(2, 50), u), (torch.empty(2, 0, device="cuda"), u)):
        with pytest.raises(ValueError):
            serving.sample_tokens(*args)
    with pytest.raises(TypeError):
        serving.sample_tokens(logits.half(), u)


# ---- the operators together ------------------------------------------------------------------------------


def small_stack(seed=0, **over):
    from ue5m3_fp4.integrations.torchtitan.shaped_stack import NemotronHShapedStack, ShapedConfig

    torch.manual_seed(seed)
    config = ShapedConfig(**{**dict(hidden_size=256, intermediate_size=512, mamba_inner=256, mamba_extra=64, attention_heads=8,
                                    kv_heads=2, head_dim=64, vocab_size=1000, num_hidden_layers=6,
                                    hybrid_override_pattern="M-*-M*"), **over})
    model = NemotronHShapedStack(config, device="cuda").eval()
    with torch.no_grad():
        for p in model.parameters():
            if p.ndim == 2:
                p.mul_(3.0)
    return model


def test_stack_served_in_steps_equals_its_forward_pass():
    """Prompts of different lengths in chunks and single tokens against whole forward passes: the same
    sums in other orders, rounded to bf16 after every layer."""

    model = small_stack()
    g = torch.Generator().manual_seed(1)
    ids = [torch.randint(0, 1000, (n,), generator=g).cuda() for n in (57, 20, 91)]
    cache = model.make_cache(sequences=3, max_length=128, page_size=16)
    at = [0, 0, 0]
    seen = [None] * 3
    for counts in ([40, 1, 0], [1, 1, 33], [1, 16, 50], [15, 2, 8]):
        cache.begin_step(counts)
        logits = model.serve(torch.cat([ids[b][at[b]:at[b] + n] for b, n in enumerate(counts)]), cache)
        for b, n in enumerate(counts):
            at[b] += n
            if n:
                seen[b] = logits[b]
    for b in range(3):
        assert at[b] == ids[b].numel()
        with torch.no_grad():
            expect = model(ids[b][None])[0, -1].double()
        # six layers, each with a handful of bf16 roundings of 2^-8 that add up like independent errors
        assert float((seen[b].double() - expect).norm() / expect.norm()) < 6 * 4 ** 0.5 * 2.0 ** -8


def test_frozen_stack_generates_with_packed_linears():
    """Post-load lifecycle -> packed linears -> token loop: the linears' outputs are those of the frozen
    weights, and the loop's tokens those that its own logits and numbers imply."""

    from ue5m3_fp4 import FP4InferenceScalingController
    from ue5m3_fp4 import serving
    from ue5m3_fp4.nn import PackedFP4Linear, UE5M3Linear, convert_linear_modules, exclude_lm_head, pack_frozen_linears

    model = small_stack(seed=3)
    convert_linear_modules(model, selector=exclude_lm_head)
    model.eval()
    controller = FP4InferenceScalingController(model, activation_mode="current_tensor", checkpoint_identity={"name": "none"})
    controller.reset_after_checkpoint_load()
    controller.calibrate_and_freeze_weights()
    layer = model.layers[1].mixer.up_proj
    x = torch.randn(3, 256, device="cuda").to(torch.bfloat16)
    packed = layer.packed_weight()
    expect = x.double() @ packed.dequantize().double().T
    records = pack_frozen_linears(model)
    assert len(records) == 2 * 2 + 2 * 2 + 2 * 4 and not any(isinstance(m, UE5M3Linear) for m in model.modules())
    got = model.layers[1].mixer.up_proj(x)
    assert isinstance(model.layers[1].mixer.up_proj, PackedFP4Linear)
    assert bool(((got.double() - expect).abs() <= 2.0 ** -8 * expect.abs() + 1e-4).all())
    prompts = [torch.arange(5, device="cuda"), torch.arange(30, 75, device="cuda")]
    uniforms = torch.rand(6, 2, device="cuda")
    settings = dict(temperature=0.8, top_k=20, top_p=0.9)
    tokens = model.generate(prompts, 6, uniforms=uniforms, **settings)
    assert tokens.shape == (2, 6) and bool(((tokens >= 0) & (tokens < 1000)).all())
    # the same loop, step by step, with the sampling checked against the definition
    cache = model.make_cache(sequences=2, max_length=51)
    counts, ids = [5, 45], torch.cat(prompts)
    for step in range(6):
        cache.begin_step(counts)
        logits = model.serve(ids, cache)
        ids, _ = check_sample(logits, uniforms[step].cpu(), **settings)
        assert torch.equal(ids, tokens[:, step])
        counts = [1, 1]


def test_captured_step_replays_with_new_lengths_and_beside_another_graph():
    """A decode step captured once is replayed as the sequences grow; two graphs alive at a time share
    no workspace."""

    model = small_stack(seed=5)
    prompts = [torch.arange(3, device="cuda"), torch.arange(100, 180, device="cuda")]
    uniforms = torch.rand(8, 2, device="cuda")
    expect = model.generate(prompts, 8, uniforms=uniforms, top_p=0.9)

    from ue5m3_fp4 import serving

    def capture(cache, ids, u):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # warm-up: libraries load and allocate outside the capture
            serving.sample_tokens(model.serve(ids, cache), u, top_p=0.9)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            tokens, logprobs = serving.sample_tokens(model.serve(ids, cache), u, top_p=0.9)
        return graph, tokens

    runs = []
    for _ in range(2):
        cache = model.make_cache(sequences=2, max_length=128, page_size=16)
        cache.begin_step([3, 80])
        first, _ = serving.sample_tokens(model.serve(torch.cat(prompts), cache), uniforms[0], top_p=0.9)
        ids, u = first.clone(), uniforms[1].clone()
        cache.begin_step([1, 1])
        cache.max_kv_length = 128  # the graph's launches are sized for the longest
        graph, tokens = capture(cache, ids, u)
        runs.append((cache, ids, u, graph, tokens, [first]))
    for step in range(1, 8):
        for cache, ids, u, graph, tokens, out in runs:
            if step > 1:
                cache.begin_step([1, 1])
            ids.copy_(out[-1])
            u.copy_(uniforms[step])
        for cache, ids, u, graph, tokens, out in runs:
            graph.replay()
        for cache, ids, u, graph, tokens, out in runs:
            out.append(tokens.clone())
    for *_, out in runs:
        assert torch.equal(torch.stack(out, 1), expect)


def test_operators_on_another_stream():
    from ue5m3_fp4 import serving

    codes, scales = (t.cuda() for t in packed_weight(512, 1024, 16, True, 0))
    x = torch.randn(4, 1024, device="cuda").to(torch.bfloat16)
    logits, u = torch.randn(4, 30000, device="cuda"), torch.rand(4, device="cuda")
    kw = dict(rows=512, cols=1024, block_size=16, two_dimensional=True, tensor_amax=1.0)
    expect = serving.packed_matvec(x, codes, scales, **kw), serving.sample_tokens(logits, u, top_p=0.9)[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for _ in range(5):
        for stream in streams:
            with torch.cuda.stream(stream):
                results.append((serving.packed_matvec(x, codes, scales, **kw), serving.sample_tokens(logits, u, top_p=0.9)[0]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, expect[0]) and torch.equal(b, expect[1]) for a, b in results)
