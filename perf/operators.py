"""The operators with which a frozen, packed FP4 model answers token by token: cases, plain forms
and exact values.

* ``matvec``: a few rows of activations times a packed weight (E2M1 codes, UE5M3 block scales);
* ``attention``: a chunk of new tokens per sequence is written into a paged key/value cache and
  attends to everything the cache then holds of its sequence;
* ``sample``: the next token of every row of logits, with temperature, top-k, top-p and min-p, from
  given uniform numbers.

``run`` computes the plain form where ``own`` is false, and calls the framework's entry points where
it is true.  Sizes are those of the package's Nemotron-H-shaped stack (hidden 4096, MLP 21504, 32
query heads over 4 key/value heads of width 128, vocabulary 131072) and odd ones between.
"""

import math
import random
import sys
from pathlib import Path

import torch

# the package lies in a folder of its own below the repository's root
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "ue5m3-fp4_b200"))

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one token through k_proj: the smallest product of a decode step, where latency counts
        _matvec("matvec_one_token_512x4096", 1, 512, 4096, 16, True, "bf16", False),
        # one token through up_proj, the largest weight of the stack
        _matvec("matvec_one_token_21504x4096", 1, 21504, 4096, 16, True, "bf16", False),
        # eight sequences decoding together through down_proj, 1 x 32 blocks
        _matvec("matvec_8_rows_4096x21504", 8, 4096, 21504, 32, False, "bf16", False),
        # a small projection with ragged sizes, fp32 activations and a bias
        _matvec("matvec_fp32_5_rows_777x1003", 5, 777, 1003, 16, False, "fp32", True),
        # one sequence, one new token, a long context: the batch-1 decode step
        _attention("attention_1_token_of_32768", 1, 1, 32768, 4, 8, 128, 64, 0),
        # a serving batch of single tokens with contexts from one token to 8192
        _attention("attention_64_tokens_ragged", 64, 1, 8192, 4, 8, 128, 16, 7),
        # a prompt's chunk of 2048 tokens behind 6144 that the cache already holds
        _attention("attention_chunk_2048_of_8192", 1, 2048, 8192, 4, 8, 128, 64, 0),
        # prompts and single tokens in one batch, narrow heads, odd lengths, short pages
        _attention("attention_mixed_chunks_head64", 9, 411, 3001, 2, 7, 64, 16, 11),
        # one row over the whole vocabulary, as in a batch-1 token loop
        _sample("sample_1_row_top_k_top_p", 1, 131072, "fp32", 0.0, 50, 0.95, 0.0, 0),
        # a batch with nucleus sampling only: the whole row carries weight
        _sample("sample_64_rows_top_p", 64, 131072, "fp32", 0.1, 0, 0.9, 0.0, 0),
        # rows that each bring their own settings, bf16 logits (many ties), an odd vocabulary
        _sample("sample_17_rows_mixed_bf16", 17, 32003, "bf16", 0.3, 40, 0.9, 0.05, 5),
    ]


def draw(rng):
    kind = rng.choice(("matvec", "attention", "sample"))
    if kind == "matvec":
        m = _spread(rng, 1, 64)
        n, k = _spread(rng, 16, 21504), _spread(rng, 16, 21504)
        n = max(16, min(n, 4096 * 21504 * 8 // (k * m), 4096 * 21504 // k))
        return _matvec(None, m, n, k, rng.choice((16, 32)), rng.random() < 0.5, rng.choice(("bf16", "fp32")),
                       rng.random() < 0.5)
    if kind == "attention":
        kv_heads, group, head_dim = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 5, 8)), rng.choice((64, 128))
        batch = _spread(rng, 1, 64)
        kv = _spread(rng, 1, 16384 if batch < 16 else 4096)
        pairs = 2048 * 6000 * 32 // (batch * kv_heads * group * kv)  # what the largest listed case has
        query = min(kv, 2048, max(1, pairs), _spread(rng, 1, 2048))
        return _attention(None, batch, query, kv, kv_heads, group, head_dim, rng.choice((16, 32, 64, 128)),
                          rng.randrange(1, 1 << 20))
    rows, vocabulary = _spread(rng, 1, 64), _spread(rng, 100, 131072)
    return _sample(None, rows, vocabulary, rng.choice(("bf16", "fp32")), rng.choice((0.0, 0.2)),
                   rng.choice((0, _spread(rng, 1, 1000))), rng.choice((1.0, round(rng.uniform(0.1, 0.99), 3))),
                   rng.choice((0.0, round(rng.uniform(0.001, 0.3), 4))), rng.randrange(0, 1 << 20))


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _named(name, case):
    return case if name is None else {"name": name, **case}


def _matvec(name, rows, n, k, block, two_dimensional, dtype, bias):
    return _named(name, {"kind": "matvec", "rows": rows, "n": n, "k": k, "block": block,
                         "two_dimensional": two_dimensional, "dtype": dtype, "bias": bias})


def _attention(name, batch, query, kv, kv_heads, group, head_dim, page, ragged):
    """ragged = 0: every sequence has ``query`` new tokens and ``kv`` in all; otherwise lengths between
    one and these, from a generator started with that number (one sequence has the full lengths)."""

    return _named(name, {"kind": "attention", "batch": batch, "query": query, "kv": kv, "kv_heads": kv_heads,
                         "group": group, "head_dim": head_dim, "page": page, "ragged": ragged})


def _sample(name, rows, vocabulary, dtype, masked, top_k, top_p, min_p, mixed):
    """masked: share of the vocabulary at minus infinity; mixed != 0: settings differ from row to row."""

    return _named(name, {"kind": "sample", "rows": rows, "vocabulary": vocabulary, "dtype": dtype, "masked": masked,
                         "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed})


def _lengths(case):
    batch, query, kv = case["batch"], case["query"], case["kv"]
    if not case["ragged"]:
        return [query] * batch, [kv] * batch
    rng = random.Random(case["ragged"])
    kvs = [rng.randint(1, kv) for _ in range(batch)]
    kvs[rng.randrange(batch)] = kv
    queries = [min(length, 1 if rng.random() < 0.3 else rng.randint(1, query)) for length in kvs]
    queries[kvs.index(kv)] = query
    return queries, kvs


def _settings(case):
    """Temperature, top-k, top-p and min-p of every row."""

    rows = case["rows"]
    if not case["mixed"]:
        return [0.8] * rows, [case["top_k"]] * rows, [case["top_p"]] * rows, [case["min_p"]] * rows
    rng = random.Random(case["mixed"])
    return ([rng.choice((0.0, 0.5, 0.7, 1.0, 1.3)) for _ in range(rows)],
            [rng.choice((0, 1, case["top_k"], case["top_k"])) for _ in range(rows)],
            [rng.choice((1.0, case["top_p"], case["top_p"])) for _ in range(rows)],
            [rng.choice((0.0, case["min_p"], case["min_p"])) for _ in range(rows)])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"matvec": _prepare_matvec, "attention": _prepare_attention, "sample": _prepare_sample}[case["kind"]](case, g)


def _prepare_matvec(case, g):
    m, n, k, block = case["rows"], case["n"], case["k"], case["block"]
    dtype = _DTYPES[case["dtype"]]
    x = torch.randn(m, k, device="cuda", generator=g)
    # a few channels of the activations are an order of magnitude larger, as after a norm's gain
    x = x * torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, 20.0, 1.0)
    codes = torch.randint(0, 256, (n, (k + 1) // 2), device="cuda", generator=g, dtype=torch.uint8)
    if k % 2:
        codes[:, -1] &= 15
    scale_rows = (n + block - 1) // block if case["two_dimensional"] else n
    # block scales of normal weights under the target 448 lie within a few binades below it
    scales = torch.randint(100, 180, (scale_rows, (k + block - 1) // block), device="cuda", generator=g,
                           dtype=torch.uint8)
    bias = torch.randn(n, device="cuda", generator=g).to(dtype) if case["bias"] else None
    return {"kind": "matvec", "x": x.to(dtype), "codes": codes, "scales": scales, "bias": bias, "n": n, "k": k,
            "block": block, "two_dimensional": case["two_dimensional"], "amax": 0.11, "target": 448.0}


def _prepare_attention(case, g):
    queries, kvs = _lengths(case)
    heads, kv_heads, d, page = case["kv_heads"] * case["group"], case["kv_heads"], case["head_dim"], case["page"]
    batch, tokens = case["batch"], sum(queries)
    pages = [(length + page - 1) // page for length in kvs]
    count, width = sum(pages) + 3, max(pages)
    bf16 = torch.bfloat16
    state = {"kind": "attention", "scale": d ** -0.5, "page": page, "max_query": max(queries), "max_kv": max(kvs)}
    state["q"] = torch.randn(tokens, heads, d, device="cuda", generator=g).mul_(2.0).to(bf16)
    state["new_k"] = torch.randn(tokens, kv_heads, d, device="cuda", generator=g).to(bf16)
    state["new_v"] = torch.randn(tokens, kv_heads, d, device="cuda", generator=g).to(bf16)
    state["k_pages"] = torch.randn(count, page, kv_heads, d, device="cuda", generator=g).to(bf16)
    state["v_pages"] = torch.randn(count, page, kv_heads, d, device="cuda", generator=g).to(bf16)
    # pages of a sequence lie anywhere in the cache; entries behind its last page are not set
    order = torch.randperm(count, device="cuda", generator=g).to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(width, device="cuda")[None, :] < torch.tensor(pages, device="cuda")[:, None]
    table[held] = order[:sum(pages)]
    state["page_table"] = table
    state["kv_lengths"] = torch.tensor(kvs, dtype=torch.int32, device="cuda")
    starts = [0]
    for length in queries:
        starts.append(starts[-1] + length)
    state["query_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    return state


def _prepare_sample(case, g):
    rows, vocabulary = case["rows"], case["vocabulary"]
    logits = torch.randn(rows, vocabulary, device="cuda", generator=g).mul_(2.5)
    # a handful of likely tokens stand above the rest, as in a language model's logits
    likely = torch.randint(0, vocabulary, (rows, 12), device="cuda", generator=g)
    logits.scatter_add_(1, likely, torch.rand(rows, 12, device="cuda", generator=g) * 8.0)
    if case["masked"]:
        logits.masked_fill_(torch.rand(rows, vocabulary, device="cuda", generator=g) < case["masked"], -math.inf)
    temperature, top_k, top_p, min_p = _settings(case)
    on_gpu = lambda values, dtype: torch.tensor(values, dtype=dtype, device="cuda")  # noqa: E731
    return {"kind": "sample", "logits": logits.to(_DTYPES[case["dtype"]]),
            "uniforms": torch.rand(rows, device="cuda", generator=g),
            "temperature": on_gpu(temperature, torch.float32), "top_k": on_gpu(top_k, torch.int32),
            "top_p": on_gpu(top_p, torch.float32), "min_p": on_gpu(min_p, torch.float32)}


def run(state):
    if own:
        return _run_own(state)
    return {"matvec": _plain_matvec, "attention": _plain_attention, "sample": _plain_sample}[state["kind"]](state)


def _run_own(s):
    from ue5m3_fp4 import serving

    if s["kind"] == "matvec":
        return serving.packed_matvec(s["x"], s["codes"], s["scales"], rows=s["n"], cols=s["k"], block_size=s["block"],
                                     two_dimensional=s["two_dimensional"], tensor_amax=s["amax"],
                                     scale_target=s["target"], bias=s["bias"])
    if s["kind"] == "attention":
        out = serving.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_lengths"],
                                      s["query_starts"], max_query_length=s["max_query"], max_kv_length=s["max_kv"],
                                      scale=s["scale"], new_k=s["new_k"], new_v=s["new_v"])
        return out, s["k_pages"], s["v_pages"]
    return serving.sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                                 top_p=s["top_p"], min_p=s["min_p"])


# ---- plain forms: elementary operations, 32 bits or 64 ------------------------------------------


def _decode_scales(scales, dtype):
    """A scale byte E<<3|M: (8 + M) * 2^(E - 18), and M * 2^-17 where E = 0."""

    byte = scales.to(torch.int32)
    exponent, mantissa = byte >> 3, (byte & 7).to(dtype)
    return torch.where(exponent == 0, mantissa * 2.0 ** -17, (8 + mantissa) * torch.exp2((exponent - 18).to(dtype)))


def _weight(s, dtype):
    """The weight's values p * (s * dec) in ``dtype``."""

    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype, device="cuda")
    codes = s["codes"]
    nibbles = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(codes.shape[0], -1)[:, :s["k"]]
    block = s["block"]
    scales = _decode_scales(s["scales"], dtype).repeat_interleave(block, 1)[:, :s["k"]]
    if s["two_dimensional"]:
        scales = scales.repeat_interleave(block, 0)[:s["n"]]
    decode = torch.tensor(s["amax"], dtype=torch.float32).to(dtype) / (6.0 * s["target"])
    return table[nibbles.long()] * (scales * decode.to("cuda"))


def _plain_matvec(s):
    y = s["x"].float() @ _weight(s, torch.float32).T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_attention(s):
    q, starts, lengths, page = s["q"], s["query_starts"].long(), s["kv_lengths"].long(), s["page"]
    tokens, heads, d = q.shape
    batch, kv_heads = lengths.shape[0], s["k_pages"].shape[2]
    # the new keys and values go to their places in the pages
    row = torch.arange(tokens, device="cuda")
    sequence = torch.searchsorted(starts, row, right=True) - 1
    new = starts[1:] - starts[:-1]
    position = lengths[sequence] - new[sequence] + row - starts[sequence]
    target = s["page_table"][sequence, position // page].long()
    s["k_pages"][target, position % page] = s["new_k"]
    s["v_pages"][target, position % page] = s["new_v"]
    # queries, keys and values of every sequence side by side, padded to the longest
    queries, longest = s["max_query"], s["max_kv"]
    index = torch.arange(queries, device="cuda")
    padded = torch.zeros(batch, queries, heads, d, device="cuda")
    padded[sequence, row - starts[sequence]] = q.float()
    padded = padded.reshape(batch, queries, kv_heads, heads // kv_heads, d).permute(0, 2, 3, 1, 4)
    padded = padded.reshape(batch, kv_heads, -1, d)
    table = s["page_table"].clamp(min=0).long()
    k = s["k_pages"][table].reshape(batch, -1, kv_heads, d)[:, :longest].permute(0, 2, 3, 1).float()
    v = s["v_pages"][table].reshape(batch, -1, kv_heads, d)[:, :longest].permute(0, 2, 1, 3).float()
    key = torch.arange(longest, device="cuda")
    last = (lengths - new)[:, None] + index[None, :]
    seen = (key[None, None, :] <= last[:, :, None]) & (key[None, None, :] < lengths[:, None, None])
    seen = seen & (index[None, :, None] < new[:, None, None])
    scores = (padded @ k).mul_(s["scale"]).reshape(batch, kv_heads, heads // kv_heads, queries, longest)
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = weights.reshape(batch, kv_heads, -1, longest) @ v
    out = out.reshape(batch, kv_heads, heads // kv_heads, queries, d) / total.clamp(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, queries, heads, d)
    return out[sequence, row - starts[sequence]].to(q.dtype), s["k_pages"], s["v_pages"]


def _plain_sample(s):
    """In 64 bits: a token is chosen by comparisons of long sums with a border."""

    logits = s["logits"].double()
    rows, vocabulary = logits.shape
    temperature = s["temperature"].double()[:, None]
    greedy = temperature <= 0
    value, order = torch.sort(logits, dim=1, descending=True, stable=True)
    weight = torch.exp((value - value[:, :1]) / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(vocabulary, device="cuda")[None, :]
    top_k = s["top_k"][:, None]
    kept = torch.where(greedy, rank < 1, (rank < top_k) | (top_k <= 0))
    weight = torch.where(kept, weight, 0.0)
    before = torch.cumsum(weight, 1) - weight
    total = weight.sum(1, keepdim=True)
    top_p = s["top_p"].double()[:, None]
    kept = kept & ((before < top_p * total) | (top_p >= 1) | (rank == 0))
    kept = kept & ((weight >= s["min_p"].double()[:, None]) | (rank == 0))
    weight = torch.where(kept, weight, 0.0)
    by_index = torch.zeros_like(weight).scatter_(1, order, weight)
    running = torch.cumsum(by_index, 1)
    border = s["uniforms"].double()[:, None] * running[:, -1:]
    token = ((running <= border) | (by_index == 0)).int().argmin(1)
    chosen = by_index.gather(1, token[:, None])
    logprob = torch.log(chosen / running[:, -1:])[:, 0].float()
    return token, logprob


# ---- exact values, apart from the plain forms ------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"matvec": _exact_matvec, "attention": _exact_attention, "sample": _exact_sample}[case["kind"]](state)


def _exact_matvec(s):
    magnitudes = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.float64, device="cuda") / 2
    low, high = s["codes"].long() % 16, s["codes"].long() // 16
    n, k, block = s["n"], s["k"], s["block"]
    signed = torch.empty(n, low.shape[1] * 2, dtype=torch.float64, device="cuda")
    signed[:, 0::2] = magnitudes[low % 8] * (1 - 2 * (low // 8))
    signed[:, 1::2] = magnitudes[high % 8] * (1 - 2 * (high // 8))
    byte = s["scales"].double()
    exponent = torch.floor(byte / 8)
    mantissa = byte - 8 * exponent
    scales = torch.where(exponent > 0, (1 + mantissa / 8) * 2.0 ** (exponent - 15), mantissa / 8 * 2.0 ** -14)
    amax = float(torch.tensor(s["amax"], dtype=torch.float32))
    y = torch.zeros(s["x"].shape[0], n, dtype=torch.float64, device="cuda")
    row = torch.arange(n, device="cuda") // (block if s["two_dimensional"] else 1)
    for start in range(0, k, 4096):  # bounded memory: the widths of the blocks divide 4096
        stop = min(k, start + 4096)
        column = torch.arange(start, stop, device="cuda") // block
        part = signed[:, start:stop] * scales[row][:, column]
        y += s["x"][:, start:stop].double() @ part.T
    y *= amax / (6.0 * s["target"])
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_attention(s):
    starts, lengths = s["query_starts"].tolist(), s["kv_lengths"].tolist()
    page, kv_heads = s["page"], s["k_pages"].shape[2]
    tokens, heads, d = s["q"].shape
    k_pages, v_pages = s["k_pages"].clone(), s["v_pages"].clone()
    out = torch.zeros(tokens, heads, d, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lengths):
        first, stop = starts[b], starts[b + 1]
        count = stop - first
        place = torch.arange(length - count, length, device="cuda")
        held = s["page_table"][b, :(length + page - 1) // page].long()
        k_pages[held[place // page], place % page] = s["new_k"][first:stop]
        v_pages[held[place // page], place % page] = s["new_v"][first:stop]
        hidden = torch.arange(length, device="cuda")[None, :] > place[:, None]
        for h in range(kv_heads):
            k = k_pages[held][:, :, h].reshape(-1, d)[:length].double()
            v = v_pages[held][:, :, h].reshape(-1, d)[:length].double()
            for head in range(h * heads // kv_heads, (h + 1) * heads // kv_heads):
                scores = s["q"][first:stop, head].double() @ k.T * s["scale"]
                out[first:stop, head] = torch.softmax(scores.masked_fill(hidden, -math.inf), -1) @ v
    return out, k_pages, v_pages


def _exact_sample(s):
    """Row by row, from the definition: threshold values instead of a sorted prefix."""

    tokens, logprobs = [], []
    for r in range(s["logits"].shape[0]):
        logits = s["logits"][r].double()
        heat, top_k = float(s["temperature"][r]), int(s["top_k"][r])
        top_p, min_p, u = float(s["top_p"][r]), float(s["min_p"][r]), float(s["uniforms"][r])
        best = int((logits == logits.max()).nonzero()[0])
        if heat <= 0:
            tokens.append(best)
            logprobs.append(0.0)
            continue
        mass = torch.exp((logits - logits[best]) / heat)
        order = torch.argsort(-logits, stable=True)
        if top_k > 0:
            mass[order[top_k:]] = 0
        if top_p < 1:
            after = torch.flip(torch.cumsum(torch.flip(mass[order], (0,)), 0), (0,))  # this one and all behind it
            drop = after <= (1 - top_p) * after[0]
            drop[0] = False
            trimmed = mass.clone()
            trimmed[order[drop]] = 0
            mass = trimmed
        kept = mass >= min_p
        kept[best] = True
        mass = torch.where(kept, mass, 0.0)
        running = torch.cumsum(mass, 0)
        choice = (running > u * running[-1]) & (mass > 0)
        token = int(choice.nonzero()[0])
        tokens.append(token)
        logprobs.append(math.log(float(mass[token])) - math.log(float(running[-1])))
    return (torch.tensor(tokens, device="cuda"), torch.tensor(logprobs, dtype=torch.float64, device="cuda"))


def work(case):
    if case["kind"] == "matvec":
        m, n, k, block = case["rows"], case["n"], case["k"], case["block"]
        size = 2 if case["dtype"] == "bf16" else 4
        scale_rows = -(-n // block) if case["two_dimensional"] else n
        weight = n * -(-k // 2) + scale_rows * -(-k // block)
        return {"bytes": weight + size * (m * k + m * n + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    if case["kind"] == "attention":
        queries, kvs = _lengths(case)
        kv_heads, d = case["kv_heads"], case["head_dim"]
        heads, tokens = kv_heads * case["group"], sum(queries)
        # keys and values of each sequence are read once, the new ones also written to the pages
        moved = 2 * 2 * kv_heads * d * (sum(kvs) + tokens) + 2 * 2 * tokens * heads * d
        pairs = sum(q * kv - q * (q - 1) // 2 for q, kv in zip(queries, kvs))
        return {"bytes": moved, "flops": 4 * d * heads * pairs}
    size = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": case["rows"] * (case["vocabulary"] * size + 32), "flops": 8 * case["rows"] * case["vocabulary"]}
