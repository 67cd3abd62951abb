"""Operators of an 8-bit paged KV cache: their plain forms, and the framework's calls for them.

The cache holds K and V as e4m3 values, ``[blocks, block_size, kv_heads, head_dim]`` per layer, and for each block of
tokens and KV head one power of two for K and one for V: ``scales[block, head, 0 or 1]`` is the biased exponent e of a
scale 2^(e - 127). A cached value stands for e4m3 * scale. Four kinds of case:

  decode    one query per row over the row's pages (``paged_attention_q8``), also under a sliding window
  prefill   packed causal chunks, one-query rows among them (``paged_prefill_attention_q8``)
  append    a step's new K/V rows quantised into the pages of one layer, whose scales may rise (``kv_append_q8``), and
            the written pages read back as the values that they stand for (``kv_read_q8``)
  metadata  a step's block tables, cumulative query counts, positions and write addresses, from the lengths that the
            requests have on the GPU (``sequence_kv_metadata``)

``listed()`` names twelve cases, ``draw(rng)`` gives others of the same ranges: 1 to 64 decode rows with contexts of 1
to 32768 tokens, 1 to 16 prompt chunks of 1 to 512 queries, appends of 1 to 8192 rows, 1 to 512 requests; 16 x 128
heads (multi-head) and 8 KV heads shared by 32 or 64 query heads; pages of 16, 32 or 64 tokens scattered over the pool.
Lengths belong to the case (``lengths`` seeds them); values and page placement come from the seed of ``prepare``.
"""

import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-rlt_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
E4M3 = torch.float8_e4m3fn
LEAST = 27  # smallest biased exponent of a scale: 2^-100


def _case(name, kind, **kw):
    case = {"kind": kind, "dtype": "bf16", "q_heads": 16, "kv_heads": 16, "head_dim": 128, "block": 16, "lengths": 2}
    case.update(kw)
    return {"name": name, **case} if name else case


def _decode(name=None, **kw):
    return _case(name, "decode", **{"layers": 1, "rows": 1, "low": 16, "high": 512, "window": 0, "width": 0, **kw})


def _prefill(name=None, **kw):
    return _case(name, "prefill", **{"prompts": 1, "q_low": 512, "q_high": 512, "prefix_low": 0, "prefix_high": 0,
                                     "decode_rows": 0, "low": 256, "high": 4096, **kw})


def _append(name=None, **kw):
    return _case(name, "append", **{"prompts": 1, "q_low": 1, "q_high": 1, "prefix_low": 0, "prefix_high": 0,
                                    "decode_rows": 0, "low": 16, "high": 512, **kw})


def _metadata(name=None, **kw):
    case = {"kind": "metadata", "block": 16, "lengths": 2, "slots": 256, "width": 512, "spare": 0, "prompts": 1, "q_low": 1,
            "q_high": 512, "prefix_low": 0, "prefix_high": 4096, "decode_rows": 0, "low": 16, "high": 4096, **kw}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One user's chat deep into a long context: a single row, latency of one token.
        _decode("decode_one_row_long", rows=1, low=24001, high=24001),
        # The fp32 check-out shape: 8 rows, short contexts, float32 queries.
        _decode("decode_f32_8_rows", dtype="f32", rows=8, low=64, high=512),
        # The headline step: 64 requests, 16 x 128 heads, a pool of several layers.
        _decode("decode_64_rows", rows=64, layers=4, low=512, high=4096),
        # Grouped-query heads in float16, a batch that is no power of two.
        _decode("decode_gqa_f16", dtype="f16", q_heads=32, kv_heads=8, rows=37, low=300, high=6000),
        # Sliding-window attention under the fixed-width tables of a captured graph.
        _decode("decode_window_wide_table", rows=24, low=64, high=8192, window=1024, width=2048),
        # One request's prompt chunk with nothing else to run: time to first token.
        _prefill("prefill_one_chunk", prompts=1, prefix_low=6656, prefix_high=6656),
        # The mixed step: 16 prompts' chunks packed with 48 decode rows.
        _prefill("prefill_mixed", prompts=16, q_low=212, q_high=512, prefix_low=0, prefix_high=7680, decode_rows=48),
        # Short ragged prompts over grouped-query heads in float16, head_dim 64.
        _prefill("prefill_gqa_ragged_f16", dtype="f16", q_heads=32, kv_heads=8, head_dim=64, prompts=7, q_low=17,
                 q_high=390, prefix_low=0, prefix_high=2900),
        # A decode step's append: one new token of 64 requests, in the middle of their pages.
        _append("append_decode_step", prompts=0, decode_rows=64, low=512, high=4096),
        # The mixed step's append: 16 prompts' chunks that start anywhere in a page.
        _append("append_chunks", prompts=16, q_low=480, q_high=512, prefix_low=0, prefix_high=7680, decode_rows=39),
        # The mixed step's metadata: chunks and decode rows of 64 requests, from lengths on the GPU.
        _metadata("metadata_mixed_step", prompts=16, q_low=480, q_high=512, prefix_high=7680, decode_rows=48, spare=100),
        # A wide decode step: 500 requests under tables of a captured graph.
        _metadata("metadata_wide_tables", slots=1024, width=2048, prompts=0, decode_rows=500, low=16, high=32768, spare=12),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["decode"] * 4 + ["prefill"] * 3 + ["append"] * 2 + ["metadata"])
    seed = rng.randrange(1 << 20)
    block = rng.choice([16, 16, 16, 32, 64])
    if kind == "metadata":
        top = _log(rng, 64, 32000)
        return _metadata(block=block, lengths=seed, slots=1024, width=-(-32768 // block), spare=rng.choice([0, rng.randint(1, 200)]),
                         prompts=rng.choice([0, _log(rng, 1, 16)]), q_high=_log(rng, 1, 512), prefix_low=0, prefix_high=top,
                         decode_rows=_log(rng, 1, 496), low=1, high=top)
    q_heads, kv_heads = rng.choice([(16, 16), (16, 16), (32, 8), (64, 8)])
    shape = {"q_heads": q_heads, "kv_heads": kv_heads, "head_dim": rng.choice([64, 128, 128]), "block": block, "lengths": seed}
    if kind == "append":
        high = _log(rng, 1, 512)
        prefix = rng.choice([0, _log(rng, 16, 7680)])
        return _append(dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), prompts=_log(rng, 1, 15), q_low=rng.randint(1, high),
                       q_high=high, prefix_low=rng.randint(0, prefix), prefix_high=prefix,
                       decode_rows=rng.choice([0, _log(rng, 1, 64)]), low=1, high=_log(rng, 16, 7680), **shape)
    if kind == "prefill":
        high = _log(rng, 16, 512)
        prefix = rng.choice([0, _log(rng, 16, 7680)])
        return _prefill(dtype=rng.choice(["bf16", "bf16", "f16"]), q_low=rng.randint(1, high), q_high=high,
                        prompts=_log(rng, 1, 16 if q_heads == 16 else 8 if q_heads == 32 else 4),
                        prefix_low=rng.randint(0, prefix), prefix_high=prefix, decode_rows=rng.choice([0, _log(rng, 1, 48)]), **shape)
    rows = _log(rng, 1, 64)
    # No more K/V than the listed 64 rows read.
    high = _log(rng, 16, min(32768, 64 * 2200 * 16 // (rows * kv_heads)))
    return _decode(dtype=rng.choice(["bf16", "bf16", "bf16", "f16", "f32"]), rows=rows, low=rng.randint(1, high), high=high,
                   window=rng.choice([0, 0, 0, _log(rng, 16, 2048)]), width=rng.choice([0, 0, -(-33000 // block)]), **shape)


# ------------------------------------------------------------------- lengths
def _spread(seed, count, low, high):
    rng = random.Random(seed)
    return [rng.randint(low, high) for _ in range(count)]


def _sequences(case):
    """(query count, context length) of every sequence: the chunks, then the decode rows."""
    if case["kind"] == "decode":
        return [(1, n) for n in _spread(case["lengths"], case["rows"], case["low"], case["high"])]
    qs = _spread(case["lengths"], case["prompts"], case["q_low"], case["q_high"])
    before = _spread(case["lengths"] + 1, case["prompts"], case["prefix_low"], case["prefix_high"])
    rows = _spread(case["lengths"] + 2, case["decode_rows"], case["low"], case["high"])
    return [(q, p + q) for q, p in zip(qs, before)] + [(1, n) for n in rows]


def _cut(case):
    """Metadata: (query count, context length) that fit the tables."""
    cap = case["width"] * case["block"]
    return [(q - max(0, n - cap), min(n, cap)) for q, n in _sequences(case)]


def _touched(case):
    """Pages that an append writes, and tokens of them that an earlier append wrote."""
    bs, pages, old = case["block"], 0, 0
    for q, n in _sequences(case):
        pages += -(-n // bs) - (n - q) // bs
        old += (n - q) % bs
    return pages, old


# ------------------------------------------------------------------ prepare
def _exponents(amax):
    """Biased exponent of the least power of two s with amax <= 448 s (448 = 0.875 * 2^9, the largest e4m3 value)."""
    mantissa, exponent = torch.frexp(amax)
    e = exponent.to(torch.int32) - 9 + (mantissa > 0.875).to(torch.int32) + 127
    return torch.where(amax > 0, e, torch.zeros_like(e)).clamp(LEAST, 254)


def _power(e):
    return torch.exp2(e.to(torch.float32) - 127)


def _pool(case, blocks, gen, device):
    """One layer of a pool that earlier steps filled: heads and pages differ in magnitude."""
    layers, bs, heads, dim = case.get("layers", 1), case["block"], case["kv_heads"], case["head_dim"]
    scales = torch.zeros((blocks, layers, heads, 2), dtype=torch.uint8, device=device)
    caches = []
    for part in range(2):
        store = torch.zeros((blocks, layers, heads, bs, dim), dtype=torch.uint8, device=device)
        for first in range(0, blocks, 4096):
            n = min(4096, blocks - first)
            x = torch.empty((n, heads, bs, dim), device=device).normal_(generator=gen)
            x *= torch.empty((n, heads, 1, 1), device=device).uniform_(-1.5, 1.5, generator=gen).exp()
            e = _exponents(x.abs().amax((2, 3)))
            store[first : first + n, layers // 2] = (x / _power(e)[:, :, None, None]).to(E4M3).view(torch.uint8)
            scales[first : first + n, layers // 2, :, part] = e.to(torch.uint8)
        caches.append(store.view(E4M3)[:, layers // 2].transpose(1, 2))
    return caches[0], caches[1], scales[:, layers // 2]


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    seqs = _sequences(case)
    bs = case["block"]
    ints = {"dtype": torch.int32, "device": device}
    lengths = torch.tensor([n for _, n in seqs], **ints)
    if case["kind"] == "metadata":
        order = torch.randperm(case["slots"], generator=gen, device=device)[: len(seqs)]
        tables = torch.randint(0, 1 << 20, (case["slots"], case["width"]), generator=gen, **ints)
        return {"kind": "metadata", "block": bs, "tables": tables, "rows": order, "lengths": lengths, "width": case["width"],
                "counts": torch.tensor([q for q, _ in seqs], **ints), "tokens": sum(q for q, _ in seqs) + case["spare"]}
    counts = [-(-n // bs) for _, n in seqs]
    order = torch.randperm(sum(counts), generator=gen, device=device).to(torch.int32)
    tables = torch.full((len(seqs), max(case.get("width", 0), max(counts))), -1, **ints)
    at, cu, touched = 0, [0], []
    for r, (q, n) in enumerate(seqs):
        tables[r, : counts[r]] = order[at : at + counts[r]]
        at += counts[r]
        cu.append(cu[-1] + q)
        touched.append(tables[r, (n - q) // bs : counts[r]])
    key_cache, value_cache, scales = _pool(case, sum(counts), gen, device)
    s = {"kind": case["kind"], "key_cache": key_cache, "value_cache": value_cache, "scales": scales, "tables": tables, "lengths": lengths,
         "cu": torch.tensor(cu, **ints), "max_q": max(q for q, _ in seqs), "max_n": max(n for _, n in seqs), "window": case.get("window", 0)}
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "append":
        # New tokens of another magnitude than the pages' older ones, so that some scales rise.
        for name in ("k", "v"):
            x = torch.empty((cu[-1], case["kv_heads"], case["head_dim"]), device=device).normal_(generator=gen)
            s[name] = (x * torch.empty((cu[-1], 1, 1), device=device).uniform_(-1.5, 1.5, generator=gen).exp()).to(dtype)
        return {**s, "pages": torch.cat(touched).long(), "dtype": dtype}
    s["q"] = torch.empty((cu[-1], case["q_heads"], case["head_dim"]), dtype=dtype, device=device).normal_(generator=gen)
    return s


# ---------------------------------------------------------------------- run
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    cache = () if s["kind"] == "metadata" else (s["key_cache"], s["value_cache"], s["scales"])
    if s["kind"] == "decode":
        from vllm_rlt.kernels.hip_attention_q8 import paged_attention_q8

        return paged_attention_q8(s["q"], *cache, s["tables"], s["lengths"], s["window"])
    if s["kind"] == "prefill":
        from vllm_rlt.kernels.hip_attention_q8 import paged_prefill_attention_q8

        return paged_prefill_attention_q8(s["q"], *cache, s["tables"], s["lengths"], s["cu"], s["max_q"])
    if s["kind"] == "append":
        from vllm_rlt.kernels.hip_attention_q8 import kv_append_q8, kv_read_q8

        kv_append_q8(*cache, s["k"], s["v"], s["tables"], s["lengths"], s["cu"])
        return kv_read_q8(*cache, s["pages"], s["dtype"])
    from vllm_rlt.worker.metadata import sequence_kv_metadata

    m = sequence_kv_metadata(s["tables"], s["rows"], s["lengths"], s["counts"], block_size=s["block"], tokens=s["tokens"], width=s["width"])
    return (m.position_ids, m.write_blocks, m.write_offsets, m.write_mask, m.block_tables, m.context_lengths, m.cu_seqlens_q)


def _plain(s):
    if s["kind"] == "metadata":
        return _plain_metadata(s)
    if s["kind"] == "append":
        return _plain_append(s)
    return _plain_attention(s)


def _read(cache, scales, pages):
    """The values that pages stand for, in float32: [*pages.shape, block, heads, dim]."""
    raw = cache.view(torch.uint8)[pages].view(E4M3).float()
    return raw * _power(scales[pages])[..., None, :, None]


def _plain_attention(s):
    q, cu, lengths = s["q"], s["cu"].long(), s["lengths"].long()
    rows, heads, dim = lengths.shape[0], q.shape[1], q.shape[2]
    bs, kv = s["key_cache"].shape[1:3]
    group, most, device = heads // kv, s["max_q"], q.device
    pages = s["tables"][:, : -(-s["max_n"] // bs)].long().clamp(min=0)
    k = _read(s["key_cache"], s["scales"][..., 0], pages).flatten(1, 2).permute(0, 2, 3, 1)  # [rows, kv, dim, tokens]
    v = _read(s["value_cache"], s["scales"][..., 1], pages).flatten(1, 2).permute(0, 2, 1, 3)
    # Queries of a sequence side by side, padded to the longest chunk.
    step = torch.arange(most, device=device)
    count = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + step).clamp(max=q.shape[0] - 1)
    qs = q[at].float().view(rows, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(rows, kv, group * most, dim)
    scores = torch.matmul(qs, k).view(rows, kv, group, most, -1) / math.sqrt(dim)
    position = (lengths - count)[:, None] + step
    token = torch.arange(k.shape[-1], device=device)
    hidden = token > position[..., None]
    if s["window"]:
        hidden |= token <= position[..., None] - s["window"]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(rows, kv, group * most, -1), v).view(rows, kv, group, most, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.permute(0, 3, 1, 2, 4).reshape(rows, most, heads, dim)[step < count[:, None]].to(q.dtype)


def _plain_append(s):
    """Every page that a sequence's new tokens reach, side by side: [sequences, pages, block, heads, dim]."""
    tables, lengths, cu = s["tables"].long(), s["lengths"].long(), s["cu"].long()
    bs, device = s["key_cache"].shape[1], tables.device
    before = lengths - (cu[1:] - cu[:-1])
    page = before[:, None] // bs + torch.arange((s["max_q"] + bs - 2) // bs + 1, device=device)
    written = page * bs < lengths[:, None]
    block = tables.gather(1, page.clamp(max=tables.shape[1] - 1))[written]
    position = (page[..., None] * bs + torch.arange(bs, device=device))[written]  # [pages, block]
    first = before[:, None].expand_as(page)[written][:, None]
    end = lengths[:, None].expand_as(page)[written][:, None]
    row = (cu[:-1, None].expand_as(page)[written][:, None] + position - first).clamp(0, s["k"].shape[0] - 1)
    new = ((position >= first) & (position < end))[..., None, None]
    old = (position < first)[..., None, None]
    store = s["scales"].clone()
    out = []
    for part, (cache, values) in enumerate(((s["key_cache"], s["k"]), (s["value_cache"], s["v"]))):
        x = values[row].float() * new
        e = _exponents(x.abs().amax((1, 3)))
        was = store[block][..., part].to(torch.int32)
        e = torch.where(old.any(1)[:, :, 0], torch.maximum(e, was), e)
        raw = cache.view(torch.uint8)[block]
        again = (raw.view(E4M3).float() * torch.exp2((was - e).float())[:, None, :, None]).to(E4M3)
        fresh = (x * torch.exp2((127 - e).float())[:, None, :, None]).to(E4M3)
        raw = torch.where(new, fresh.view(torch.uint8), torch.where(old, again.view(torch.uint8), raw))
        cache.view(torch.uint8)[block] = raw
        s["scales"][block, :, part] = e.to(torch.uint8)
        out.append(_read(cache, s["scales"][..., part], s["pages"]).to(s["dtype"]))
    return tuple(out)


def _plain_metadata(s):
    tables, rows, bs, tokens = s["tables"].long(), s["rows"], s["block"], s["tokens"]
    device = tables.device
    width = min(tables.shape[1], s["width"])
    length = s["lengths"].long().clamp(min=0)
    count = torch.minimum(s["counts"].long().clamp(min=0), length)
    fits = length.clamp(max=width * bs)
    count = (count - (length - fits)).clamp(min=0)
    end = count.cumsum(0)
    keep = (tokens - (end - count)).clamp(min=0).minimum(count)  # the step's tokens end at `tokens`
    length = fits - (count - keep)
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=device), keep.cumsum(0)])
    column = torch.arange(s["width"], device=device)
    mine = tables[rows][:, : s["width"]]
    block_tables = torch.where(column < ((length + bs - 1) // bs)[:, None], mine, torch.full_like(mine, -1))
    token = torch.arange(tokens, device=device)
    sequence = (token[:, None] >= cu[1:]).sum(1)
    mask = sequence < rows.shape[0]
    sequence = sequence.clamp(max=rows.shape[0] - 1)
    position = torch.where(mask, (length - keep)[sequence] + token - cu[sequence], torch.zeros_like(token))
    blocks = torch.where(mask, mine[sequence, position // bs], torch.zeros_like(token))
    return position, blocks, position % bs * mask, mask, block_tables.int(), length.int(), cu.int()


# --------------------------------------------------------------------- work
def work(case):
    seqs = _sequences(case)
    bs = case["block"]
    if case["kind"] == "metadata":
        entries = sum(-(-n // bs) for _, n in _cut(case))
        tokens = sum(q for q, _ in seqs) + case["spare"]
        # Page ids in, whole tables out; 25 bytes a token, and per request its slot, lengths and cumulative count.
        return {"bytes": 4 * entries + 4 * case["width"] * len(seqs) + 25 * tokens + 24 * len(seqs), "flops": 0}
    es = BYTES[case["dtype"]]
    slot = case["kv_heads"] * case["head_dim"]
    if case["kind"] == "append":
        rows = sum(q for q, _ in seqs)
        pages, old = _touched(case)
        # New rows in and quantised; the touched pages back, as values, with their scales. The older tokens of a
        # touched page are read with it.
        return {"bytes": 2 * rows * slot * (es + 1) + 2 * pages * bs * slot * (1 + es) + 4 * pages * case["kv_heads"], "flops": 2 * (3 * rows + 2 * old) * slot}
    total = read = 0
    width = case["q_heads"] * case["head_dim"]
    for q, n in seqs:
        seen = min(n, case["window"] + q - 1) if case.get("window") else n
        total += q * n - q * (q - 1) // 2 if not case.get("window") else seen
        read += 2 * seen * slot + -(-seen // bs) * (4 + 2 * case["kv_heads"]) + 2 * q * width * es
    return {"bytes": read, "flops": 4 * width * total}


# -------------------------------------------------------------------- exact
def _e4m3(x):
    """x in float64, rounded to e4m3: 4 significant bits down to 2^-6, multiples of 2^-9 below, ties to even."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def _values(cache, scales, pages):
    pages = pages.long()
    return cache.view(torch.uint8)[pages].view(E4M3).double() * torch.exp2(scales[pages].double() - 127)[:, None, :, None]


def _attend(q, k, v, first, start, window):
    """Softmax attention in float64: q [n, Hq, D] at positions first.., k and v [m, Hkv, D] at positions start.. ."""
    n, heads, dim = q.shape
    kv = k.shape[1]
    group = heads // kv
    qd = q.double().view(n, kv, group, dim).permute(1, 2, 0, 3).reshape(kv, group * n, dim).contiguous()
    kd, vd = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    scores = torch.matmul(qd, kd).view(kv, group, n, -1) / math.sqrt(dim)
    at = torch.arange(k.shape[0], device=q.device) + start
    here = first + torch.arange(n, device=q.device)[:, None]
    scores.masked_fill_(at > here, -math.inf)
    if window:
        scores.masked_fill_(at <= here - window, -math.inf)
    out = torch.matmul(torch.softmax(scores, -1).view(kv, group * n, -1), vd)
    return out.view(kv, group, n, dim).permute(2, 0, 1, 3).reshape(n, heads, dim)


def exact(case, seed):
    s = prepare(case, seed)
    seqs, bs = _sequences(case), case["block"]
    if case["kind"] == "metadata":
        return _exact_metadata(case, s)
    if case["kind"] == "append":
        return _exact_append(case, s)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    at = 0
    for r, (q, n) in enumerate(seqs):
        start = max(0, n - q + 1 - case["window"]) if case.get("window") else 0
        pages = s["tables"][r, start // bs : -(-n // bs)]
        cut = slice(start % bs, start % bs + n - start)
        k, v = (_values(c, s["scales"][..., i], pages).flatten(0, 1)[cut] for i, c in enumerate((s["key_cache"], s["value_cache"])))
        out[at : at + q] = _attend(s["q"][at : at + q], k, v, n - q, start, case.get("window", 0))
        at += q
    return out


def _exact_append(case, s):
    bs, outs = case["block"], []
    for part, (cache, new) in enumerate(((s["key_cache"], s["k"]), (s["value_cache"], s["v"]))):
        got, at = [], 0
        for r, (q, n) in enumerate(_sequences(case)):
            x = new[at : at + q].double()
            at += q
            lead = (n - q) % bs
            pages = s["tables"][r, (n - q) // bs : -(-n // bs)].long()
            raw = cache.view(torch.uint8)[pages].view(E4M3).double()
            was = s["scales"][pages, :, part].double() - 127
            bare = torch.zeros((len(pages) * bs, *x.shape[1:]), dtype=torch.float64, device=x.device)
            bare[lead : lead + q] = x
            bare = bare.view(len(pages), bs, *x.shape[1:])
            top = bare.abs().amax((1, 3))
            e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -120) / 448)).clamp(min=LEAST - 127)
            if lead:
                e[0] = torch.maximum(e[0], was[0])
            scale = torch.exp2(e)[:, None, :, None]
            kept = _e4m3(raw * torch.exp2(was - e)[:, None, :, None])
            token = torch.arange(len(pages) * bs, device=x.device).view(len(pages), bs, 1, 1)
            done = torch.where(token < lead, kept, torch.where(token < lead + q, _e4m3(bare / scale), raw))
            got.append(done * scale)
        outs.append(torch.cat(got))
    return tuple(outs)


def _exact_metadata(case, s):
    tables, rows, bs = s["tables"].tolist(), s["rows"].tolist(), case["block"]
    positions, blocks, offsets, block_tables, cu = [], [], [], [], [0]
    for row, (q, n) in zip(rows, _cut(case)):
        mine = range(n - q, n)
        positions += mine
        blocks += [tables[row][p // bs] for p in mine]
        offsets += [p % bs for p in mine]
        used = -(-n // bs)
        block_tables.append(tables[row][:used] + [-1] * (case["width"] - used))
        cu.append(cu[-1] + q)
    pad = [0] * (s["tokens"] - len(positions))
    mask = [True] * len(positions) + [False] * len(pad)
    long = {"dtype": torch.int64, "device": s["tables"].device}
    ints = {"dtype": torch.int32, "device": s["tables"].device}
    return (torch.tensor(positions + pad, **long), torch.tensor(blocks + pad, **long), torch.tensor(offsets + pad, **long),
            torch.tensor(mask, device=s["tables"].device), torch.tensor(block_tables, **ints), torch.tensor([n for _, n in _cut(case)], **ints),
            torch.tensor(cu, **ints))
