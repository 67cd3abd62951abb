"""The torch operators of the 8-bit cache: schemas, no CPU kernels, and one result by every way
to the library (the adapter's one-step calls, its ctypes path, the dispatcher's ops)."""

import numpy as np
import pytest
import torch

from vllm_rlt.kernels._extension import load_extension

SCHEMAS = {
    "paged_attention_q8": "(Tensor q, Tensor key_cache, Tensor value_cache, Tensor scales, Tensor block_tables, "
    "Tensor context_lengths, int window=0) -> Tensor",
    "paged_prefill_q8": "(Tensor q, Tensor key_cache, Tensor value_cache, Tensor scales, Tensor block_tables, "
    "Tensor context_lengths, Tensor cu_seqlens_q, int max_seqlen_q) -> Tensor",
    "kv_append_q8": "(Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor(c!) scales, Tensor k, Tensor v, "
    "Tensor block_tables, Tensor context_lengths, Tensor? cu_seqlens_q=None) -> ()",
    "kv_read_q8": "(Tensor key_cache, Tensor value_cache, Tensor scales, Tensor pages, ScalarType dtype) "
    "-> (Tensor, Tensor)",
    "sequence_metadata": "(Tensor tables, Tensor table_rows, Tensor context_lengths, Tensor query_lengths, int page, "
    "int tokens, int out_width) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
}


def test_schemas():
    load_extension()
    for name, schema in SCHEMAS.items():
        assert str(getattr(torch.ops.vllm_rlt_hip, name).default._schema) == f"vllm_rlt_hip::{name}{schema}"


def test_no_cpu_kernels():
    load_extension()
    cache = torch.zeros((1, 16, 1, 8), dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(NotImplementedError):
        torch.ops.vllm_rlt_hip.kv_read_q8(cache, cache, torch.zeros((1, 1, 2), dtype=torch.uint8),
                                          torch.zeros(1, dtype=torch.int64), torch.float32)


def _case(gpu, dtype, packed=True):
    from test_gpu_q8 import Layer, ints, tables_of

    rng = np.random.default_rng(0)
    lengths, counts = [40, 7, 200], [20, 1, 9]
    tables, blocks = tables_of(rng, lengths, 16)
    layer = Layer(gpu, blocks, 16, 2, 64)
    gen = torch.Generator().manual_seed(1)
    total = sum(counts) if packed else 3
    q = torch.randn((total, 4, 64), generator=gen).to(dtype).to(gpu)
    k, v = torch.randn((2, total, 2, 64), generator=gen).to(dtype).to(gpu)
    cu = ints(np.concatenate([[0], np.cumsum(counts)]), gpu) if packed else None
    return layer, q, k, v, ints(tables, gpu), ints(lengths, gpu), cu, ints(rng.permutation(blocks), gpu, torch.int64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_every_way_gives_the_same_bits(gpu, dtype, monkeypatch):
    from vllm_rlt.kernels import hip_attention, hip_attention_q8 as q8

    load_extension()
    ops = torch.ops.vllm_rlt_hip

    def run(way):
        got = []
        for packed in (True, False):
            layer, q, k, v, tables, lengths, cu, pages = _case(gpu, dtype, packed)
            append = ops.kv_append_q8 if way == "op" else q8.kv_append_q8
            append(*layer.args, k, v, tables, lengths, cu)
            got += [layer.views[0].view(torch.uint8), layer.views[1].view(torch.uint8), layer.scales]
            got += (ops.kv_read_q8 if way == "op" else q8.kv_read_q8)(*layer.args, pages, dtype)
            if packed:
                prefill = ops.paged_prefill_q8 if way == "op" else q8.paged_prefill_attention_q8
                got.append(prefill(q, *layer.args, tables, lengths, cu, 20))
            decode = ops.paged_attention_q8 if way == "op" else q8.paged_attention_q8
            got += [decode(q[:3], *layer.args, tables, lengths, w) for w in (0, 33)]
            meta = ops.sequence_metadata if way == "op" else (
                lambda t, r, n, c, page, tokens, width: hip_attention.sequence_metadata(
                    t, r, n, c, page, tokens=tokens, out_width=width))
            got += meta(tables, torch.tensor([2, 0, 1], device=gpu), lengths, lengths - 5, 16, 250, 15)
        return got

    one_step, op = run("adapter"), run("op")
    monkeypatch.setattr(q8, "plain_calls", lambda: None)
    monkeypatch.setattr(hip_attention, "plain_calls", lambda: None)
    for a, b, c in zip(one_step, op, run("adapter"), strict=True):
        assert a.dtype == b.dtype == c.dtype and torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_one_step_calls_take_plain_calls_only(gpu):
    from vllm_rlt.kernels._extension import plain_calls

    layer, q, k, v, tables, lengths, cu, pages = _case(gpu, torch.bfloat16)
    m = plain_calls()
    cache = layer.args
    assert m.prefill_q8(q, *cache, tables, lengths, cu, 20) is not None
    assert m.decode_q8(q[:3], *cache, tables, lengths, 0) is not None
    assert m.append_q8(*cache, k, v, tables, lengths, cu) is True
    assert m.read_q8(*cache, pages, torch.float32) is not None
    rows = torch.arange(3, device=gpu)
    assert m.sequence_metadata(tables, rows, lengths, lengths, 16, 300, 8) is not None
    wide = torch.zeros((6,), dtype=torch.int32, device=gpu)
    assert m.decode_q8(q[:3], *cache, tables, wide[::2], 0) is None  # would need a copy
    assert m.decode_q8(q[:3], *cache, tables, lengths, -1) is None
    assert m.decode_q8(q, *cache, tables, lengths, 0) is None
    assert m.decode_q8(q[:3].double(), *cache, tables, lengths, 0) is None
    assert m.decode_q8(q[:3].cpu(), *cache, tables, lengths, 0) is None
    assert m.prefill_q8(q, *cache, tables, lengths, cu, 0) is None
    assert m.prefill_q8(q, *cache, tables, lengths, cu[:2], 20) is None
    assert m.append_q8(*cache, k, v[:5], tables, lengths, cu) is None
    assert m.append_q8(*cache, k, v, tables, lengths, None) is None
    assert m.append_q8(cache[0], cache[1][:1], cache[2], k, v, tables, lengths, cu) is None
    assert m.read_q8(*cache, pages, torch.float64) is None
    assert m.read_q8(*cache, pages.int(), torch.float32) is None
    assert m.sequence_metadata(tables, rows, lengths, lengths, 0, 300, 8) is None
    assert m.sequence_metadata(tables, rows[:2], lengths, lengths, 16, 300, 8) is None
    # What needs a copy goes through the adapter and gives the same.
    from vllm_rlt.kernels.hip_attention_q8 import paged_attention_q8

    wide[::2] = lengths
    assert torch.equal(paged_attention_q8(q[:3], *cache, tables, wide[::2]),
                       paged_attention_q8(q[:3], *cache, tables, lengths))


@pytest.mark.gpu
def test_ops_refuse(gpu):
    load_extension()
    ops = torch.ops.vllm_rlt_hip
    layer, q, k, v, tables, lengths, cu, pages = _case(gpu, torch.bfloat16)
    cache = layer.args
    raw = (cache[0].view(torch.uint8), cache[1].view(torch.uint8), cache[2])
    for call, message in (
            (lambda: ops.paged_attention_q8(q[:3], *raw, tables, lengths), "float8_e4m3fn"),
            (lambda: ops.paged_attention_q8(q, *cache, tables, lengths), "one row per query"),
            (lambda: ops.paged_attention_q8(q[:3], *cache, tables, lengths, -1), "window"),
            (lambda: ops.paged_attention_q8(q[:3, :3], *cache, tables, lengths), "multiple"),
            (lambda: ops.paged_prefill_q8(q, *cache, tables, lengths, cu[:2], 20), "one entry more"),
            (lambda: ops.paged_prefill_q8(q, *cache, tables, lengths, cu, 0), "positive"),
            (lambda: ops.kv_append_q8(*cache, k, v, tables, lengths), "one row per sequence"),
            (lambda: ops.kv_append_q8(*cache, k, v.float(), tables, lengths, cu), "same shape and dtype"),
            (lambda: ops.kv_read_q8(*cache, pages, torch.float64), "not Double"),
            (lambda: ops.kv_read_q8(*cache, pages.int(), torch.float32), "pages"),
            (lambda: ops.sequence_metadata(tables, lengths, lengths, lengths, 16, 1, 1), "table_rows"),
            (lambda: ops.sequence_metadata(tables, lengths.long(), lengths, lengths, 0, 1, 1), "page")):
        with pytest.raises(RuntimeError, match=message):
            call()
