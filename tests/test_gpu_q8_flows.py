"""The 8-bit cache as a serving step uses it: metadata from lengths on the GPU, append, attention;
captured graphs, other streams, refusals."""

import numpy as np
import pytest
import torch

from oracle import q8_ref as ref
from test_gpu_q8 import Layer, check_attention, ints, tables_of, to64

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------- metadata
def host_metadata(tables, rows, lengths, counts, page, tokens, out_width):
    """What sequence_metadata returns, in Python."""
    positions, blocks, offsets, out_tables, out_lengths, cu = [], [], [], [], [], [0]
    cap = min(tables.shape[1], out_width) * page
    for row, n, q in zip(rows, lengths, counts):
        n = max(0, n) if 0 <= row < tables.shape[0] else 0
        q = min(max(0, q), n)
        q, n = max(0, q - max(0, n - cap)), min(n, cap)
        keep = min(q, tokens - cu[-1])
        n -= q - keep
        mine = range(n - keep, n)
        positions += mine
        blocks += [int(tables[row, p // page]) for p in mine]
        offsets += [p % page for p in mine]
        used = -(-n // page)
        out_tables.append([int(x) for x in tables[row, :used]] + [-1] * (out_width - used) if used else [-1] * out_width)
        out_lengths.append(n)
        cu.append(cu[-1] + keep)
    pad = tokens - len(positions)
    return (positions + [0] * pad, blocks + [0] * pad, offsets + [0] * pad,
            [True] * len(positions) + [False] * pad, out_tables, out_lengths, cu)


METADATA = [
    # rows of the tables, width, out width, page, lengths, counts, spare tokens
    (4, 8, 8, 16, [1, 17, 0, 128], [1, 17, 0, 30], 0),
    (9, 8, 5, 16, [80, 128, 33, 5, 79], [3, 60, 33, 9, 1], 7),
    (3, 4, 9, 5, [20, 21, 60], [20, 2, 60], 0),
    (5, 16, 16, 1, [16, 3, -4], [2, -1, 5], 300),
    (2, 8, 8, 16, [128, 128], [128, 128], -150),
    (1, 1, 1, 16, [7], [7], 0),
]


@pytest.mark.parametrize("count,width,out_width,page,lengths,counts,spare", METADATA)
def test_sequence_metadata(gpu, count, width, out_width, page, lengths, counts, spare):
    from vllm_rlt.worker.metadata import sequence_kv_metadata

    rng = np.random.default_rng(1)
    tables = rng.integers(0, 1000, (count, width)).astype(np.int32)
    rows = [int(x) for x in rng.integers(0, count, len(lengths))]
    if count > 4:
        rows[1], rows[-1] = -1, count
    tokens = max(0, sum(max(0, min(q, n)) for q, n in zip(counts, lengths)) + spare)
    got = sequence_kv_metadata(ints(tables, gpu), ints(rows, gpu, torch.int64), ints(lengths, gpu),
                               ints(counts, gpu), block_size=page, tokens=tokens, width=out_width)
    want = host_metadata(tables, rows, lengths, counts, page, tokens, out_width)
    have = (got.position_ids, got.write_blocks, got.write_offsets, got.write_mask, got.block_tables,
            got.context_lengths, got.cu_seqlens_q)
    types = [torch.int64] * 3 + [torch.bool] + [torch.int32] * 3
    for h, w, t in zip(have, want, types):
        assert h.dtype == t and torch.equal(h.cpu(), torch.tensor(w, dtype=t).reshape(h.shape))


@pytest.mark.parametrize("n", [0, 1, 63, 65, 1023, 1024, 1025, 3000])
def test_sequence_metadata_of_many_requests(gpu, n):
    from vllm_rlt.worker.metadata import sequence_kv_metadata

    rng = np.random.default_rng(n)
    tables = rng.integers(0, 1 << 30, (2 * n + 1, 12)).astype(np.int32)
    rows = rng.permutation(2 * n + 1)[:n]
    lengths = rng.integers(0, 190, n)
    counts = np.where(rng.random(n) < 0.8, 1, rng.integers(0, 40, n))
    tokens = int(np.minimum(counts, lengths).sum()) + 5
    strided = torch.zeros((2 * n + 1, 20), dtype=torch.int32, device=gpu)
    strided[:, :12] = ints(tables, gpu)
    got = sequence_kv_metadata(strided[:, :12], ints(rows, gpu, torch.int64), ints(lengths, gpu),
                               ints(counts, gpu), block_size=16, tokens=tokens, width=14)
    want = host_metadata(tables, rows, [int(x) for x in lengths], [int(x) for x in counts], 16, tokens, 14)
    have = (got.position_ids, got.write_blocks, got.write_offsets, got.write_mask, got.block_tables,
            got.context_lengths, got.cu_seqlens_q)
    for h, w in zip(have, want):
        assert torch.equal(h.cpu(), torch.tensor(w, dtype=h.dtype).reshape(h.shape))


def test_sequence_metadata_equals_the_host_builder(gpu):
    from vllm_rlt.worker.metadata import build_kv_metadata, sequence_kv_metadata

    rng = np.random.default_rng(0)
    pages = rng.permutation(64).reshape(4, 16)
    work = [(0, 30, 12), (2, 100, 1), (3, 255, 40)]  # table row, length, new tokens
    positions = [p for _, n, q in work for p in range(n - q, n)]
    lists = [tuple(pages[r, : n // 16 + 1]) for r, n, q in work for _ in range(q)]
    keys = [(r, 0) for r, n, q in work for _ in range(q)]
    want = build_kv_metadata(lists, positions, block_size=16, device=gpu, sequence_keys=keys, packed=True)
    got = sequence_kv_metadata(ints(pages, gpu), ints([r for r, _, _ in work], gpu, torch.int64),
                               ints([n for _, n, _ in work], gpu), ints([q for _, _, q in work], gpu),
                               block_size=16, tokens=len(positions), width=16)
    for name in ("position_ids", "write_blocks", "write_offsets", "context_lengths", "cu_seqlens_q"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name
    assert torch.equal(got.block_tables[:, : want.block_tables.shape[1]], want.block_tables)


# -------------------------------------------------------------------- steps
class Program:
    """Requests whose lengths live on the GPU: one layer's step from metadata to attention."""

    def __init__(self, device, dtype, hq, hkv, dim, slots=5, width=24, bs=16):
        from vllm_rlt.core.paged_kv import QuantizedKVPool

        rng = np.random.default_rng(8)
        self.device, self.dtype, self.shape = device, dtype, (hq, hkv, dim)
        self.tables = rng.permutation(slots * width).reshape(slots, width).astype(np.int32)
        self.pool = QuantizedKVPool(slots * width, 2, bs, hkv, dim, device=device)
        self.d_tables = ints(self.tables, device)
        self.width, self.bs = width, bs

    def rows(self, tokens, seed):
        hq, hkv, dim = self.shape
        gen = torch.Generator().manual_seed(seed)
        return [torch.randn((tokens, h, dim), generator=gen).to(self.dtype) for h in (hq, hkv, hkv)]

    def step(self, slots, lengths, counts, q, k, v, max_q):
        from vllm_rlt.worker.metadata import sequence_kv_metadata

        m = sequence_kv_metadata(self.d_tables, slots, lengths, counts, block_size=self.bs,
                                 tokens=q.shape[0], width=self.width, max_seqlen_q=max_q)
        self.pool.append(1, k, v, m.block_tables, m.context_lengths, m.cu_seqlens_q)
        return self.pool.prefill(1, q, m.block_tables, m.context_lengths, m.cu_seqlens_q, max_q)


@pytest.mark.parametrize("dtype,hq,hkv,dim", [(torch.bfloat16, 4, 4, 128), (torch.float16, 8, 2, 64),
                                              (torch.float32, 2, 1, 64)])
def test_steps_of_growing_requests(gpu, dtype, hq, hkv, dim):
    """Chunks, then decode steps with a new chunk beside them, against the oracle's cache."""
    p = Program(gpu, dtype, hq, hkv, dim)
    blocks = p.tables.size
    raw = [np.zeros((blocks, p.bs, hkv, dim), np.uint8) for _ in range(2)]
    exps = np.zeros((blocks, hkv, 2), np.uint8)
    have = [0] * 5
    steps = [([0, 3], [40, 17]), ([3, 1, 0], [30, 20, 1]), ([0, 1, 3], [1, 1, 1]), ([4, 0, 1, 3], [100, 1, 1, 0]),
             ([4, 0, 1, 3], [1, 1, 1, 1])]
    for number, (slots, counts) in enumerate(steps):
        for s, c in zip(slots, counts):
            have[s] += c
        lengths = [have[s] for s in slots]
        q, k, v = p.rows(sum(counts) + 3, number)
        k *= 1.5 ** number
        got = p.step(ints(slots, gpu, torch.int64), ints(lengths, gpu), ints(counts, gpu),
                     q.to(gpu), k.to(gpu), v.to(gpu), max(counts))
        cu = np.concatenate([[0], np.cumsum(counts)])
        for part, x in enumerate((k, v)):
            ref.append(raw[part], exps, part, to64(x), p.tables[slots], lengths, cu)
        for i, (s, n, c) in enumerate(zip(slots, lengths, counts)):
            if not c:
                continue
            pages = p.tables[s, : -(-n // p.bs)]
            context = [ref.values(raw[j], exps, j, pages).reshape(-1, hkv, dim)[:n] for j in range(2)]
            rows = slice(int(cu[i]), int(cu[i + 1]))
            check_attention(got[rows], *ref.attend(to64(q[rows]), *context, n - c), dtype, dim, n)
    n = have[0]
    read = p.pool.read(1, p.tables[0], n, torch.float32)
    for part in range(2):
        want = ref.values(raw[part], exps, part, p.tables[0]).reshape(-1, hkv, dim)[:n]
        assert np.array_equal(to64(read[part]), want)


@pytest.mark.parametrize("dtype,hq,hkv,dim", [(torch.bfloat16, 4, 4, 128), (torch.float16, 8, 2, 64),
                                              (torch.float32, 2, 1, 64)])
@pytest.mark.parametrize("max_q", [1, 40])
def test_captured_step_replays(gpu, dtype, hq, hkv, dim, max_q):
    """A step captured once and replayed as the requests grow, next to a second captured step
    of another pool and the program's own eager work: each replay equals the eager step."""
    programs = [Program(gpu, dtype, hq, hkv, dim) for _ in range(2)]
    eager = Program(gpu, dtype, hq, hkv, dim)
    slots, start = [2, 0, 4], [33, 1, 100]
    tokens = 3 if max_q == 1 else 60
    counts = [1, 1, 1] if max_q == 1 else [max_q, 1, 13]
    static = []
    for p in programs:
        q, k, v = (x.to(gpu) for x in p.rows(tokens, 0))
        s = {"q": q, "k": k, "v": v, "slots": ints(slots, gpu, torch.int64), "lengths": ints(start, gpu),
             "counts": ints(counts, gpu)}
        args = lambda s=s: (s["slots"], s["lengths"], s["counts"], s["q"], s["k"], s["v"], max_q)  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            p.step(*args())
        torch.cuda.current_stream().wait_stream(side)
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            s["out"] = p.step(*args())
        for store in (p.pool.key_store, p.pool.value_store, p.pool.scales):
            store.zero_()
        static.append(s)
    lengths = list(start)
    for step in range(4):
        q, k, v = eager.rows(tokens, 10 + step)
        for s in static:
            for name, x in (("q", q), ("k", k), ("v", v), ("lengths", ints(lengths, "cpu"))):
                s[name].copy_(x)
        want = eager.step(ints(slots, gpu, torch.int64), ints(lengths, gpu), ints(counts, gpu), q.to(gpu),
                          k.to(gpu), v.to(gpu), max_q)
        used = sum(min(c, n) for c, n in zip(counts, lengths))  # counts are cut to the lengths
        for p, s in zip(programs, static):
            s["graph"].replay()
        torch.cuda.synchronize()
        for p, s in zip(programs, static):
            assert torch.equal(s["out"][:used], want[:used]), step
            assert torch.equal(p.pool.key_store, eager.pool.key_store)
            assert torch.equal(p.pool.scales, eager.pool.scales)
        lengths = [n + c for n, c in zip(lengths, counts)]


def test_calls_run_on_the_current_stream(gpu):
    """Inputs produced on a side stream, used there, with no synchronisation in between."""
    p = Program(gpu, torch.bfloat16, 4, 4, 128)
    q, k, v = (x.to(gpu) for x in p.rows(40, 0))
    slots, lengths, counts = ints([1], gpu, torch.int64), ints([40], gpu), ints([40], gpu)
    want = p.step(slots, lengths, counts, q, k, v, 40)
    other = Program(gpu, torch.bfloat16, 4, 4, 128)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        big = torch.randn((4096, 4096), device=gpu)
        for _ in range(10):
            big = big @ big * 1e-3
        late = k + 0 * big[:40, :512].reshape(40, 4, 128).nan_to_num(0.0).bfloat16()
        got = other.step(slots, lengths, counts, q, late, v, 40)
    stream.synchronize()
    assert torch.equal(got, want)


def test_pool_copies_blocks_with_their_scales(gpu):
    from vllm_rlt.core.paged_kv import QuantizedKVPool

    pool = QuantizedKVPool(8, 3, 16, 2, 64, device=gpu)
    rows = torch.randn((20, 2, 64), generator=torch.Generator().manual_seed(0)).bfloat16().to(gpu)
    tables = ints([[5, 2]], gpu)
    pool.append(1, rows, 2 * rows, tables, ints([20], gpu), ints([0, 20], gpu))
    want = pool.read(1, [5, 2], 20)
    pool.copy_blocks([5, 2], [0, 7])
    got = pool.read(1, [0, 7], 20)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and want[0].any()
    q = torch.randn((1, 4, 64), device=gpu).bfloat16()
    a = pool.attend(1, q, tables, ints([20], gpu))
    assert torch.equal(a, pool.attend(1, q, ints([[0, 7]], gpu), ints([20], gpu)))
    assert not torch.equal(a, pool.attend(1, q, tables, ints([20], gpu), window=5))
    with pytest.raises(ValueError, match="out of range"):
        pool.copy_blocks([1], [8])
    with pytest.raises(ValueError, match="disjoint"):
        pool.copy_blocks([1, 2], [2, 3])
    with pytest.raises(ValueError, match="layer"):
        pool.layer(3)
    with pytest.raises(ValueError, match="window"):
        pool.attend(1, q, tables, ints([20], gpu), window=0)


# ----------------------------------------------------------------- refusals
def test_refusals(gpu):
    from vllm_rlt.kernels.hip_attention import sequence_metadata
    from vllm_rlt.kernels.hip_attention_q8 import (
        kv_append_q8,
        kv_read_q8,
        paged_attention_q8,
        paged_prefill_attention_q8,
    )

    layer = Layer(gpu, 4, 16, 2, 64)
    k, v, scales = layer.args
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=gpu)
    rows = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device=gpu)
    tables, lengths, cu = ints([[0], [1]], gpu), ints([3, 4], gpu), ints([0, 1, 2], gpu)
    decode = lambda **kw: paged_attention_q8(**{  # noqa: E731
        "q": q, "key_cache": k, "value_cache": v, "scales": scales, "block_tables": tables,
        "context_lengths": lengths, **kw})
    prefill = lambda **kw: paged_prefill_attention_q8(**{  # noqa: E731
        "q": q, "key_cache": k, "value_cache": v, "scales": scales, "block_tables": tables,
        "context_lengths": lengths, "cu_seqlens_q": cu, "max_seqlen_q": 1, **kw})
    append = lambda **kw: kv_append_q8(**{  # noqa: E731
        "key_cache": k, "value_cache": v, "scales": scales, "k": rows, "v": rows,
        "block_tables": tables, "context_lengths": lengths, **kw})
    decode(), prefill(), append()
    both = (decode, prefill)
    cases = [
        (both, {"q": q.double()}, "float32, float16 and bfloat16"),
        (both, {"q": q[0]}, "rows, q_heads"),
        (both, {"q": q[:, :3]}, "multiple"),
        (both, {"q": q[..., :32]}, "head_dim"),
        (both, {"q": q.cpu()}, "ROCm"),
        (both, {"out": q[:1]}, "out must match"),
        (both, {"out": q.float()}, "out must match"),
        ((decode, prefill, append), {"key_cache": k.view(torch.uint8)}, "float8_e4m3fn"),
        ((decode, prefill, append), {"value_cache": v[:3]}, "same shape"),
        ((decode, prefill, append), {"value_cache": v.contiguous()}, "same shape and strides"),
        ((decode, prefill, append), {"scales": scales.int()}, "uint8"),
        ((decode, prefill, append), {"scales": scales[:, :1]}, "scales"),
        ((decode, prefill, append), {"scales": scales.cpu()}, "ROCm"),
        ((decode, prefill, append), {"block_tables": tables.long()}, "int32"),
        ((decode, prefill, append), {"block_tables": ints([[0, 1], [1, 0]], gpu).t()}, "contiguous"),
        ((decode, prefill, append), {"context_lengths": lengths[:1]}, "same rows"),
        ((decode,), {"block_tables": tables[:1], "context_lengths": lengths[:1]}, "one row per query"),
        ((decode,), {"window": -1}, "window"),
        ((decode,), {"window": True}, "window"),
        ((decode,), {"window": 1 << 31}, "window"),
        ((prefill, append), {"cu_seqlens_q": cu[:2]}, "one entry more"),
        ((prefill, append), {"cu_seqlens_q": cu.long()}, "int32"),
        ((prefill,), {"max_seqlen_q": 0}, "positive"),
        ((append,), {"k": rows.float()}, "same shape and dtype"),
        ((append,), {"k": rows[:1], "v": rows[:1]}, "one row per sequence"),
        ((append,), {"k": rows[:, :1]}, "k must be"),
        ((append,), {"v": rows.cpu()}, "ROCm"),
    ]
    for calls, kw, message in cases:
        for call in calls:
            with pytest.raises(ValueError, match=message):
                call(**kw)
    with pytest.raises(ValueError, match="int64"):
        kv_read_q8(k, v, scales, ints([0], gpu))
    with pytest.raises(ValueError, match="not torch.float64"):
        kv_read_q8(k, v, scales, ints([0], gpu, torch.int64), torch.float64)
    good = (tables, ints([0, 1], gpu, torch.int64), lengths, ints([1, 1], gpu), 16)
    sequence_metadata(*good, tokens=2, out_width=1)
    for at, bad, message in ((0, tables.long(), "int32"), (1, lengths, "int64"), (2, lengths[:1], "equal lengths"),
                             (4, 0, "page"), (4, (1 << 32) + 16, "32-bit")):
        with pytest.raises(ValueError, match=message):
            sequence_metadata(*[bad if i == at else x for i, x in enumerate(good)], tokens=2, out_width=1)
    with pytest.raises(ValueError, match="tokens"):
        sequence_metadata(*good, tokens=-1, out_width=1)


def test_empty_calls(gpu):
    from vllm_rlt.kernels.hip_attention_q8 import (
        kv_append_q8,
        kv_read_q8,
        paged_attention_q8,
        paged_prefill_attention_q8,
    )

    layer = Layer(gpu, 4, 16, 2, 64)
    q = torch.zeros((0, 4, 64), dtype=torch.bfloat16, device=gpu)
    none, tables = ints([], gpu), torch.zeros((0, 3), dtype=torch.int32, device=gpu)
    assert paged_attention_q8(q, *layer.args, tables, none).shape == (0, 4, 64)
    assert paged_prefill_attention_q8(q, *layer.args, tables, none, ints([0], gpu), 1).shape == (0, 4, 64)
    kv_append_q8(*layer.args, q[:, :2], q[:, :2], tables, none)
    assert kv_read_q8(*layer.args, none.long())[0].shape == (0, 16, 2, 64)
    # No table columns: every row is empty.
    q = torch.ones((2, 4, 64), dtype=torch.bfloat16, device=gpu)
    wide = torch.zeros((2, 0), dtype=torch.int32, device=gpu)
    assert not paged_attention_q8(q, *layer.args, wide, ints([5, 0], gpu)).any()
    before = layer.now()[0][0].copy()
    kv_append_q8(*layer.args, q[:, :2], q[:, :2], wide, ints([5, 1], gpu))
    assert np.array_equal(layer.now()[0][0], before)
