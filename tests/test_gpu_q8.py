"""The 8-bit paged cache on the GPU against the float64 restatement in oracle/q8_ref.py."""

import numpy as np
import pytest
import torch

from oracle import q8_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# Half a step of each type, relative to the value.
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


class Layer:
    """One layer of a pool: bytes and scales on the GPU as views, and their numpy copies."""

    def __init__(self, device, blocks, bs, heads, dim, *, seed=0, order="head", offset=0, spread=3.0):
        rng = np.random.default_rng(seed)
        shape = {"head": (blocks, 2, heads, bs, dim), "token": (blocks, 2, bs, heads, dim)}[order]
        self.views = []
        self.bytes = []
        for _ in range(2):
            raw = rng.integers(0, 256, shape, dtype=np.uint8)
            raw[raw & 127 == 127] = 0x11
            store = torch.empty(raw.size + offset, dtype=torch.uint8, device=device)
            view = store[offset:].view(shape)
            view.copy_(torch.from_numpy(raw))
            view = view[:, 1]
            view = view.transpose(1, 2) if order == "head" else view
            self.views.append(view.view(torch.float8_e4m3fn))
            self.bytes.append(raw[:, 1].swapaxes(1, 2).copy() if order == "head" else raw[:, 1].copy())
        # Magnitudes of a few hundredths to tens; the largest byte is 448.
        exps = rng.integers(127 - 8 - int(spread), 127 - 8 + int(spread) + 1, (blocks, 2, heads, 2))
        self.scale_store = torch.from_numpy(exps.astype(np.uint8)).to(device)
        self.scales = self.scale_store[:, 1]
        self.exps = exps[:, 1].astype(np.uint8).copy()

    @property
    def args(self):
        return (*self.views, self.scales)

    def now(self):
        return [v.view(torch.uint8).cpu().numpy() for v in self.views], self.scales.cpu().numpy()

    def context(self, table, n):
        bs = self.bytes[0].shape[1]
        pages = np.asarray(table[: -(-n // bs)], np.int64)
        return [ref.values(b, self.exps, i, pages).reshape(-1, *b.shape[2:])[:n]
                for i, b in enumerate(self.bytes)]


def tables_of(rng, lengths, bs, width=0, extra=3):
    counts = [-(-max(0, n) // bs) for n in lengths]
    order = rng.permutation(sum(counts) + extra)
    tables = np.full((len(lengths), max([width, 1] + counts)), -1, np.int32)
    at = 0
    for r, c in enumerate(counts):
        tables[r, :c] = order[at : at + c]
        at += c
    return tables, sum(counts) + extra


def ints(x, device, dtype=torch.int32):
    return torch.tensor(np.asarray(x), dtype=dtype, device=device)


def to64(t):
    return t.double().cpu().numpy()


def check_attention(got, want, mean, reach, dtype, dim, n, weights=None):
    """Every score is off by at most (dim + 16) 2^-24 of sum |q k| (fp32 products, sums, the factor
    and the exponent's argument), a weight by that and by its rounding to ``weights`` (the query's
    type, or none), the sums of n weights by n 2^-24, and the output by its own rounding."""
    weights = HALF[weights or dtype]
    rel = weights + 2 * (dim + 16) * 2.0 ** -24 * (reach + 1) + 2 * (n + 64) * 2.0 ** -24
    least = 2.0 ** -24 if dtype == torch.float16 else 1e-30
    tol = mean * rel * 1.01 + np.abs(want) * HALF[dtype] * 1.01 + least
    bad = np.abs(to64(got) - want) > tol
    assert not bad.any(), (int(bad.sum()), float((np.abs(to64(got) - want) / tol).max()))


# ------------------------------------------------------------------- append
APPENDS = [
    # dtype, block, heads, dim, order, lengths after, new counts
    (torch.bfloat16, 16, 4, 128, "head", [1, 16, 17, 40, 100, 0, 33], [1, 16, 1, 30, 0, 0, 33]),
    (torch.bfloat16, 16, 2, 64, "token", [300, 5, 47], [200, 5, 2]),
    (torch.float16, 16, 3, 128, "head", [31, 64, 200], [15, 64, 17]),
    (torch.float32, 16, 2, 128, "head", [31, 64, 200], [15, 64, 17]),
    (torch.bfloat16, 64, 2, 128, "head", [130, 63, 64], [70, 1, 64]),
    (torch.bfloat16, 5, 3, 96, "token", [23, 4, 5, 6], [20, 4, 1, 2]),
    (torch.float16, 1, 2, 32, "head", [7, 1], [5, 1]),
    (torch.bfloat16, 16, 2, 20, "head", [18, 3], [18, 1]),
    (torch.float32, 3, 1, 1, "token", [7, 9], [6, 9]),
    (torch.bfloat16, 256, 1, 256, "head", [300, 255], [299, 1]),
]


@pytest.mark.parametrize("dtype,bs,heads,dim,order,lengths,counts", APPENDS)
def test_append_and_read_equal_the_oracle(gpu, dtype, bs, heads, dim, order, lengths, counts):
    from vllm_rlt.kernels.hip_attention_q8 import kv_append_q8, kv_read_q8

    rng = np.random.default_rng(1)
    tables, blocks = tables_of(rng, lengths, bs)
    layer = Layer(gpu, blocks, bs, heads, dim, order=order)
    cu = np.concatenate([[0], np.cumsum(counts)])
    gen = torch.Generator().manual_seed(2)
    rows = torch.randn((int(cu[-1]), 3, heads, dim), generator=gen)
    rows = (rows * torch.exp(4 * torch.rand((int(cu[-1]), 3, 1, 1), generator=gen) - 2)).to(dtype)
    rows[0, 0, 0, 0], rows[0, 1, 0, 0] = float("nan"), -float("inf")
    packed = rows.to(gpu)  # k and v are strided views of one projection
    kv_append_q8(*layer.args, packed[:, 0], packed[:, 1], ints(tables, gpu), ints(lengths, gpu),
                 ints(cu, gpu))
    for part in range(2):
        ref.append(layer.bytes[part], layer.exps, part, to64(rows[:, part]), tables, lengths, cu)
    got, scales = layer.now()
    assert np.array_equal(scales, layer.exps)
    for part in range(2):
        nan = lambda b: b & 127 == 127  # noqa: E731
        assert np.array_equal(nan(got[part]), nan(layer.bytes[part]))
        keep = ~nan(got[part])
        assert np.array_equal(got[part][keep], layer.bytes[part][keep])
    pages = rng.permutation(blocks)
    read = kv_read_q8(*layer.args, ints(pages, gpu, torch.int64), dtype)
    for part in range(2):
        want = torch.from_numpy(ref.values(layer.bytes[part], layer.exps, part, pages)).to(dtype)
        assert torch.equal(read[part].cpu().nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_token_by_token_appends_raise_scales(gpu, dtype):
    """A page filled one token at a time by growing values: its older tokens are rounded again."""
    from vllm_rlt.kernels.hip_attention_q8 import kv_append_q8

    rng = np.random.default_rng(5)
    bs, heads, dim = 16, 4, 128
    lengths = [20, 3, 0, 1]
    tables, blocks = tables_of(rng, [40, 40, 40, 40], bs)
    layer = Layer(gpu, blocks, bs, heads, dim)
    for step in range(18):
        rows = torch.randn((2, 4, heads, dim), generator=torch.Generator().manual_seed(step))
        rows = (rows * 2.0 ** (step / 2 - 6)).to(dtype)
        kv_append_q8(*layer.args, *rows.to(gpu), ints(tables, gpu), ints(lengths, gpu))
        for part in range(2):
            ref.append(layer.bytes[part], layer.exps, part, to64(rows[part]), tables, lengths)
        got, scales = layer.now()
        assert np.array_equal(scales, layer.exps), step
        assert all(np.array_equal(g, b) for g, b in zip(got, layer.bytes)), step
        lengths = [n + (i != 2) for i, n in enumerate(lengths)]


def test_append_extremes(gpu):
    """Zeros, the least and largest values, and values next to where the exponent changes."""
    from vllm_rlt.kernels.hip_attention_q8 import kv_append_q8

    tops = [0.0, 1e-45, 2.0 ** -100, 448.0, np.nextafter(np.float32(448), np.float32(500)), 447.99,
            3.4e38, 1.75 * 2.0 ** -60, 65504.0]
    rows = torch.zeros((len(tops), 1, 64))
    for i, t in enumerate(tops):
        rows[i, 0, :3] = torch.tensor([t, -t / 3, t / 7000], dtype=torch.float32)
    rows[-1, 0, 3] = float("inf")
    lengths = [1] * len(tops)
    tables = np.arange(len(tops), dtype=np.int32)[:, None]
    layer = Layer(gpu, len(tops), 16, 1, 64)
    kv_append_q8(*layer.args, rows.to(gpu), rows.to(gpu), ints(tables, gpu), ints(lengths, gpu))
    for part in range(2):
        ref.append(layer.bytes[part], layer.exps, part, to64(rows), tables, lengths)
    got, scales = layer.now()
    assert np.array_equal(scales, layer.exps)
    assert all(np.array_equal(g, b) for g, b in zip(got, layer.bytes))


def test_append_leaves_pages_that_are_not_the_pools(gpu):
    """Ids outside the pool, lengths past the table, counts past the length: nothing outside the
    sequence's own pages changes, and what has a place is written."""
    from vllm_rlt.kernels.hip_attention_q8 import kv_append_q8, kv_read_q8

    bs, blocks = 16, 6
    layer = Layer(gpu, blocks, bs, 2, 64)
    tables = np.array([[-1, 0], [1, blocks], [2, 3], [4, 5]], np.int32)
    lengths, counts = [20, 20, 40, 3], [20, 20, 20, 5]
    cu = np.concatenate([[0], np.cumsum(counts)])
    rows = torch.randn((cu[-1], 2, 64), generator=torch.Generator().manual_seed(0))
    kv_append_q8(*layer.args, rows.to(gpu), rows.to(gpu), ints(tables, gpu), ints(lengths, gpu),
                 ints(cu, gpu))
    for part in range(2):
        ref.append(layer.bytes[part], layer.exps, part, to64(rows), tables, lengths, cu)
    got, scales = layer.now()
    assert np.array_equal(scales, layer.exps)
    assert all(np.array_equal(g, b) for g, b in zip(got, layer.bytes))
    k, v = kv_read_q8(*layer.args, ints([-1, blocks, 2, -(1 << 40)], gpu, torch.int64))
    assert not k[[0, 1, 3]].any() and not v[[0, 1, 3]].any() and k[2].any()


# ------------------------------------------------------------------- decode
DECODES = [
    # dtype, q heads, kv heads, dim, block, order, window, lengths
    (torch.bfloat16, 16, 16, 128, 16, "head", 0, [1, 0, 15, 16, 17, 31, 33, 127, 128, 129, 300]),
    (torch.bfloat16, 4, 4, 128, 16, "token", 0, [2300, 777, 4100]),
    (torch.float16, 8, 8, 64, 16, "head", 0, [5, 4500, 129]),
    (torch.float32, 4, 4, 128, 16, "head", 0, [1, 64, 512, 0, 1500]),
    (torch.bfloat16, 32, 8, 128, 16, "head", 0, [1, 300, 1000]),
    (torch.float16, 32, 8, 128, 32, "head", 0, [19, 640, 257]),
    (torch.bfloat16, 16, 2, 64, 64, "token", 0, [63, 64, 65, 1030]),
    (torch.bfloat16, 16, 1, 128, 16, "head", 0, [100, 999]),
    (torch.bfloat16, 40, 2, 128, 16, "head", 0, [100, 300]),
    (torch.bfloat16, 12, 4, 128, 16, "head", 100, [1, 99, 100, 101, 116, 2000]),
    (torch.float16, 4, 4, 64, 16, "head", 1, [1, 16, 17, 200]),
    (torch.float32, 4, 2, 64, 16, "head", 300, [299, 301, 2000]),
    (torch.bfloat16, 4, 2, 96, 5, "token", 0, [1, 5, 6, 300]),
    (torch.float32, 2, 1, 20, 3, "head", 7, [1, 50]),
    (torch.float16, 2, 2, 256, 16, "head", 0, [40, 400]),
    (torch.bfloat16, 3, 1, 33, 1, "head", 0, [40, 1]),
    (torch.bfloat16, 2, 2, 128, 128, "head", 50, [1, 128, 129, 600]),
    (torch.bfloat16, 2, 1, 128, 24, "head", 0, [1, 24, 25, 500]),
    (torch.float32, 40, 2, 128, 16, "token", 100, [1, 100, 101, 700]),
    (torch.float32, 16, 16, 64, 64, "head", 0, [1, 0, 63, 65, 2500]),
    (torch.float32, 6, 3, 128, 24, "head", 0, [1, 24, 25, 500]),
]


@pytest.mark.parametrize("dtype,hq,hkv,dim,bs,order,window,lengths", DECODES)
def test_decode(gpu, dtype, hq, hkv, dim, bs, order, window, lengths):
    from vllm_rlt.kernels.hip_attention_q8 import paged_attention_q8

    rng = np.random.default_rng(3)
    tables, blocks = tables_of(rng, lengths, bs)
    layer = Layer(gpu, blocks, bs, hkv, dim, order=order)
    q = torch.randn((len(lengths), hq, dim), generator=torch.Generator().manual_seed(4)).to(dtype)
    got = paged_attention_q8(q.to(gpu), *layer.args, ints(tables, gpu), ints(lengths, gpu), window)
    assert got.dtype == dtype and got.shape == q.shape
    for r, n in enumerate(lengths):
        if n == 0:
            assert not got[r].any()
            continue
        want = ref.attend(to64(q[r : r + 1]), *layer.context(tables[r], n), n - 1, window)
        check_attention(got[r : r + 1], *want, dtype, dim, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 2)])
def test_decode_ignores_what_it_does_not_see(gpu, dtype, hq, hkv):
    """NaN bytes behind the last token and before the window, NaN scales of unused pages, -1 and
    wild page ids past a row's pages: the same bits as without them."""
    from vllm_rlt.kernels.hip_attention_q8 import paged_attention_q8

    rng = np.random.default_rng(3)
    bs, dim, window = 16, 128, 50
    lengths = [1, 77, 200, 130]
    tables, blocks = tables_of(rng, lengths, bs, width=20)
    layer = Layer(gpu, blocks, bs, hkv, dim)
    q = torch.randn((4, hq, dim), generator=torch.Generator().manual_seed(4)).to(dtype).to(gpu)
    call = lambda t: paged_attention_q8(q, *layer.args, ints(t, gpu), ints(lengths, gpu), window)  # noqa: E731
    clean = call(tables)
    used = set()
    for r, n in enumerate(lengths):
        pages = tables[r, : -(-n // bs)]
        first = max(0, n - window)
        used |= {int(p) for p in pages[first // bs :]}
        for view in layer.views:
            raw = view.view(torch.uint8)
            if n % bs:
                raw[int(pages[-1]), n % bs :] = 0x7F
            raw[int(pages[first // bs]), : first % bs] = 0xFF
            for p in pages[: first // bs]:
                raw[int(p)] = 0x7F
        tables[r, len(pages) :] = [(1 << 30, -5)[i % 2] for i in range(20 - len(pages))]
    for p in set(range(blocks)) - used:
        layer.scales[p] = 255
    assert torch.equal(call(tables), clean)
    assert clean.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_shows_nan_of_a_seen_token(gpu, dtype):
    """A NaN key or value of a visible token reaches its row and KV head, and no other."""
    from vllm_rlt.kernels.hip_attention_q8 import paged_attention_q8

    rng = np.random.default_rng(3)
    lengths = [40, 2, 300]
    tables, blocks = tables_of(rng, lengths, 16)
    for part in range(2):
        layer = Layer(gpu, blocks, 16, 2, 128)
        for r in (0, 1, 2):
            layer.views[part].view(torch.uint8)[int(tables[r, 0]), 1, 1, 5] = 0x7F
        q = torch.randn((3, 4, 128), generator=torch.Generator().manual_seed(4)).to(dtype).to(gpu)
        got = paged_attention_q8(q, *layer.args, ints(tables, gpu), ints(lengths, gpu))
        assert got[:, :2].isfinite().all()
        assert (got[:, 2:].isnan().all() if part == 0 else got[:, 2:, 5].isnan().all())


@pytest.mark.parametrize("dtype,hq,hkv,dim", [(torch.bfloat16, 16, 16, 128), (torch.float16, 32, 8, 64),
                                              (torch.float32, 4, 4, 128)])
def test_decode_rows_do_not_depend_on_the_batch(gpu, dtype, hq, hkv, dim):
    from vllm_rlt.kernels.hip_attention_q8 import paged_attention_q8

    rng = np.random.default_rng(3)
    lengths = [int(n) for n in rng.integers(1, 5000, 20)]
    tables, blocks = tables_of(rng, lengths, 16, width=400)
    layer = Layer(gpu, blocks, 16, hkv, dim)
    q = torch.randn((20, hq, dim), generator=torch.Generator().manual_seed(4)).to(dtype).to(gpu)
    batch = paged_attention_q8(q, *layer.args, ints(tables, gpu), ints(lengths, gpu))
    for r in range(0, 20, 3):
        width = -(-lengths[r] // 16)
        alone = paged_attention_q8(q[r : r + 1], *layer.args, ints(tables[r : r + 1, :width], gpu),
                                   ints(lengths[r : r + 1], gpu))
        assert torch.equal(alone[0], batch[r])


@pytest.mark.parametrize("rows,most,hq,hkv,dtype,dim", [
    (65, 900, 4, 4, torch.bfloat16, 64),  # more rows than a wave counts at once
    (200, 2600, 16, 16, torch.bfloat16, 128),  # more splits than waves: shares of several
    (512, 300, 16, 2, torch.float16, 64),
    (513, 300, 4, 1, torch.bfloat16, 128),  # beyond the rows that are counted
    (700, 200, 2, 2, torch.float32, 64),
])
def test_decode_of_many_rows(gpu, rows, most, hq, hkv, dtype, dim):
    from vllm_rlt.kernels.hip_attention_q8 import paged_attention_q8

    rng = np.random.default_rng(rows)
    lengths = [int(n) for n in rng.integers(0, most, rows)]
    lengths[0], lengths[rows // 2], lengths[-1] = most, 0, most - 1
    # Rows share pages: the pool needs no more than the longest.
    tables, blocks = tables_of(rng, [most] * 4, 16)
    tables = tables[rng.integers(0, 4, rows)]
    layer = Layer(gpu, blocks, 16, hkv, dim)
    q = torch.randn((rows, hq, dim), generator=torch.Generator().manual_seed(4)).to(dtype).to(gpu)
    got = paged_attention_q8(q, *layer.args, ints(tables, gpu), ints(lengths, gpu))
    for r in {0, 1, 63, 64, rows // 2, rows // 2 + 1, rows - 2, rows - 1}:
        alone = paged_attention_q8(q[r : r + 1], *layer.args, ints(tables[r : r + 1], gpu),
                                   ints(lengths[r : r + 1], gpu))
        assert torch.equal(alone[0], got[r]), r
    assert got.isfinite().all() and not got[rows // 2].any()
    for r in (0, rows - 1):
        want = ref.attend(to64(q[r : r + 1]), *layer.context(tables[r], lengths[r]), lengths[r] - 1)
        check_attention(got[r : r + 1], *want, dtype, dim, lengths[r])


@pytest.mark.parametrize("dtype,bs,n", [(torch.bfloat16, 16, 70001), (torch.float16, 32, 140000),
                                        (torch.float32, 16, 70001), (torch.bfloat16, 128, 9000)])
def test_decode_of_one_very_long_row(gpu, dtype, bs, n):
    """Splits of more pages than a wave keeps ids of."""
    from vllm_rlt.kernels.hip_attention_q8 import paged_attention_q8

    rng = np.random.default_rng(3)
    tables, blocks = tables_of(rng, [n], bs)
    layer = Layer(gpu, blocks, bs, 1, 64)
    q = torch.randn((1, 3, 64), generator=torch.Generator().manual_seed(4)).to(dtype)
    for window in (0, n - 5):
        got = paged_attention_q8(q.to(gpu), *layer.args, ints(tables, gpu), ints([n], gpu), window)
        want = ref.attend(to64(q), *layer.context(tables[0], n), n - 1, window)
        check_attention(got, *want, dtype, 64, n)


def test_decode_of_more_waves_than_a_launch_holds(gpu):
    """2200 rows x 512 heads x 64 split slots: the rows take several launches."""
    from vllm_rlt.kernels.hip_attention_q8 import paged_attention_q8

    rng = np.random.default_rng(3)
    tables, blocks = tables_of(rng, [40], 16, width=1024)
    layer = Layer(gpu, blocks, 16, 1, 4)
    lengths = rng.integers(0, 41, 2200)
    lengths[[0, -1]] = 40, 39
    q = torch.randn((2200, 512, 4), generator=torch.Generator().manual_seed(4)).to(gpu)
    got = paged_attention_q8(q, *layer.args, ints(tables, gpu).expand(2200, -1).contiguous(), ints(lengths, gpu))
    for r in (0, 1, 1000, 2046, 2047, 2048, 2199):
        n = int(lengths[r])
        if n == 0:
            assert not got[r].any()
            continue
        want = ref.attend(to64(q[r : r + 1]), *layer.context(tables[0], n), n - 1)
        check_attention(got[r : r + 1], *want, torch.float32, 4, n)


def test_append_and_read_of_more_pages_than_a_launch_holds(gpu):
    """Pages of one token and one value that has four significant bits: all are exact."""
    from vllm_rlt.kernels.hip_attention_q8 import kv_append_q8, kv_read_q8

    pages = (1 << 23) + 1000
    gen = torch.Generator(device=gpu).manual_seed(1)
    k, v = (torch.randint(8, 16, (pages, 1, 1), generator=gen, device=gpu) *
            2.0 ** torch.randint(-20, 20, (pages, 1, 1), generator=gen, device=gpu) for _ in range(2))
    k, v = k.bfloat16(), v.bfloat16()
    caches = [torch.zeros((pages, 1, 1, 1), dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)
              for _ in range(2)]
    scales = torch.zeros((pages, 1, 2), dtype=torch.uint8, device=gpu)
    tables = torch.randperm(pages, generator=gen, device=gpu).int()[None]
    kv_append_q8(*caches, scales, k, v, tables, ints([pages], gpu), ints([0, pages], gpu))
    got = kv_read_q8(*caches, scales, tables[0].long(), torch.bfloat16)
    assert torch.equal(got[0].view(-1), k.view(-1)) and torch.equal(got[1].view(-1), v.view(-1))


def test_decode_in_a_pool_past_32_bit_offsets(gpu):
    """Blocks more than 2^31 and 2^32 bytes into the cache."""
    from vllm_rlt.kernels.hip_attention_q8 import kv_append_q8, kv_read_q8, paged_attention_q8

    blocks = (5 << 30) // (16 * 2 * 128)
    caches = [torch.empty((blocks, 2, 16, 128), dtype=torch.uint8, device=gpu).transpose(1, 2)
              .view(torch.float8_e4m3fn) for _ in range(2)]
    scales = torch.full((blocks, 2, 2), 127, dtype=torch.uint8, device=gpu)
    tables = np.array([[blocks - 1, 2, blocks // 2 + 1]], np.int32)
    gen = torch.Generator().manual_seed(0)
    k, v = torch.randn((2, 45, 2, 128), generator=gen).bfloat16()
    kv_append_q8(*caches, scales, k.to(gpu), v.to(gpu), ints(tables, gpu), ints([45], gpu), ints([0, 45], gpu))
    raw = [np.zeros((3, 16, 2, 128), np.uint8) for _ in range(2)]
    exps = np.zeros((3, 2, 2), np.uint8)
    small = np.array([[0, 1, 2]], np.int32)
    for part, x in enumerate((k, v)):
        ref.append(raw[part], exps, part, to64(x), small, [45], [0, 45])
    read = kv_read_q8(*caches, scales, ints(tables[0], gpu, torch.int64), torch.float32)
    context = []
    for part in range(2):
        want = ref.values(raw[part], exps, part, np.arange(3)).reshape(48, 2, 128)[:45]
        assert np.array_equal(to64(read[part]).reshape(48, 2, 128)[:45], want)
        context.append(want)
    q = torch.randn((1, 4, 128), generator=gen).bfloat16()
    got = paged_attention_q8(q.to(gpu), *caches, scales, ints(tables, gpu), ints([45], gpu))
    check_attention(got, *ref.attend(to64(q), *context, 44), torch.bfloat16, 128, 45)


# ------------------------------------------------------------------ prefill
PREFILLS = [
    # dtype, q heads, kv heads, dim, block, order, lengths, counts
    (torch.bfloat16, 16, 16, 128, 16, "head", [40, 33, 1, 300], [40, 20, 1, 3]),
    (torch.float16, 4, 4, 64, 16, "token", [130, 257], [129, 1]),
    (torch.bfloat16, 8, 2, 128, 16, "head", [70, 500, 9, 0], [33, 65, 9, 0]),
    (torch.float16, 16, 2, 64, 32, "head", [300, 20, 700], [17, 20, 150]),
    (torch.bfloat16, 12, 4, 96, 16, "head", [50, 200], [50, 31]),
    (torch.float16, 4, 4, 32, 16, "head", [90], [61]),
    (torch.float32, 4, 2, 128, 16, "head", [30, 50], [20, 30]),
    (torch.bfloat16, 4, 2, 64, 5, "head", [30, 50], [20, 30]),
    (torch.bfloat16, 2, 2, 20, 16, "token", [30, 50], [20, 30]),
    (torch.bfloat16, 4, 4, 128, 16, "head", [5, 2, 900], [5, 2, 8]),
    (torch.bfloat16, 4, 4, 128, 16, "head", [1500], [200]),
    (torch.float16, 2, 2, 128, 64, "head", [1300, 64], [100, 64]),
    (torch.bfloat16, 2, 1, 128, 24, "head", [50, 100], [30, 60]),
]


@pytest.mark.parametrize("dtype,hq,hkv,dim,bs,order,lengths,counts", PREFILLS)
def test_prefill(gpu, dtype, hq, hkv, dim, bs, order, lengths, counts):
    from vllm_rlt.kernels.hip_attention_q8 import paged_prefill_attention_q8

    rng = np.random.default_rng(3)
    tables, blocks = tables_of(rng, lengths, bs)
    layer = Layer(gpu, blocks, bs, hkv, dim, order=order)
    cu = np.concatenate([[0], np.cumsum(counts)]) + 2  # rows before and behind the sequences
    total = int(cu[-1]) + 3
    q = torch.randn((total, hq, dim), generator=torch.Generator().manual_seed(4)).to(dtype)
    out = torch.full_like(q, 3.0).to(gpu)
    got = paged_prefill_attention_q8(q.to(gpu), *layer.args, ints(tables, gpu), ints(lengths, gpu),
                                     ints(cu, gpu), max(counts), out=out)
    assert got is out
    assert (got[:2] == 3).all() and (got[total - 3 :] == 3).all()
    for s, (n, c) in enumerate(zip(lengths, counts)):
        if c == 0:
            continue
        rows = slice(int(cu[s]), int(cu[s + 1]))
        want = ref.attend(to64(q[rows]), *layer.context(tables[s], n), n - c)
        check_attention(got[rows], *want, dtype, dim, n)


@pytest.mark.parametrize("dtype,dim,bs", [(torch.bfloat16, 128, 16), (torch.float16, 64, 16),
                                          (torch.float16, 128, 32), (torch.bfloat16, 96, 16)])
def test_prefill_of_more_pages_than_are_staged_at_once(gpu, dtype, dim, bs):
    """Pages and their scales are staged 512 at a time; with more than 64 sequences no tile is split,
    so that a tile's keys run past a first and a second such segment."""
    from vllm_rlt.kernels.hip_attention_q8 import paged_prefill_attention_q8

    rng = np.random.default_rng(8)
    lengths = [1040 * bs - 7, 521 * bs + 3] + [1] * 64
    counts = [70, 33] + [1] * 64
    tables, blocks = tables_of(rng, lengths, bs)
    layer = Layer(gpu, blocks, bs, 1, dim, seed=2)
    cu = np.concatenate([[0], np.cumsum(counts)])
    q = torch.randn((int(cu[-1]), 2, dim), generator=torch.Generator().manual_seed(4)).to(dtype)
    got = paged_prefill_attention_q8(q.to(gpu), *layer.args, ints(tables, gpu), ints(lengths, gpu),
                                     ints(cu, gpu), max(counts))
    for s, (n, c) in enumerate(zip(lengths, counts)):
        rows = slice(int(cu[s]), int(cu[s + 1]))
        want = ref.attend(to64(q[rows]), *layer.context(tables[s], n), n - c)
        check_attention(got[rows], *want, dtype, dim, n)


@pytest.mark.parametrize("dtype,hq,hkv,dim", [(torch.bfloat16, 16, 16, 128), (torch.float16, 32, 8, 64),
                                              (torch.float32, 4, 2, 64), (torch.bfloat16, 4, 4, 96)])
def test_short_packed_queries_equal_decode(gpu, dtype, hq, hkv, dim):
    from vllm_rlt.kernels.hip_attention_q8 import paged_attention_q8, paged_prefill_attention_q8

    rng = np.random.default_rng(3)
    lengths, counts = [5, 129, 700, 4200, 33], [5, 3, 1, 8, 0]
    tables, blocks = tables_of(rng, lengths, 16)
    layer = Layer(gpu, blocks, 16, hkv, dim)
    cu = np.concatenate([[0], np.cumsum(counts)])
    q = torch.randn((int(cu[-1]), hq, dim), generator=torch.Generator().manual_seed(4)).to(dtype).to(gpu)
    got = paged_prefill_attention_q8(q, *layer.args, ints(tables, gpu), ints(lengths, gpu), ints(cu, gpu), 8)
    rows = [(s, n - c + i + 1) for s, (n, c) in enumerate(zip(lengths, counts)) for i in range(c)]
    alone = paged_attention_q8(q, *layer.args, ints(tables[[s for s, _ in rows]], gpu), ints([n for _, n in rows], gpu))
    assert torch.equal(got, alone)


@pytest.mark.parametrize("dtype,hq,hkv,dim", [(torch.bfloat16, 4, 4, 128), (torch.float16, 8, 2, 64),
                                              (torch.float32, 2, 2, 64)])
def test_prefill_ignores_what_a_query_does_not_see(gpu, dtype, hq, hkv, dim):
    """NaN behind the last token, and NaN values of later tokens of the chunk: queries before them
    keep their bits, queries from them on are NaN in those dims."""
    from vllm_rlt.kernels.hip_attention_q8 import paged_prefill_attention_q8

    rng = np.random.default_rng(3)
    lengths, counts = [90, 300], [70, 44]
    tables, blocks = tables_of(rng, lengths, 16, width=30)
    layer = Layer(gpu, blocks, 16, hkv, dim)
    cu = np.concatenate([[0], np.cumsum(counts)])
    q = torch.randn((int(cu[-1]), hq, dim), generator=torch.Generator().manual_seed(4)).to(dtype).to(gpu)
    call = lambda: paged_prefill_attention_q8(  # noqa: E731
        q, *layer.args, ints(tables, gpu), ints(lengths, gpu), ints(cu, gpu), 70)
    clean = call()
    for s, n in enumerate(lengths):
        for view in layer.views:
            view.view(torch.uint8)[int(tables[s, (n - 1) // 16]), (n - 1) % 16 + 1 :] = 0x7F
    assert torch.equal(call(), clean)
    at = 55  # a token of sequence 0's chunk: queries 35.. see it
    layer.views[1].view(torch.uint8)[int(tables[0, at // 16]), at % 16, 0, 3] = 0x7F
    got = call()
    first = at - (lengths[0] - counts[0])
    group = hq // hkv
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[first : counts[0], :group, 3] = True
    assert got[hit].isnan().all()
    assert torch.equal(got[~hit], clean[~hit])
    layer.views[0].view(torch.uint8)[int(tables[1, 280 // 16]), 280 % 16, hkv - 1, 0] = 0x7F
    got = call()
    first = int(cu[1]) + 280 - (lengths[1] - counts[1])
    hit[first:, (hkv - 1) * group :] = True
    assert got[hit].isnan().all()
    assert torch.equal(got[~hit], clean[~hit])
