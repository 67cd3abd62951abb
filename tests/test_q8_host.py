"""The 8-bit cache without a GPU: the oracle's format, the append's page slots, refusals."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import q8_ref as ref


def test_oracle_bytes_are_torchs():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(every, ref.E4M3, equal_nan=True)
    x = torch.randn(20000, generator=torch.Generator().manual_seed(0)) * 60
    x = torch.cat([x, x * 1e-4, torch.tensor([0.0, -0.0, 448, 464, 2.0 ** -10, 3 * 2.0 ** -10])])
    mids = torch.tensor((ref.E4M3[:126] + ref.E4M3[1:127]) / 2, dtype=torch.float32)
    x = torch.cat([x, mids, -mids])
    assert np.array_equal(ref.encode(x.double().numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert (ref.encode([np.nan, np.inf, -np.inf, 465.0]) & 127 == 127).all()


def test_every_touched_page_has_a_slot_of_its_sequence():
    """The append's work items: slot j belongs to the last s with cu[s] // bs + 2 s <= j, and the
    slots of s are at least as many as the pages its tokens can touch, for any offset."""
    rng = np.random.default_rng(0)
    for bs in (1, 2, 5, 16, 64):
        for _ in range(50):
            counts = rng.integers(0, 3 * bs + 2, rng.integers(1, 90))
            cu = np.concatenate([[rng.integers(0, 5)], counts]).cumsum()
            base = cu[:-1] // bs + 2 * np.arange(len(counts))
            room = np.diff(np.append(base, cu[-1] // bs + 2 * len(counts)))
            pages = np.where(counts > 0, (bs - 1 + counts - 1) // bs + 1, 0)
            assert (room >= pages).all()
            for slot in range(int(cu[-1]) // bs + 2 * len(counts)):
                # The search of 64 candidates at a time.
                lo, hi, found = 0, len(counts), True
                while True:
                    step = (hi - lo + 63) // 64
                    at = [lo + i * step < hi and base[lo + i * step] <= slot for i in range(64)]
                    if not any(at):
                        found = False
                        break
                    lo += max(i for i in range(64) if at[i]) * step
                    if step == 1:
                        break
                    hi = min(hi, lo + step)
                want = [s for s in range(len(counts)) if base[s] <= slot]
                if found and slot >= base[lo]:
                    assert lo == want[-1]
                else:
                    assert not want


def test_adapter_refuses_host_tensors():
    from vllm_rlt.kernels.hip_attention import sequence_metadata
    from vllm_rlt.kernels.hip_attention_q8 import kv_append_q8, kv_read_q8, paged_attention_q8

    cache = torch.zeros((2, 16, 2, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.zeros((2, 2, 2), dtype=torch.uint8)
    rows = torch.zeros((1, 2, 64))
    tables, lengths = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm"):
        kv_append_q8(cache, cache, scales, rows, rows, tables, lengths)
    with pytest.raises(ValueError, match="ROCm"):
        kv_read_q8(cache, cache, scales, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="ROCm"):
        paged_attention_q8(rows, cache, cache, scales, tables, lengths)
    with pytest.raises(ValueError, match="ROCm"):
        sequence_metadata(tables, lengths.long(), lengths, lengths, 16, tokens=1, out_width=1)


def test_entry_points_refuse_before_any_launch():
    """Bad sizes, types and missing pointers and workspaces are errors of the host code."""
    from vllm_rlt.kernels._hip import library

    lib = library()
    p = ctypes.c_void_p(256)  # never dereferenced on the host

    def decode(dtype=2, out=p, rows=2, heads=4, kv=2, dim=64, blocks=8, bs=16, width=64, window=0, ws=p, nbytes=1 << 30):
        return lib.vrh_paged_decode_q8(dtype, out, p, p, p, p, p, p, rows, heads, kv, dim, blocks, bs, width, width,
                                       heads * dim, dim, heads * dim, dim, 1, 1, 1, 1, 1, window, ws, nbytes, None)

    for bad in ({"dtype": 7}, {"out": None}, {"rows": -1}, {"heads": 3}, {"heads": 0}, {"dim": 0}, {"dim": 257},
                {"blocks": 0}, {"bs": 0}, {"width": -1}, {"window": -1}, {"ws": None}, {"nbytes": 100}):
        assert decode(**bad) == 1, bad
        assert lib.vrh_last_error().startswith(b"vrh_paged_decode_q8")
    assert decode(rows=0) == 0

    def prefill(dtype=2, cu=p, seqs=2, total=40, most=20, heads=4, kv=2, dim=64, bs=16, ws=p, nbytes=1 << 32):
        return lib.vrh_paged_prefill_q8(dtype, p, p, p, p, p, p, p, cu, seqs, total, most, heads, kv, dim, 8, bs, 64, 64,
                                        heads * dim, dim, heads * dim, dim, 1, 1, 1, 1, 1, ws, nbytes, None)

    for bad in ({"dtype": 7}, {"cu": None}, {"seqs": -1}, {"total": -1}, {"most": -1}, {"most": 0}, {"heads": 3}, {"dim": 300},
                {"bs": 0}, {"most": 2, "nbytes": 100}, {"most": 2, "ws": None}, {"seqs": 1 << 40}):
        assert prefill(**bad) == 1, bad
        assert lib.vrh_last_error().startswith(b"vrh_paged_prefill_q8")
    assert prefill(seqs=0) == 0 and prefill(total=0) == 0

    def append(dtype=2, k=p, cu=p, seqs=2, total=40, heads=2, dim=64, blocks=8, bs=16, width=4):
        return lib.vrh_kv_append_q8(dtype, p, p, p, 1, 1, 1, 1, 1, k, p, 1, 1, 1, 1, p, p, cu, seqs, total, heads, dim, blocks,
                                    bs, width, width, None)

    for bad in ({"dtype": 7}, {"k": None}, {"cu": None}, {"seqs": -1}, {"total": -1}, {"heads": 0}, {"dim": 0}, {"bs": 0},
                {"width": -1}, {"bs": 1 << 30}):
        assert append(**bad) == 1, bad
        assert lib.vrh_last_error().startswith(b"vrh_kv_append_q8")
    assert append(seqs=0, total=0) == 0 and append(width=0) == 0 and append(blocks=0) == 0

    def read(dtype=2, out=p, pages=2, heads=2, dim=64, bs=16):
        return lib.vrh_kv_read_q8(dtype, out, p, p, p, p, 1, 1, 1, 1, 1, p, pages, heads, dim, 8, bs, None)

    for bad in ({"dtype": 7}, {"out": None}, {"pages": -1}, {"heads": 0}, {"dim": 0}, {"bs": 0}):
        assert read(**bad) == 1, bad
        assert lib.vrh_last_error().startswith(b"vrh_kv_read_q8")
    assert read(pages=0) == 0

    def metadata(cu=p, positions=p, rows=p, n=2, tokens=4, width=4, out_width=4, stride=4, page=16):
        return lib.vrh_sequence_metadata(p, 3, 4, rows, p, p, positions, p, p, p, p, stride, p, cu, n, tokens, width, out_width,
                                         page, None)

    for bad in ({"cu": None}, {"positions": None}, {"rows": None}, {"n": -1}, {"tokens": -1}, {"tokens": 1 << 31}, {"width": -1},
                {"out_width": -1}, {"stride": 3}, {"page": 0}):
        assert metadata(**bad) == 1, bad
        assert lib.vrh_last_error().startswith(b"vrh_sequence_metadata")


def test_workspaces_follow_the_shapes():
    from vllm_rlt.kernels._hip import library

    lib = library()
    size = lib.vrh_paged_decode_q8_workspace_bytes
    assert size(4, 16, 128, 16, 8, 0) == 0  # one split of 128 tokens: written by its wave
    assert size(0, 16, 128, 16, 800, 0) == 0
    assert 0 < size(4, 16, 128, 16, 800, 512) < size(4, 16, 128, 16, 800, 0)
    assert size(4, 16, 128, 16, 2000, 0) == size(4, 16, 128, 16, 8000, 0)  # splits are bounded
    assert size(8, 16, 128, 16, 800, 0) == 2 * size(4, 16, 128, 16, 800, 0)
