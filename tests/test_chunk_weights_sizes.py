"""Sizes at which the weights of a chunk could go wrong: tables wider than any sequence (on the GPU), numbers of tiles that 32 bits do not hold (on the
CPU: they are refused before anything is launched)."""
import ctypes as C

import numpy as np
import pytest
import torch

from scicompute_attention_b200 import _lib


def _entry(**fields):
    raw = C.create_string_buffer(192)
    at = (C.addressof(raw) + 63) // 64 * 64
    p, w = _lib.FlashPagedParams(), _lib.ChunkWeights(at, at, 1 << 40, 0)
    cu, lens = np.array([0, 4], np.int32), np.array([fields.pop("tokens", 20)], np.int32)
    p.q = p.out = p.k_pool = p.v_pool = p.page_table = p.workspace = at
    p.total_q, p.num_heads, p.num_kv_heads, p.head_dim, p.num_seqs, p.num_blocks, p.block_size, p.max_blocks_per_seq = 4, 8, 2, 64, 1, 10, 16, 8
    p.cu_seqlens_q, p.seq_lens_kv, p.scale, p.causal, p.dtype_id, p.workspace_bytes = cu.ctypes.data, lens.ctypes.data, 0.1, 1, _lib.DTYPE_BF16, 1 << 20
    for name, value in fields.items():
        setattr(p, name, value)
    return _lib.lib().sca_launch_flash_paged_weights(C.byref(p), C.byref(w), None), _lib.lib().sca_last_error().decode()


@pytest.mark.parametrize("blocks", [1 << 27, 1 << 40, 1 << 60])
def test_rows_of_more_tokens_than_32_bits_hold_are_refused(blocks):
    rc, message = _entry(max_blocks_per_seq=blocks)
    assert rc == 4 and "2^31 tokens" in message, message


# 2^30 + 128 tiles; and 2^31 - 128, to which the number of CTAs cannot be added in 32 bits
@pytest.mark.parametrize("kv_heads,tokens", [(128, (1 << 30) + 128), (384, 5592405 * 128)])
def test_more_tiles_than_a_launch_has_are_refused_ahead_of_it(kv_heads, tokens):
    rc, message = _entry(num_heads=kv_heads, num_kv_heads=kv_heads, max_blocks_per_seq=(1 << 27) - 16, tokens=tokens)
    assert rc == 4 and "tiles of keys" in message, message


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [524281, 600_000])  # of 16 tokens: the first is the least that is wider than 65535 tiles of 128
def test_wide_tables(pages):
    import cache_reference as ref
    from scicompute_attention_b200 import ops
    b = ref.Batch([300, 1000], hq=4, hkv=1, stale=1.5)
    cu = np.array([0, 40, 300], np.int32)
    q = torch.randn((300, 4, 64), generator=b.gen, device="cuda").to(b.dtype)
    narrow = b.weights.clone()
    want = ops.flash_attention_paged_weights(q, b.k, b.v, b.table, cu, b.lens_host, narrow)
    table = torch.full((2, pages), -1, dtype=torch.int32, device="cuda")
    table[:, :b.width] = b.table
    wide = torch.zeros((2, 1, pages * 16), device="cuda")
    wide[:, :, :b.width * 16] = b.weights
    assert torch.equal(ops.flash_attention_paged_weights(q, b.k, b.v, table, cu, b.lens_host, wide), want)
    assert torch.equal(wide[:, :, :b.width * 16], narrow) and not wide[:, :, b.width * 16:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("n,longest,hkv,launched", [(3, 30_000, 2, 1), (160, 5000, 1, 1), (161, 5000, 2, 2), (400, 700, 1, 3)])
def test_ragged_batches(n, longest, hkv, launched):
    """One sequence far longer than the others, anywhere in the batch, equal ones, every number of tiles below that: only tiles that exist are dealt, those of
    up to 160 sequences to a launch."""
    import test_chunk_weights_gpu as chunks
    from launches import CHUNK, launches
    from scicompute_attention_b200 import ops
    lens = [1 + (113 * i) % 640 for i in range(n)]
    lens[n // 3] = longest
    new = [min(k, 1 + i % 5) for i, k in enumerate(lens)]
    b = chunks._batch(lens, hq=2 * hkv, hkv=hkv)
    q, cu = chunks._chunk(b, new)
    call = lambda: ops.flash_attention_paged_weights(q, b.k, b.v, b.table, cu, b.lens_host, b.weights.clone())
    assert launches(call)[-launched - 1:].count(CHUNK) == launched
    chunks._run(b, new)
    chunks._run(b, new, causal=False, last=2)
