"""What Fp8Pool and the header say about head dims and pages: attention over the 8-bit cache takes those and refuses the others, before any launch."""
import ctypes as C

import numpy as np
import pytest

from scicompute_attention_b200 import _lib, ops

ATTENDED = (32, 64, 96, 128, 160, 192, 256)
AT = 1 << 20  # an address that nothing reads: every call here is refused on the host


def _decode(d, block_size):
    p = _lib.DecodeFwdParams()
    p.q = p.k = p.v = p.out = p.partial_m = p.partial_l = p.partial_o = p.page_table = AT
    p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = 2, 4, 2, 100, d, 2
    p.q_stride = p.o_stride = _lib.DecodeStrides(4 * d, d, d)
    p.scale, p.dtype, p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = 0.1, 2, block_size, 4, 8
    return _lib.lib().sca_launch_paged_attention_fp8(C.byref(p), AT, AT, None, None)


def _chunk(d, block_size):
    p = _lib.FlashPagedParams()
    cu, lens = np.array([0, 9], np.int32), np.array([20], np.int32)
    p.q = p.out = p.k_pool = p.v_pool = p.page_table = p.workspace = AT
    p.total_q, p.num_heads, p.num_kv_heads, p.head_dim, p.num_seqs = 9, 4, 2, d, 1
    p.num_blocks, p.block_size, p.max_blocks_per_seq = 8, block_size, 20
    p.cu_seqlens_q, p.seq_lens_kv, p.scale, p.causal, p.dtype_id, p.workspace_bytes = cu.ctypes.data, lens.ctypes.data, 0.1, 1, 2, 4096
    return _lib.lib().sca_launch_flash_paged_fp8(C.byref(p), AT, AT, None)


@pytest.mark.parametrize("d", [d for d in range(16, 273, 16) if d not in ATTENDED])
def test_other_head_dims_are_for_storage(d):
    for call in (_decode, _chunk):
        assert call(d, 16) == 4
        assert b"head_dim" in _lib.lib().sca_last_error()


@pytest.mark.parametrize("d", ATTENDED)
def test_pages(d):
    for bs in (1, 2, 3, 6, 18, 63):
        assert _decode(d, bs) == 4 and b"block_size" in _lib.lib().sca_last_error()
    for bs in (1, 4, 12, 24, 48, 128):
        assert _chunk(d, bs) == 4 and b"block_size" in _lib.lib().sca_last_error()


def test_the_docstring_names_them():
    text = " ".join(ops.Fp8Pool.__doc__.split())
    assert "D = 32, 64, 96, 128, 160, 192 and 256" in text and "multiple of 4" in text and "8, 16, 32 or 64" in text
