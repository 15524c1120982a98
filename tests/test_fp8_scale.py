"""The scale of attention over the 8-bit cache: the C entry of a decode refuses what is not a positive number, the operators take None, 0 and below
as the default."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from scicompute_attention_b200 import _lib

BAD = [0.0, -0.0, -1.0, -1e-30, math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("scale", BAD)
def test_the_decode_entry_refuses_it(scale):
    at = 1 << 20  # an address that nothing reads: the call is refused on the host
    p = _lib.DecodeFwdParams()
    p.q = p.k = p.v = p.out = p.partial_m = p.partial_l = p.partial_o = p.page_table = at
    p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = 2, 4, 2, 100, 80, 2  # a head_dim without a kernel: nothing is launched
    p.q_stride = p.o_stride = _lib.DecodeStrides(320, 80, 80)
    p.scale, p.dtype, p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = scale, 2, 16, 4, 8
    assert _lib.lib().sca_launch_paged_attention_fp8(C.byref(p), at, at, None, None) == 4
    assert b"scale" in _lib.lib().sca_last_error()


@pytest.mark.gpu
def test_operators_take_the_default_for_it():
    from scicompute_attention_b200 import ops
    gen = torch.Generator("cuda").manual_seed(1)
    rows = torch.randn(20, 2, 64, device="cuda", generator=gen).half()
    k, v = ops.fp8_pool(2, 16, 2, 64), ops.fp8_pool(2, 16, 2, 64)
    ops.kv_append_fp8(k, v, rows, -rows, torch.arange(20, dtype=torch.int32, device="cuda"))
    table, lens = torch.arange(2, dtype=torch.int32, device="cuda")[None], torch.tensor([20], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 1, 64, device="cuda", generator=gen).half()
    for stream in (None, torch.cuda.current_stream()):
        step = lambda scale: ops.paged_attention_fp8(q, k, v, table, lens, block_size=16, scale=scale, stream=stream)
        chunk = lambda scale: ops.flash_attention_paged_fp8(q[:, :, 0], k, v, table, np.array([0, 1]), np.array([20]), scale=scale, stream=stream)
        for call in (step, chunk):
            want = call(None)
            assert all(torch.equal(call(s), want) for s in (0.0, -1.0, math.nan, 0.125))
            assert not torch.equal(call(0.5), want)
        with pytest.raises(_lib.ScaError):
            step(math.inf)
