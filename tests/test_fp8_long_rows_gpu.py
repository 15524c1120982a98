"""Rows of the 8-bit decode kernel that go on for hundreds of tiles of a warp: the running sums are not touched while the maximum stands still."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _one_slot(q, k, v, table, lens, block_size, scale):
    """paged_attention_fp8 with one slot to a row and a launch sized for very long sequences: a column's first CTA takes all of it."""
    from scicompute_attention_b200 import _lib, ops
    seqs, hq, _, d = q.shape
    hkv = k.codes.shape[2]
    out, part = torch.empty_like(q), torch.empty(seqs * hq * (2 + d) + 4, device="cuda")
    p = _lib.DecodeFwdParams()
    rows = seqs * hq
    p.q, p.k, p.v, p.out, p.page_table, p.seq_lens = q.data_ptr(), k.codes.data_ptr(), v.codes.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr()
    p.partial_m, p.partial_l, p.partial_o = part.data_ptr(), part.data_ptr() + 4 * rows, part.data_ptr() + 4 * (-(-2 * rows // 4) * 4)
    p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = seqs, hq, hkv, table.shape[1] * block_size, d, 1
    p.q_stride = p.o_stride = _lib.DecodeStrides(hq * d, d, d)
    p.scale, p.dtype, p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = scale, ops.dtype_id(q.dtype), block_size, table.shape[1], k.codes.shape[0]
    cluster = C.c_int32(-1)
    _lib.check(_lib.lib().sca_launch_paged_attention_fp8(C.byref(p), k.scales.data_ptr(), v.scales.data_ptr(), C.byref(cluster), None))
    assert cluster.value == 0
    return out


# score = size * scale, whose product with log2(e) in fp32 is off by nearly half a step of [32, 64): downwards, upwards
@pytest.mark.parametrize("d,size", [(64, 345.0), (64, 180.0), (128, 320.0), (128, 448.0), (256, 499.0), (256, 525.0)])
@pytest.mark.parametrize("clusters", [True, False])
def test_equal_keys_weigh_the_same(d, size, clusters):
    """Every key is the same, values are 1 and -1: behind a first maximum nothing moves, every sum is a whole number below 2^24, and the result is 0
    to the bit. With sums that every tile multiplies by 1 + 2^-20, 500 tiles leave 1e-4."""
    from scicompute_attention_b200 import ops
    bs, sharers = 64, 8 if clusters else 1
    each = 4 * 500 * (16 if d > 128 else 32)  # tokens of a CTA: 500 tiles to a warp
    n = each * sharers
    x, signs = torch.zeros(n, 1, d, dtype=torch.float16, device="cuda"), torch.ones(n, 1, d, dtype=torch.float16, device="cuda")
    x[:, :, 0] = 1
    signs.view(sharers, each, d)[:, each // 2:] = -1
    k, v = ops.fp8_pool(n // bs, bs, 1, d), ops.fp8_pool(n // bs, bs, 1, d)
    ops.kv_append_fp8(k, v, x, signs, torch.arange(n, dtype=torch.int32, device="cuda"))
    q = torch.zeros(1, 3, 1, d, dtype=torch.float16, device="cuda")
    q[..., 0] = size
    table, lens = torch.arange(n // bs, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda")
    if clusters:  # hints of a short call
        out, stats = ops.paged_attention_fp8(q, k, v, table, lens, block_size=bs, typical_len=1, longest_len=1, return_stats=True)
        assert stats["cluster"] == 8
    else:
        out = _one_slot(q, k, v, table, lens, bs, ops.effective_scale(None, d))
    assert not out.any(), out.abs().max()


def test_a_maximum_that_moves_carries_the_sums_along():
    """Scores that rise by a step every 128 tokens, against 64 bits: the sums follow the maximum without an error per tile."""
    from scicompute_attention_b200 import ops
    d, bs, steps = 64, 64, 240
    n = 128 * steps
    level = np.repeat(np.arange(steps), 128)
    rng = np.random.default_rng(3)
    x = np.zeros((n, 1, d), np.float32)
    x[:, 0, :8] = (level[:, None] >> (4 * np.arange(2))[None].repeat(4, 1).reshape(8)[None]) % 16  # whole numbers up to 15: exact in e4m3
    values = rng.choice([-1.0, -0.5, 0.5, 1.0], (n, 1, d)).astype(np.float32)
    k, v = ops.fp8_pool(n // bs, bs, 1, d), ops.fp8_pool(n // bs, bs, 1, d)
    ops.kv_append_fp8(k, v, torch.from_numpy(x).cuda(), torch.from_numpy(values).cuda(), torch.arange(n, dtype=torch.int32, device="cuda"))
    q = torch.zeros(1, 1, 1, d, dtype=torch.float16, device="cuda")
    q[..., 0], q[..., 4] = 0.37, 0.37 * 16
    table, lens = torch.arange(n // bs, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda")
    got = _one_slot(q, k, v, table, lens, bs, 0.125).double().cpu().numpy()[0, 0, 0]
    s = 0.125 * x[:, 0].astype(np.float64) @ q[0, 0, 0].double().cpu().numpy()
    w = np.exp(s - s.max())
    want = w @ values[:, 0] / w.sum()
    # P: 2^-11 of a weight, 2^-25 at least (of `n` keys); a shift off by 2^-24 of scores up to 2^7 in log2 units, twice; the output's 2^-11
    spread = w @ np.abs(values[:, 0]) / w.sum()
    bound = spread * (2.0 ** -11 + 2 * 2.0 ** -17 + 2.0 ** -20) + n * 2.0 ** -25 / w.sum() + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()
