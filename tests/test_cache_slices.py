"""Decode with weights whose scores are too many for the scratch runs in slices of sequences: the scratch stays bounded (on the CPU), and every sequence
is right whichever slice it is in (on the GPU)."""
import ctypes as C

import numpy as np
import pytest
import torch

from scicompute_attention_b200 import _lib

GB = 1 << 28  # floats


def _floats(batch, heads, kv_heads, d, width, groups=(), prefix=(), **more):
    p, x = _lib.DecodeFwdParams(), _lib.PagedStep()
    p.batch, p.num_heads, p.num_kv_heads, p.head_dim, p.scale, p.dtype = batch, heads, kv_heads, d, 0.1, _lib.DTYPE_BF16
    p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = 16, width // 16, 1 << 16
    x.weights, x.weights_row = 64, width
    lists = [np.array(v, np.int32) for v in (groups, prefix)]
    if len(prefix):
        x.cu_groups, x.prefix_lens, x.num_groups = lists[0].ctypes.data, lists[1].ctypes.data, len(prefix)
    for name, value in more.items():
        setattr(x, name, value)
    return _lib.lib().sca_paged_step_scratch_floats(C.byref(p), C.byref(x))


@pytest.mark.parametrize("batch,heads,kv_heads,d,width,more", [
    (192, 32, 8, 128, 131072, {}), (192, 32, 8, 128, 1 << 20, {}), (1000, 64, 8, 64, 1 << 20, {}), (192, 32, 8, 128, 1 << 20, dict(longest_len=100_000, typical_len=2000)),
    (128, 32, 8, 128, 131072, dict(groups=[0, 60, 128], prefix=[3000, 5000]))])
def test_scratch_is_bounded(batch, heads, kv_heads, d, width, more):
    # 64 slots and 32 parts of a prefix to a row at most, {m, l, O} each
    assert 0 < _floats(batch, heads, kv_heads, d, width, **more) <= 2 * GB + batch * heads * (64 + 32) * (d + 2) + 64


def test_one_sequence_is_the_least():
    assert _floats(3, 128, 1, 64, 1 << 23) >= 128 << 23
    assert _floats(3, 128, 1, 64, 1 << 23) < 2 * (128 << 23)


def test_what_fits_has_a_score_for_every_token():
    assert _floats(192, 32, 8, 128, 6016) >= 192 * 32 * 6016


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,dtype,n,slices", [(128, 1, 64, torch.bfloat16, 70, 3), (32, 8, 128, torch.float16, 130, 2), (40, 2, 96, torch.bfloat16, 110, 2)])
def test_weights_in_slices(hq, hkv, d, dtype, n, slices):
    import cache_reference as ref
    from launches import TWO, launches
    from scicompute_attention_b200 import ops
    from test_cache_weights_gpu import _check
    b = ref.Batch([(37 * i) % 300 + i % 2 for i in range(n)], hq=hq, hkv=hkv, d=d, dtype=dtype, extra_pages=8192 - 19)
    run = lambda w: ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, w, block_size=b.bs)
    assert launches(lambda: run(b.weights.clone())) == TWO * slices
    before, again = b.weights.clone(), b.weights.clone()
    out = run(b.weights)
    _check(b, out, b.weights, before)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = run(again)
    for _ in range(2):
        again.copy_(before)
        graph.replay()
        assert torch.equal(got, out) and torch.equal(again, b.weights)


@pytest.mark.gpu
def test_groups_that_slices_cut():
    """Slices end behind sequences 24 and 48: the first group leaves one sequence to the second slice, the fourth goes over into the last one."""
    import test_cache_shared_gpu as shared
    from launches import THREE, launches
    from scicompute_attention_b200 import ops
    b, cu, prefix = shared._batch([(25, 300), (1, 40), (10, 70), (30, 529), (4, 16)], [1, 30, 0, 200], hq=128, hkv=1, d=64, extra_pages=8192 - 46)
    run = lambda w: ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, cu, prefix, block_size=b.bs, weights=w)
    assert launches(lambda: run(b.weights.clone())) == THREE * 3
    shared._run(b, cu, prefix, True)
