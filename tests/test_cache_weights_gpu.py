"""Decode with the weights of the cached tokens: output and weights against 64 bits."""
import numpy as np
import pytest
import torch

import cache_reference as ref
import helpers
import oracle_lib as ol

pytestmark = pytest.mark.gpu

DT = {torch.float16: ol.DT_F16, torch.bfloat16: ol.DT_BF16}


def _check(b, out, weights, before, own_from=None, scale=None):
    for s in range(len(b.lens_host)):
        want, p, at, size = ref.attend(b, b.q[s].transpose(0, 1), s, scale=scale)
        helpers.check_close(out[s, :, 0].float().cpu().numpy(), want[0].cpu().numpy(), DT[b.dtype], f"sequence {s}")
        added = torch.zeros_like(before[s], dtype=torch.float64)
        group = b.hq // b.hkv
        per_kv = p[0].view(b.hkv, group, -1).sum(1)
        start = 0 if own_from is None else int(own_from[s])
        keep = torch.from_numpy(at >= start).cuda()
        added[:, torch.from_numpy(at).cuda()[keep]] = per_kv[:, keep]
        ref.check_weights(weights[s], before[s], added, ref.weights_bound(b.d, len(at), group, size), f"sequence {s}")
        untouched = added == 0
        assert torch.equal(weights[s][untouched], before[s][untouched])


def _run(b, **more):
    from scicompute_attention_b200 import ops
    before = b.weights.clone()
    out = ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, b.weights, block_size=b.bs, **more)
    _check(b, out, b.weights, before, scale=more.get("scale"))
    return out


@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 64, torch.bfloat16), (8, 8, 128, torch.float16), (32, 2, 64, torch.float16), (6, 3, 96, torch.bfloat16),
                                            (16, 1, 256, torch.bfloat16), (5, 1, 32, torch.float16), (40, 1, 128, torch.bfloat16), (9, 1, 160, torch.float16),
                                            (4, 2, 192, torch.bfloat16)])
def test_heads_and_types(hq, hkv, d, dtype):
    _run(ref.Batch([1, 15, 16, 17, 63, 64, 65, 500, 1100], hq=hq, hkv=hkv, d=d, dtype=dtype))


@pytest.mark.parametrize("lens,bs", [([1], 16), ([0], 16), ([701], 16), ([7, 0, 900, 3], 1), ([130, 4000], 24), ([2500] * 3, 64), ([33] * 70, 8), ([12000], 32), ([1 + i % 60 for i in range(200)], 16)])
def test_lengths_and_pages(lens, bs):
    b = ref.Batch(lens, bs=bs)
    _run(b)
    _run(b, typical_len=max(1, sum(lens) // len(lens)), longest_len=max(1, max(lens)))  # weights that are there already


def test_unmapped_pages_weigh_nothing():
    b = ref.Batch([200, 64, 70], holes=[(0, 0), (0, 5), (1, 0), (1, 1), (1, 2), (1, 3)])
    b.table[2, 1] = b.blocks
    b.table_host[2, 1] = -1
    out = _run(b)
    assert (out[1] == 0).all()


def test_every_row_of_the_table_without_lengths():
    from scicompute_attention_b200 import ops
    b = ref.Batch([96, 96], extra_pages=0)
    before = b.weights.clone()
    out = ops.paged_attention_weights(b.q, b.k, b.v, b.table, None, b.weights, block_size=b.bs, scale=0.3)
    _check(b, out, b.weights, before, scale=0.3)


def test_same_output_and_the_same_bits_again():
    from scicompute_attention_b200 import ops
    b = ref.Batch([300, 2000, 5])
    first = b.weights.clone()
    out = ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, first, block_size=b.bs)
    for _ in range(3):
        w = b.weights.clone()
        assert torch.equal(out, ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, w, block_size=b.bs)) and torch.equal(w, first)


def test_large_scores():
    """Outputs of up to 20: helpers.check_close's absolute bound is for numbers of about 1, where half a step of bfloat16 is 2^-8."""
    from scicompute_attention_b200 import ops
    b = ref.Batch([300, 40], d=128, size=6.0)
    before = b.weights.clone()
    out = ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, b.weights, block_size=b.bs)
    for s in range(2):
        want, p, at, size = ref.attend(b, b.q[s].transpose(0, 1), s)
        bound = ref.weights_bound(b.d, len(at), 4, size)
        ref.check_output(out[s, :, 0], want[0], p[0], b.keys(s)[2], bound, 2.0 ** -15)  # P is two bfloat16 numbers: 2^-16 of it, twice
        added = torch.zeros_like(before[s], dtype=torch.float64)
        added[:, :len(at)] = p[0].view(2, 4, -1).sum(1)
        ref.check_weights(b.weights[s], before[s], added, bound)


def test_nan_queries_stay_in_their_rows():
    from scicompute_attention_b200 import ops
    b = ref.Batch([100, 300], hq=8, hkv=2)
    clean, before = b.weights.clone(), b.weights.clone()
    out = ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, clean, block_size=b.bs)
    b.q[1, 5] = float("nan")  # kv head 1
    got = ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, b.weights, block_size=b.bs)
    assert got[1, 5].isnan().all()
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[1, 5] = False
    assert torch.equal(got[rest], out[rest])
    assert b.weights[1, 1, :300].isnan().all() and torch.equal(b.weights[1, 1, 300:], before[1, 1, 300:])
    assert torch.equal(b.weights[0], clean[0]) and torch.equal(b.weights[1, 0], clean[1, 0])


def test_wider_weights():
    from scicompute_attention_b200 import ops
    b = ref.Batch([100, 300])
    for extra in (1, 2, 7):  # rows that do not start on 16 bytes
        wide = torch.full((5, 2, b.width * b.bs + extra), 3.0, device="cuda")
        wide[:2, :, :b.width * b.bs] = b.weights
        before = wide.clone()
        out = ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, wide, block_size=b.bs)
        _check(b, out, wide[:2, :, :b.width * b.bs], before[:2, :, :b.width * b.bs])
        assert (wide[2:] == 3).all() and (wide[:, :, b.width * b.bs:] == 3).all()


def test_bound_on_the_lengths():
    from scicompute_attention_b200 import ops
    b = ref.Batch([300, 90])
    short = torch.tensor([128, 90], dtype=torch.int32, device="cuda")
    w = b.weights.clone()
    want = ops.paged_attention_weights(b.q, b.k, b.v, b.table, short, w, block_size=b.bs)
    got = ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, b.weights, block_size=b.bs, longest_len=128)
    assert torch.allclose(want.float(), got.float(), atol=2e-2) and torch.equal(b.weights[:, :, 128:], w[:, :, 128:])


def test_captured_and_on_another_stream():
    from scicompute_attention_b200 import ops
    b = ref.Batch([100, 900, 30])
    w0 = b.weights.clone()
    run = lambda w, **more: ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, w, block_size=b.bs, **more)
    want = run(b.weights)
    w1, w2 = w0.clone(), w0.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = run(w1, stream=stream)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want) and torch.equal(w1, b.weights)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = run(w2)
    w3 = w0.clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(other):  # its scratch is its own
        got3 = run(w3)
    for _ in range(3):
        w2.copy_(w0)
        w3.copy_(w0)
        graph.replay()
        other.replay()
        assert torch.equal(got, want) and torch.equal(w2, b.weights) and torch.equal(got3, want) and torch.equal(w3, b.weights)
