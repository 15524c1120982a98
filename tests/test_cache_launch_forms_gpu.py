"""The forms that a rule chooses among, at sizes that reach them, and proof that it was this form that ran: decode over shared prefixes in three kernels (prefix
kernel, own tokens beside it, finish kernel), decode with weights in two, chunks whose CTAs take more than one tile of keys."""
import threading

import numpy as np
import pytest
import torch

import cache_reference as ref
import test_cache_shared_gpu as shared
import test_cache_weights_gpu as weighed
import test_chunk_weights_gpu as chunks
from launches import CHUNK, THREE, TWO, launches

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _long(d):
    """A prefix of which a CTA of a cluster of 8 would have more steps of 64 tokens than the one-launch form is taken for: 20, 12, 2."""
    return 10500 if d <= 64 else 6500 if d <= 128 else 1100


def _call(b, cu, prefix, weights=True):
    from scicompute_attention_b200 import ops
    return lambda w=None, **more: ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, np.array(cu, np.int32), np.array(prefix, np.int32), block_size=b.bs,
                                                             weights=(b.weights.clone() if w is None else w) if weights else None, **more)


def _three(b, cu, prefix, weights=True):
    assert launches(_call(b, cu, prefix, weights)) == THREE
    return shared._run(b, cu, prefix, weights)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("hq,hkv,d", [(5, 1, 32), (32, 2, 32), (8, 2, 64), (32, 2, 64), (6, 3, 96), (24, 1, 96), (8, 8, 128), (16, 4, 128), (32, 2, 128), (12, 1, 128), (4, 2, 160),
                                      (8, 2, 192), (16, 1, 256), (6, 2, 256)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_three_kernels(dtype, hq, hkv, d, weights):
    _three(*shared._batch([(3, _long(d)), (1, 100), (9, 1000), (2, 16)], [1, 2, 40, 130, 16], hq=hq, hkv=hkv, d=d, dtype=dtype), weights)


@pytest.mark.parametrize("d,dtype", [(64, HF), (96, BF), (128, BF), (128, HF), (256, BF)])
def test_three_kernels_over_sequences_shorter_than_their_prefix(d, dtype):
    b, cu, prefix = shared._batch([(6, _long(d)), (4, 64)], [20, 3], stale=None, d=d, dtype=dtype)
    b.lens_host[[1, 2, 4, 7]] = [200, 0, _long(d) // 16 * 16 - 1, 1]
    b.lens = torch.from_numpy(b.lens_host).cuda()
    out = _three(b, cu, prefix)
    assert (out[2] == 0).all()


@pytest.mark.parametrize("d,dtype", [(64, BF), (128, BF), (128, HF), (192, HF)])
def test_three_kernels_over_unmapped_pages(d, dtype):
    """Holes in a prefix, a group without a page, a hole in a sequence's own tokens, and a sequence that has nothing at all."""
    n = _long(d)
    b, cu, prefix = shared._batch([(5, n), (3, 48), (2, 32)], [20, 100, 0], holes=[(i, j) for i in range(5) for j in (0, 3, 17, 18, 19)] + [(1, n // 16 + 1)] +
                                  [(i, j) for i in (5, 6, 7) for j in range(3)] + [(i, j) for i in (8, 9) for j in range(2)], d=d, dtype=dtype)
    out = _three(b, cu, prefix)
    assert b.lens_host[8] == 32 and (out[8] == 0).all()


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF), (128, HF), (256, HF)])
def test_three_kernels_where_all_end_with_the_prefix(d, dtype):
    _three(*shared._batch([(6, _long(d) // 16 * 16)], [0], d=d, dtype=dtype))


@pytest.mark.parametrize("bs,tail", [(8, 8), (16, 120), (32, 96), (64, 64)])
def test_three_kernels_over_every_page(bs, tail):
    _three(*shared._batch([(4, 6500 // 64 * 64 + tail), (37, 128 - bs + 1)], [30, 5], bs=bs, d=128))


def test_three_kernels_without_lengths():
    b, cu, prefix = shared._batch([(5, 6400)], [160], d=128, extra_pages=0)
    before, lens = b.weights.clone(), b.lens
    out = _three(b, cu, prefix)
    b.lens = None  # all of every row
    again = before.clone()
    assert launches(_call(b, cu, prefix)) == THREE
    assert torch.equal(_call(b, cu, prefix)(again), out) and torch.equal(again, b.weights) and (lens == b.width * b.bs).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_three_kernels_captured_and_on_another_stream(dtype):
    b, cu, prefix = shared._batch([(3, 6500), (40, 300)], [20, 200], hq=8, hkv=8, d=128, dtype=dtype)
    run = _call(b, cu, prefix)
    assert launches(run) == THREE
    w0 = b.weights.clone()
    want = run(b.weights)
    w = [w0.clone() for _ in range(3)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = run(w[0], stream=stream)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want) and torch.equal(w[0], b.weights)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, mine in zip(graphs, w[1:]):  # each with scratch of its own
        with torch.cuda.graph(graph):
            outs.append(run(mine))
    for _ in range(3):
        for mine in w[1:]:
            mine.copy_(w0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[1].replay()
        graphs[0].replay()
        eager = run(w[0].copy_(w0))
        torch.cuda.synchronize()
        for got, mine in zip([eager, *outs], w):
            assert torch.equal(got, want) and torch.equal(mine, b.weights)


def test_three_kernels_back_to_back():
    """Calls of different sizes that use the same scratch, and one-launch calls between them."""
    batches = [shared._batch([(30, 2000), (20, 500)], [5, 300], hq=8, hkv=8, d=128, seed=1), shared._batch([(7, 900), (90, 700)], [40], hq=16, hkv=4, d=128, dtype=HF, seed=2),
               shared._batch([(3, 400)], [40], seed=3)]
    calls = [_call(*x) for x in batches]
    assert [len(launches(call)) for call in calls] == [3, 3, 1]
    weights = [x[0].weights for x in batches]
    want = [(call(w := weights[i].clone()), w) for i, call in enumerate(calls)]
    torch.cuda.synchronize()
    got = []
    for i in range(45):
        w = weights[i % 3].clone()
        got.append((calls[i % 3](w), w))
    for i, (out, w) in enumerate(got):
        assert torch.equal(out, want[i % 3][0]) and torch.equal(w, want[i % 3][1])


def test_three_kernels_from_two_threads():
    batches = [shared._batch([(30, 2000)], [5 + i, 300], hq=8, hkv=8, d=128, seed=i) for i in range(2)]
    want = [_call(*x)() for x in batches]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(15):
                got = _call(*batches[i])()
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[i]):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("group", [1, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 256])
def test_weights_in_two_kernels(d, group):
    """More (sequence, kv head) than clusters of two have room for."""
    from scicompute_attention_b200 import ops
    b = ref.Batch([(83 * i) % 700 + 1 if i % 9 else 0 for i in range(90)], hq=8 * group, hkv=8, d=d, dtype=HF if (d // 32 + group) % 2 else BF, holes=[(4, 0), (7, 2), (7, 3)])
    call = lambda: ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, b.weights.clone(), block_size=b.bs)
    assert launches(call) == TWO
    weighed._run(b)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,hq", [(64, 8), (128, 4), (128, 12), (192, 8), (256, 16)])
def test_several_tiles_of_keys_to_a_cta(d, hq, dtype, causal):
    """332 tiles for 148 CTAs: every CTA takes a second one - at D above 128 into the slot of the first - and some a third."""
    from scicompute_attention_b200 import ops
    b = chunks._batch([3000, 2500, 700, 4000, 100], hq=hq, hkv=4, d=d, dtype=dtype)
    new = [40, 600, 700, 1, 13]
    q, cu = chunks._chunk(b, new)
    call = lambda: ops.flash_attention_paged_weights(q, b.k, b.v, b.table, cu, b.lens_host, b.weights.clone(), causal=causal)
    assert launches(call)[-1] == CHUNK
    chunks._run(b, new, causal)
    chunks._run(b, new, causal, last=9)
