"""Decode over prefixes that sequences share: the output of every sequence against 64 bits, and the weights of its own tokens."""
import numpy as np
import pytest
import torch

import cache_reference as ref
import helpers
import oracle_lib as ol
from test_cache_weights_gpu import _check

pytestmark = pytest.mark.gpu


def _run(b, cu, prefix, weights=False, **more):
    from scicompute_attention_b200 import ops
    before = b.weights.clone()
    out = ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, np.array(cu, np.int32), np.array(prefix, np.int32), block_size=b.bs,
                                     weights=b.weights if weights else None, **more)
    own_from = np.zeros(len(b.lens_host), np.int64)
    for first, end, tokens in zip(cu, cu[1:], prefix):
        if end - first > 1:
            own_from[first:end] = tokens // b.bs * b.bs
    if weights:
        _check(b, out, b.weights, before, own_from)
    else:
        assert torch.equal(b.weights, before)
        dt = {torch.float16: ol.DT_F16, torch.bfloat16: ol.DT_BF16}[b.dtype]
        for s in range(len(b.lens_host)):
            want = ref.attend(b, b.q[s].transpose(0, 1), s)[0]
            helpers.check_close(out[s, :, 0].float().cpu().numpy(), want[0].cpu().numpy(), dt, f"sequence {s}")
    return out


def _batch(groups, own, **more):
    """groups: (sequences, prefix tokens); own: tokens behind the prefix, dealt in turn."""
    lens, prefixes, cu = [], [], [0]
    for n, tokens in groups:
        prefixes.append((cu[-1], cu[-1] + n, tokens))
        lens += [tokens + own[(cu[-1] + i) % len(own)] for i in range(n)]
        cu.append(cu[-1] + n)
    return ref.Batch(lens, prefixes=prefixes, **more), cu, [tokens for _, tokens in groups]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 64, torch.bfloat16), (8, 8, 128, torch.float16), (32, 2, 128, torch.bfloat16), (6, 3, 96, torch.float16),
                                            (16, 1, 256, torch.bfloat16), (5, 1, 32, torch.float16), (24, 1, 64, torch.float16), (4, 2, 160, torch.float16),
                                            (8, 2, 192, torch.bfloat16)])
def test_heads_and_types(hq, hkv, d, dtype, weights):
    _run(*_batch([(3, 400), (1, 100), (9, 1000), (2, 16)], [1, 2, 40, 130, 16], hq=hq, hkv=hkv, d=d, dtype=dtype), weights)


@pytest.mark.parametrize("groups,own,bs", [
    ([(2, 16)], [1], 16), ([(5, 501)], [1, 100, 200], 16), ([(40, 128)], [3], 16), ([(70, 129)], [30, 5], 8), ([(3, 4000)], [64, 1], 64),
    ([(300, 64)], [1, 2, 3], 32), ([(1, 500), (1, 30)], [7], 16), ([(4, 15), (4, 0)], [20], 16), ([(2, 10000), (33, 32)], [9, 0], 16),
    ([(2, 48)] * 20, [5, 17], 16), ([(130, 2000)], [10], 16)])
def test_groups_and_pages(groups, own, bs):
    b, cu, prefix = _batch(groups, own, bs=bs)
    _run(b, cu, prefix)
    _run(b, cu, prefix, True, typical_len=int(b.lens_host.mean()), longest_len=int(b.lens_host.max()))


def test_as_many_groups_as_a_call_takes():
    b, cu, prefix = _batch([(2, 16 + i % 5) for i in range(128)] + [(1, 40)] * 7 + [(3, 5)], [3, 1])  # the last ones share no page
    _run(b, cu, prefix, True)


def test_sequences_that_end_with_the_prefix():
    b, cu, prefix = _batch([(6, 256)], [0])
    _run(b, cu, prefix, True)


def test_a_sequence_shorter_than_its_prefix():
    b, cu, prefix = _batch([(6, 640), (4, 64)], [20, 3], stale=None)
    b.lens_host[[1, 2, 4, 7]] = [200, 0, 639, 1]
    b.lens = torch.from_numpy(b.lens_host).cuda()
    out = _run(b, cu, prefix, True)
    assert (out[2] == 0).all()


def test_unmapped_pages():
    b, cu, prefix = _batch([(5, 320), (3, 48)], [20, 100], holes=[(i, 3) for i in range(5)] + [(1, 21)] + [(i, j) for i in (5, 6, 7) for j in range(3)])
    _run(b, cu, prefix, True)


def test_nothing_shared_is_paged_attention():
    from scicompute_attention_b200 import ops
    b, cu, prefix = _batch([(3, 100)], [20])
    got = ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, np.array([0, 3], np.int32), np.array([0], np.int32),
                                     block_size=b.bs)
    want = ops.paged_attention(b.q, b.k, b.v, b.table, b.lens, block_size=b.bs)
    assert torch.allclose(got.float(), want.float(), atol=2.0 ** -7)


def test_lists_of_every_kind():
    from scicompute_attention_b200 import ops
    b, cu, prefix = _batch([(3, 100), (4, 64)], [20])
    run = lambda c, p: ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, c, p, block_size=b.bs)
    want = run(np.array(cu, np.int32), np.array(prefix, np.int32))
    for other in (lambda x: x, lambda x: np.array(x, np.int64), lambda x: torch.tensor(x)):
        assert torch.equal(want, run(other(cu), other(prefix)))


def test_captured_and_on_another_stream():
    from scicompute_attention_b200 import ops
    b, cu, prefix = _batch([(3, 700), (20, 300)], [20, 200])
    w0 = b.weights.clone()
    run = lambda c, p, w, **more: ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, c, p, block_size=b.bs, weights=w, **more)
    want = run(cu, prefix, b.weights)
    w1, w2 = w0.clone(), w0.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = run(cu, prefix, w1, stream=stream)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want) and torch.equal(w1, b.weights)
    mine = [np.array(x, np.int32) for x in (cu, prefix)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*mine, w2)
    for x in mine:
        x[:] = -1  # the graph has what it needs
    for _ in range(3):
        w2.copy_(w0)
        graph.replay()
        assert torch.equal(got, want) and torch.equal(w2, b.weights)


def test_numbers_of_other_types():
    from scicompute_attention_b200 import ops
    b, cu, prefix = _batch([(3, 100)], [20])
    run = lambda t, n: ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, cu, prefix, block_size=b.bs, typical_len=t, longest_len=n)
    assert torch.equal(run(110, 200), run(np.int64(110), np.int32(200)))
    w = [b.weights.clone() for _ in range(2)]
    evict = lambda w, f: ops.kv_evict(b.k.clone(), b.v.clone(), w, b.table, b.lens, keep=f(110), recent=f(3), first=f(96))
    assert torch.equal(evict(w[0], int), evict(w[1], np.int64)) and torch.equal(*w)


def test_back_to_back_calls_on_one_stream():
    """The second kernel of a call may start beside the first; calls that share scratch stay apart."""
    a, b = _batch([(30, 2000)], [5, 300], seed=1), _batch([(7, 900), (9, 1500)], [40], seed=2)
    from scicompute_attention_b200 import ops
    run = lambda x: ops.paged_attention_shared(x[0].q, x[0].k, x[0].v, x[0].table, x[0].lens, x[1], x[2], block_size=16)
    want = run(a), run(b)
    torch.cuda.synchronize()
    got = [run(x) for _ in range(20) for x in (a, b)]
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))
