"""kv_evict against its definition, bit by bit: which tokens stay, where they go, what is left alone."""
import numpy as np
import pytest
import torch

import cache_reference as ref

pytestmark = pytest.mark.gpu


def _raw(x):
    """Numbers as whole numbers of their width: NaN compares too."""
    return x.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()]).cpu().numpy()


def _check(b, weights, *, keep, recent=0, first=0, k=None, v=None):
    from scicompute_attention_b200 import ops
    k, v = b.k if k is None else k, b.v if v is None else v
    first_host = first.cpu().numpy() if isinstance(first, torch.Tensor) else first
    want = ref.evict(_raw(k), _raw(v), weights.cpu().numpy(), b.table_host, b.lens_host, keep=keep, recent=recent, first=first_host)
    lens = ops.kv_evict(k, v, weights, b.table, b.lens, keep=keep, recent=recent, first=first)
    assert lens.dtype == torch.int32
    np.testing.assert_array_equal(lens.cpu().numpy(), np.maximum(want[3], 0))
    np.testing.assert_array_equal(weights.cpu().numpy().view(np.int32), want[2].view(np.int32))
    np.testing.assert_array_equal(_raw(k), want[0])
    np.testing.assert_array_equal(_raw(v), want[1])
    np.testing.assert_array_equal(b.lens.cpu().numpy(), b.lens_host)


@pytest.mark.parametrize("keep,recent,first", [(40, 8, 4), (40, 0, 0), (40, 40, 0), (40, 36, 4), (33, 1, 0), (1, 0, 0), (0, 0, 0), (1, 1, 0), (5, 30, 30),
                                               (63, 20, 0), (1000, 10, 10)])
def test_ragged_batch(keep, recent, first):
    _check(b := ref.Batch([0, 1, 2, 39, 40, 41, 64, 65, 129, 300]), b.weights, keep=keep, recent=recent, first=first)


@pytest.mark.parametrize("lens", [[1], [17, 5000], [9000, 8193, 700], [20011]])
def test_long_sequences(lens):
    b = ref.Batch(lens, hkv=2, hq=2, d=16, bs=32)
    _check(b, b.weights, keep=max(lens) // 3, recent=max(lens) // 10, first=3)


@pytest.mark.parametrize("recent,evicted", [(500, 1), (700, 30), (1500, 200), (129, 128), (128, 128)])
def test_last_tokens_that_overlap_their_new_places(recent, evicted):
    b = ref.Batch([1600 + evicted], hkv=2, hq=2, d=64)
    _check(b, b.weights, keep=1600, recent=recent, first=1)


@pytest.mark.parametrize("kind", ["equal", "two", "zeros", "nan", "inf", "signs", "tiny", "rising", "falling"])
def test_weights_of_every_kind(kind):
    b = ref.Batch([700, 300, 90], d=16)
    w = b.weights
    j = torch.arange(w.shape[2], device="cuda", dtype=torch.float32).expand_as(w)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "two":
        w.copy_((w > 0.4).float())
    elif kind == "zeros":
        w.mul_(w > 0.9)
        w[:, :, ::3] = -0.0
    elif kind == "nan":
        w[w < 0.3] = float("nan")
        w[0, 0, 5] = -float("nan")
    elif kind == "inf":
        w[w < 0.3] = float("inf")
        w[w > 0.8] = -float("inf")
    elif kind == "signs":
        w.sub_(0.5)
    elif kind == "tiny":  # differ in the last digit only, some below the normal numbers
        w.copy_((j.int() * 7919 % 1009).view(torch.float32))
    elif kind == "rising":
        w.copy_(j)
    elif kind == "falling":
        w.copy_(-j)
    _check(b, w, keep=64, recent=10, first=2)


@pytest.mark.parametrize("dtype,d,bs", [(torch.float32, 128, 16), (torch.float16, 64, 8), (torch.bfloat16, 256, 64), (torch.float16, 20, 16),
                                        (torch.bfloat16, 3, 7), (torch.float32, 5, 1)])
def test_types_and_shapes(dtype, d, bs):
    b = ref.Batch([100, 257, 31], hkv=3, hq=3, d=d, bs=bs, dtype=dtype)
    _check(b, b.weights, keep=30, recent=7, first=2)


def test_first_tokens_by_sequence():
    b = ref.Batch([100, 200, 50, 60, 10], prefixes=[(0, 4, 48)])
    first = torch.tensor([48, 48, 48, 48, -3], dtype=torch.int32, device="cuda")
    shared = b.table[0, :3].long()
    before = b.k[shared].clone()
    _check(b, b.weights, keep=56, recent=5, first=first)
    assert torch.equal(_int(b.k[shared]), _int(before))


def _int(x):
    return x.view(torch.int16)


def test_unmapped_pages_are_left_alone():
    b = ref.Batch([200, 90], holes=[(0, 1), (0, 9), (1, 5)])
    b.table[1, 0] = b.blocks  # beyond the pool
    b.table_host[1, 0] = b.blocks
    _check(b, b.weights, keep=40, recent=12, first=0)


def test_lengths_beyond_the_table_and_below_zero():
    b = ref.Batch([80, 64, 10], extra_pages=0)
    b.lens_host[:] = [1 << 30, -5, 10]
    b.lens = torch.from_numpy(b.lens_host).cuda()
    from scicompute_attention_b200 import ops
    k, v, w = _raw(b.k), _raw(b.v), b.weights.cpu().numpy()
    want = ref.evict(k, v, w, b.table_host, b.lens_host, keep=30, recent=4, first=1)
    lens = ops.kv_evict(b.k, b.v, b.weights, b.table, b.lens, keep=30, recent=4, first=1)
    assert lens.tolist() == [30, 0, 10] == want[3].tolist()
    np.testing.assert_array_equal(_raw(b.k), want[0])
    np.testing.assert_array_equal(b.weights.cpu().numpy(), want[2])


def test_more_rows_and_columns_than_needed_are_left_alone():
    b = ref.Batch([100, 200])
    wide = torch.full((4, 2, b.width * b.bs + 3), 7.0, device="cuda")
    wide[:2, :, :b.width * b.bs] = b.weights
    _check(b, wide, keep=50, recent=5)
    assert (wide[2:] == 7).all() and (wide[:2, :, b.width * b.bs:] == 7).all()


def test_twice_is_once():
    from scicompute_attention_b200 import ops
    b = ref.Batch([100, 200, 30])
    lens = ops.kv_evict(b.k, b.v, b.weights, b.table, b.lens, keep=50, recent=5, first=2)
    k, w = _raw(b.k).copy(), b.weights.clone()
    again = ops.kv_evict(b.k, b.v, b.weights, b.table, lens, keep=50, recent=5, first=2)
    assert torch.equal(lens, again) and torch.equal(w, b.weights)
    np.testing.assert_array_equal(_raw(b.k), k)


def test_captured_and_on_another_stream():
    from scicompute_attention_b200 import ops
    a, b, c = (ref.Batch([100, 900, 30]) for _ in range(3))
    run = lambda x, **w: ops.kv_evict(x.k, x.v, x.weights, x.table, x.lens, keep=60, recent=9, first=1, **w)
    want = run(a)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    lens = run(b, stream=stream)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(want, lens) and torch.equal(a.weights, b.weights) and torch.equal(_int(a.k), _int(b.k))
    keep = [x.clone() for x in (c.k, c.v, c.weights)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens = run(c)
    for _ in range(2):
        for x, y in zip((c.k, c.v, c.weights), keep):
            x.copy_(y)
        graph.replay()
        assert torch.equal(want, lens) and torch.equal(a.weights, c.weights) and torch.equal(_int(a.k), _int(c.k)) and torch.equal(_int(a.v), _int(c.v))
