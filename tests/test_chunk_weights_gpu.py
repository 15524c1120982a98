"""A chunk of new tokens with the weights of the cached ones: output and weights against 64 bits."""
import numpy as np
import pytest
import torch

import cache_reference as ref
import helpers
import oracle_lib as ol

pytestmark = pytest.mark.gpu

DT = {torch.float16: ol.DT_F16, torch.bfloat16: ol.DT_BF16}


def _chunk(b, new, seed=5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return torch.randn((int(cu[-1]), b.hq, b.d), generator=gen, device="cuda").to(b.dtype), cu


def _check(b, q, cu, out, weights, before, causal=True, last=0):
    group = b.hq // b.hkv
    for s in range(len(b.lens_host)):
        rows, new = q[cu[s]:cu[s + 1]], int(cu[s + 1] - cu[s])
        want, p, at, size = ref.attend(b, rows, s, new, causal)
        helpers.check_close(out[cu[s]:cu[s + 1]].float().cpu().numpy(), want.cpu().numpy(), DT[b.dtype], f"sequence {s}")
        counted = p[max(0, new - last):] if last else p
        added = torch.zeros_like(before[s], dtype=torch.float64)
        added[:, torch.from_numpy(at).cuda()] = counted.view(counted.shape[0], b.hkv, group, -1).sum((0, 2))
        ref.check_weights(weights[s], before[s], added, ref.weights_bound(b.d, len(at), group * new, size), f"sequence {s}")
        untouched = added == 0
        assert torch.equal(weights[s][untouched], before[s][untouched])


def _run(b, new, causal=True, last=0, **more):
    from scicompute_attention_b200 import ops
    q, cu = _chunk(b, new)
    before = b.weights.clone()
    out = ops.flash_attention_paged_weights(q, b.k, b.v, b.table, cu, b.lens_host, b.weights, causal=causal, last=last, **more)
    _check(b, q, cu, out, b.weights, before, causal, last)
    return out


# The chunk kernels read a sequence's last page whole: what lies in it behind the last token is finite here, as flash_attention_paged has it.
def _batch(lens, **more):
    return ref.Batch(lens, stale=1.5, **more)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 64, torch.bfloat16), (8, 8, 128, torch.float16), (32, 2, 64, torch.float16), (6, 3, 96, torch.bfloat16),
                                            (16, 1, 256, torch.bfloat16), (5, 1, 32, torch.float16), (24, 1, 128, torch.bfloat16), (4, 2, 160, torch.float16),
                                            (3, 1, 192, torch.bfloat16)])
@pytest.mark.parametrize("causal", [True, False])
def test_heads_and_types(hq, hkv, d, dtype, causal):
    _run(_batch([1, 130, 400, 128, 65], hq=hq, hkv=hkv, d=d, dtype=dtype), [1, 130, 37, 1, 64], causal)


@pytest.mark.parametrize("last", [0, 1, 7, 32, 64, 100000])
def test_last_tokens(last):
    _run(_batch([300, 700, 90]), [5, 300, 90], last=last)


@pytest.mark.parametrize("lens,new,bs", [([1], [1], 16), ([733], [37], 16), ([2000], [2000], 32), ([128, 129, 127], [128, 129, 127], 8), ([3000], [1], 64),
                                         ([40] * 30, [40] * 30, 16), ([1500, 20], [700, 3], 64), ([9] * 128, [2] * 128, 8), ([9] * 129, [2] * 129, 8)])
def test_lengths_and_pages(lens, new, bs):
    _run(_batch(lens, bs=bs), new)


def test_unmapped_pages_weigh_nothing():
    b = _batch([300, 64], holes=[(0, 0), (0, 9), (1, 0), (1, 1), (1, 2), (1, 3)])
    out = _run(b, [40, 20])
    assert (out[40:] == 0).all()


def test_the_output_is_that_of_the_prefill_and_the_bits_are_the_same_again():
    from scicompute_attention_b200 import ops
    b = _batch([900, 300])
    q, cu = _chunk(b, [300, 20])
    plain = ops.flash_attention_paged(q, b.k, b.v, b.table, cu, b.lens_host)
    before = b.weights.clone()
    want = ops.flash_attention_paged_weights(q, b.k, b.v, b.table, cu, b.lens_host, b.weights)
    assert torch.equal(plain, want)
    for _ in range(3):
        w = before.clone()
        assert torch.equal(plain, ops.flash_attention_paged_weights(q, b.k, b.v, b.table, cu, b.lens_host, w)) and torch.equal(w, b.weights)


def test_nan_queries_of_one_sequence_stay_there():
    from scicompute_attention_b200 import ops
    b = _batch([200, 300, 150])
    q, cu = _chunk(b, [50, 60, 70])
    clean, before = b.weights.clone(), b.weights.clone()
    ops.flash_attention_paged_weights(q, b.k, b.v, b.table, cu, b.lens_host, clean)
    q[cu[1]:cu[2], 5] = float("nan")  # kv head 1 of the one in the middle
    ops.flash_attention_paged_weights(q, b.k, b.v, b.table, cu, b.lens_host, b.weights)
    for s, g in ((0, 0), (0, 1), (1, 0), (2, 0), (2, 1)):
        assert torch.equal(b.weights[s, g], clean[s, g])
    assert b.weights[1, 1, :300].isnan().all() and torch.equal(b.weights[1, 1, 300:], before[1, 1, 300:])


def test_a_chunk_of_one_token_is_a_step():
    from scicompute_attention_b200 import ops
    b = _batch([500, 33])
    q, cu = _chunk(b, [1, 1])
    w = b.weights.clone()
    _run(b, [1, 1])
    ops.paged_attention_weights(q.unsqueeze(2), b.k, b.v, b.table, b.lens, w, block_size=b.bs)
    assert torch.allclose(w, b.weights, rtol=1e-5, atol=1e-7)


def test_captured_and_on_another_stream():
    from scicompute_attention_b200 import ops
    b = _batch([900, 300])
    q, cu = _chunk(b, [300, 20])
    w0 = b.weights.clone()
    run = lambda c, n, w, **more: ops.flash_attention_paged_weights(q, b.k, b.v, b.table, c, n, w, **more)
    want = run(cu, b.lens_host, b.weights)
    w1, w2 = w0.clone(), w0.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = run(cu, b.lens_host, w1, stream=stream)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want) and torch.equal(w1, b.weights)
    mine = cu.copy(), b.lens_host.copy()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*mine, w2)
    for x in mine:
        x[:] = -1
    for _ in range(3):
        w2.copy_(w0)
        graph.replay()
        assert torch.equal(got, want) and torch.equal(w2, b.weights)
