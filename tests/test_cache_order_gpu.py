"""The second kernel of a decode over shared prefixes may start beside the first. What the kernels ahead of the call write - tokens, lengths, queries -
it reads as written, call after call without a wait on the host."""
import numpy as np
import pytest
import torch

import cache_reference as ref
from launches import THREE, launches

pytestmark = pytest.mark.gpu

STEPS = 24


def _turn(b, cu, prefix, tokens, queries, wait):
    """Steps of a server from the state of `b`: lengths grow on the device, a token a sequence is appended, and attended with weights. A copy of the
    pools, so that both turns begin alike."""
    from scicompute_attention_b200 import ops
    k, v, weights, lens, q = b.k.clone(), b.v.clone(), b.weights.clone(), b.lens.clone(), torch.empty_like(b.q)
    outs = []
    for step in range(STEPS):
        lens.add_(1)
        q.copy_(queries[step])
        ops.kv_append_batched(k, v, tokens[0][step], tokens[1][step], b.table, lens)
        if wait:
            torch.cuda.synchronize()
        outs.append(ops.paged_attention_shared(q, k, v, b.table, lens, cu, prefix, block_size=b.bs, weights=weights))
        if wait:
            torch.cuda.synchronize()
    return outs, weights, k, v, lens


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,groups", [(128, [(30, 700), (2, 16), (18, 300)]), (64, [(90, 500), (20, 40)]), (256, [(20, 200)])])
def test_appends_and_steps_back_to_back(d, groups, dtype):
    hkv, prefixes, cu = (8 if d == 128 else 4), [], [0]
    for n, tokens in groups:
        prefixes.append((cu[-1], cu[-1] + n, tokens))
        cu.append(cu[-1] + n)
    lens = [tokens + 1 + i % 30 + STEPS for first, end, tokens in prefixes for i in range(end - first)]
    b = ref.Batch(lens, hq=4 * hkv, hkv=hkv, d=d, dtype=dtype, prefixes=prefixes)
    b.lens_host -= STEPS
    b.lens = torch.from_numpy(b.lens_host).cuda()
    cu, prefix, n = np.array(cu, np.int32), np.array([t for _, _, t in prefixes], np.int32), cu[-1]
    rand = lambda *s: torch.randn(s, generator=b.gen, device="cuda").to(dtype)
    tokens, queries = (rand(STEPS, n, hkv, d), rand(STEPS, n, hkv, d)), rand(STEPS, *b.q.shape)
    outs, *left = _turn(b, cu, prefix, tokens, queries, True)
    from scicompute_attention_b200 import ops
    step = lambda: ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, cu, prefix, block_size=b.bs, weights=b.weights.clone())
    assert launches(step) == THREE
    for _ in range(3):
        torch.cuda.synchronize()
        got, *again = _turn(b, cu, prefix, tokens, queries, False)
        assert all(torch.equal(x, y) for x, y in zip(outs, got))
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(left, again))  # the pools hold NaN
    # the last step against 64 bits
    weights, b.k, b.v, b.lens = left
    b.lens_host += STEPS
    for s in range(0, n, 7):
        want, p, at, size = ref.attend(b, queries[-1][s].transpose(0, 1), s)
        # P in fp16 over shared pages: half a step; what is too small for that is off by 2^-25 of the maximum, which `keys` steps of 2^-24 cover
        ref.check_output(outs[-1][s, :, 0], want[0], p[0], b.keys(s)[2], ref.weights_bound(d, len(at), 1, size), 2.0 ** -11)


def test_a_mark_that_is_not_there_or_left_over():
    """Scratch that begins with anything: the mark of an earlier call too."""
    from scicompute_attention_b200 import ops
    b = ref.Batch([600 + i for i in range(40)], hq=16, hkv=8, d=128, prefixes=[(0, 40, 512)])
    run = lambda: ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, np.array([0, 40], np.int32), np.array([512], np.int32), block_size=16)
    assert launches(run) == THREE
    want = run()
    scratch = ops.acquire_scratch_fp32(1, b.q.device, handle=ops._stream_ptr(None))
    assert (scratch[:2].view(torch.int64) == 0).all()  # taken away by the end of a call
    for mark in (0, -1, 0xff8b4d277f9a3c51 - (1 << 64)):
        scratch[:2].view(torch.int64).fill_(mark)
        assert torch.equal(run(), want) and (scratch[:2].view(torch.int64) == 0).all()
