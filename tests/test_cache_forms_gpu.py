"""The native form of the operators of a paged cache that stays small against their general form: the same bits; forms that the native one
leaves alone; scratch that grows, and calls from two threads and two streams at once."""
import threading

import numpy as np
import pytest
import torch

import cache_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture
def general(monkeypatch):
    from scicompute_attention_b200 import ops
    return lambda: monkeypatch.setattr(ops, "_native", lambda: ops._GeneralFormOnly())


def _calls(b, cu, prefix):
    """Eviction leaves the pages alone that sequences share."""
    from scicompute_attention_b200 import ops
    chunk = torch.randn((5 + 2 * len(b.lens_host), b.hq, b.d), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(b.dtype)
    new = np.array([7] + [2] * (len(b.lens_host) - 1))
    cu_q = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)

    def run():
        w = [b.weights.clone() for _ in range(4)]
        k, v = b.k.clone(), b.v.clone()
        return [ops.paged_attention_weights(b.q, b.k, b.v, b.table, b.lens, w[0], block_size=b.bs, typical_len=50, longest_len=int(b.lens_host.max())),
                ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, cu, prefix, block_size=b.bs, weights=w[1], scale=0.2),
                ops.paged_attention_shared(b.q, b.k, b.v, b.table, b.lens, cu, prefix, block_size=b.bs),
                ops.flash_attention_paged_weights(chunk, b.k, b.v, b.table, cu_q, b.lens_host, w[2], last=3),
                ops.kv_evict(k, v, w[3], b.table, b.lens, keep=int(prefix[0]) + 12, recent=9,
                             first=int(prefix[0]) // b.bs * b.bs), k.view(torch.int16), v.view(torch.int16), *w]
    return run


@pytest.mark.parametrize("n,tokens", [(3, 100), (40, 900)])  # one launch, and three
def test_native_and_general_form_agree(general, n, tokens):
    b = ref.Batch([tokens + 30 + i for i in range(n)], prefixes=[(0, n, tokens)], stale=0.5)
    run = _calls(b, np.array([0, n], np.int32), np.array([tokens], np.int32))
    native = run()
    general()
    for a, c in zip(native, run()):
        assert torch.equal(a, c)


def test_threads_with_streams_of_their_own():
    b = [ref.Batch([300 + 50 * i, 900, 40], prefixes=[(0, 3, 32)], stale=0.5, seed=i) for i in range(4)]
    runs = [_calls(x, np.array([0, 3], np.int32), np.array([32], np.int32)) for x in b]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = runs[i]()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, c) for a, c in zip(got, want[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_turn_of_a_server():
    """A prompt goes into pages that several answers share, their tokens are appended and attended with weights, the cache is brought down, and the
    answers go on over what is left: every step against 64 bits."""
    from scicompute_attention_b200 import ops
    hq, hkv, d, bs, n, prompt = 8, 2, 64, 16, 4, 160
    b = ref.Batch([prompt + 60] * n, hq=hq, hkv=hkv, d=d, bs=bs, prefixes=[(0, n, prompt)], extra_pages=4, stale=0.5)
    gen = torch.Generator(device="cuda").manual_seed(9)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda").to(torch.bfloat16)
    b.weights.zero_()
    pages = torch.arange(prompt, device="cuda")
    slots = (b.table[0, pages // bs] * bs + pages % bs).to(torch.int32)
    ops.kv_append(b.k, b.v, rand(prompt, hkv, d), rand(prompt, hkv, d), slots)
    first = torch.full((n,), prompt, dtype=torch.int32, device="cuda")
    cu, prefix = np.array([0, n], np.int32), np.array([prompt], np.int32)
    b.lens_host[:] = prompt
    for step in range(1, 61):
        b.lens_host += 1
        b.lens = torch.from_numpy(b.lens_host).cuda()
        ops.kv_append_batched(b.k, b.v, rand(n, hkv, d), rand(n, hkv, d), b.table, b.lens)
        q, before = rand(n, hq, 1, d), b.weights.clone()
        out = ops.paged_attention_shared(q, b.k, b.v, b.table, b.lens, cu, prefix, block_size=bs, weights=b.weights)
        if step % 20 in (1, 0):
            for s in range(n):
                want, p, at, size = ref.attend(b, q[s].transpose(0, 1), s)
                ref.check_output(out[s, :, 0], want[0], p[0], b.keys(s)[2], ref.weights_bound(d, len(at), 1, size), 2.0 ** -9)
                added = torch.zeros_like(before[s], dtype=torch.float64)
                added[:, prompt:len(at)] = p[0].view(hkv, hq // hkv, -1).sum(1)[:, prompt:]
                ref.check_weights(b.weights[s], before[s], added, ref.weights_bound(d, len(at), hq // hkv, size))
        if step % 20 == 0:
            raw = lambda x: x.view(torch.int16).cpu().numpy()
            want = ref.evict(raw(b.k), raw(b.v), b.weights.cpu().numpy(), b.table_host, b.lens_host, keep=prompt + 12, recent=5, first=[prompt] * n)
            b.lens = ops.kv_evict(b.k, b.v, b.weights, b.table, b.lens, keep=prompt + 12, recent=5, first=first)
            np.testing.assert_array_equal(raw(b.k), want[0])
            np.testing.assert_array_equal(raw(b.v), want[1])
            np.testing.assert_array_equal(b.weights.cpu().numpy(), want[2])
            b.lens_host[:] = b.lens.cpu().numpy()
            assert (b.lens_host == prompt + 12).all()
