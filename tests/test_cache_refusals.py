"""Calls of the operators of a paged cache that stays small which cannot be served are refused before anything is launched: by the operators (on
the CPU, with the launch layer replaced) and by the C entries."""
import ctypes as C

import numpy as np
import pytest
import torch

from scicompute_attention_b200 import _lib, ops

BF, I32 = torch.bfloat16, torch.int32
B, HQ, HKV, D, BS, NB, W = 2, 4, 2, 64, 16, 6, 4


def _calls(dev):
    t = lambda *shape, dtype=BF: torch.zeros(shape, dtype=dtype, device=dev)
    ints = lambda *shape: torch.zeros(shape, dtype=I32, device=dev)
    pool, other, weights = t(NB, BS, HKV, D), t(NB, BS, HKV, 2 * D), t(B, HKV, W * BS, dtype=torch.float32)
    q, q1, table, lens = t(9, HQ, D), t(B, HQ, 1, D), ints(B, W), ints(B)
    cu, new, total = np.array([0, 2], np.int32), np.array([0, 4, 9], np.int32), np.array([20, 20], np.int32)
    prefix = np.array([16], np.int32)
    step = lambda q_=q1, k=pool, v=pool, tab=table, n=lens, w=weights, bs=BS: lambda **more: ops.paged_attention_weights(q_, k, v, tab, n, w, block_size=bs, **more)
    shared = lambda q_=q1, k=pool, tab=table, n=lens, c=cu, p=prefix, w=None, bs=BS: lambda **more: ops.paged_attention_shared(
        q_, k, k, tab, n, c, p, block_size=bs, weights=w, **more)
    chunk = lambda q_=q, k=pool, v=pool, tab=table, c=new, n=total, w=weights, last=0: lambda **more: ops.flash_attention_paged_weights(
        q_, k, v, tab, c, n, w, last=last, **more)
    evict = lambda k=pool, v=pool, w=weights, tab=table, n=lens, keep=8, recent=2, first=0: lambda **more: ops.kv_evict(
        k, v, w, tab, n, keep=keep, recent=recent, first=first, **more)
    narrow = t(B, HKV, W * BS - 1, dtype=torch.float32)
    calls = [("no weights", step(w=None)), ("fp32", step(q_=q1.float(), k=pool.float(), v=pool.float())), ("q of three dims", step(q_=q)),
             ("two query tokens", step(q_=t(B, HQ, 2, D))), ("q strided", step(q_=t(B, 2 * HQ, 1, D)[:, ::2])), ("types differ", step(q_=q1.half())),
             ("head dims", step(k=other, v=other)), ("pools differ", step(v=other)), ("block size", step(bs=8)), ("heads do not divide", step(q_=t(B, 3, 1, D))),
             ("pool strided", step(k=t(NB, BS, 2 * HKV, D)[:, :, :HKV], v=t(NB, BS, 2 * HKV, D)[:, :, :HKV])), ("pool of three dims", step(k=pool[0], v=pool[0])),
             ("table sliced", step(tab=ints(B, 9)[:, :W])), ("long table", step(tab=table.long())), ("few table rows", step(tab=table[:1])),
             ("long lengths", step(n=lens.long())), ("few lengths", step(n=lens[:1])),
             ("weights of 16 bits", step(w=weights.half())), ("weights too narrow", step(w=narrow)), ("few rows of weights", step(w=weights[:1])),
             ("weights of other heads", step(w=t(B, HQ, W * BS, dtype=torch.float32))), ("weights turned", step(w=t(B, W * BS, HKV, dtype=torch.float32).transpose(1, 2))),
             ("shared, few offsets", shared(c=cu[:1])), ("shared, offsets of two dims", shared(c=cu[None])), ("shared, offsets of floats", shared(c=np.array([0.0, 2.0]))),
             ("shared, offsets that end early", shared(c=np.array([0, 1], np.int32))), ("shared, no groups for two sequences", shared(c=np.array([0]), p=np.array([], np.int32))),
             ("shared, offsets of a tensor that begin late", shared(c=torch.tensor([1, 2]))), ("shared, beyond 32 bits", shared(p=np.array([1 << 40]))), ("shared, weights too narrow", shared(w=narrow)), ("shared, head dims", shared(k=other)),
             ("chunk, fp32", chunk(q_=q.float(), k=pool.float(), v=pool.float())), ("chunk, q of four dims", chunk(q_=q1)), ("chunk, q strided", chunk(q_=t(9, 2 * HQ, D)[:, ::2])),
             ("chunk, head dims", chunk(k=other, v=other)), ("chunk, pools differ", chunk(v=other)), ("chunk, few offsets", chunk(c=new[:2])),
             ("chunk, table sliced", chunk(tab=ints(B, 9)[:, :W])), ("chunk, few table rows", chunk(tab=table[:1])), ("chunk, weights too narrow", chunk(w=narrow)),
             ("chunk, weights of 16 bits", chunk(w=weights.half())), ("chunk, last below zero", chunk(last=-1)), ("chunk, heads do not divide", chunk(q_=t(9, 3, D))),
             ("evict, keep below zero", evict(keep=-1)), ("evict, recent below zero", evict(recent=-1)), ("evict, first below zero", evict(first=-1)),
             ("evict, long first", evict(first=lens.long())), ("evict, few first", evict(first=lens[:1])), ("evict, pools differ", evict(v=other)),
             ("evict, pool strided", evict(k=t(NB, BS, 2 * HKV, D)[:, :, :HKV])), ("evict, pool of three dims", evict(k=pool[0])), ("evict, few table rows", evict(tab=table[:1])),
             ("evict, weights too narrow", evict(w=narrow)), ("evict, weights of 16 bits", evict(w=weights.half())), ("evict, long lengths", evict(n=lens.long()))]
    return calls


NAMES = [name for name, _ in _calls("meta")]


class _NoLaunch:
    def __getattr__(self, name):
        raise AssertionError(f"{name} called")


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(ops, "_require_cuda", lambda *tensors: None)
    monkeypatch.setattr(ops, "_native", lambda: ops._GeneralFormOnly())
    monkeypatch.setattr(ops, "_elsewhere", lambda t, stream: False)
    monkeypatch.setattr(ops, "lib", lambda: _NoLaunch())


@pytest.mark.parametrize("i", range(len(NAMES)), ids=NAMES)
def test_operators_refuse(no_launch, i):
    with pytest.raises(_lib.ScaError):
        _calls("cpu")[i][1]()


def test_tensors_on_the_host_are_refused():
    for name, call in _calls("cpu"):
        if "weights" in name and "few" not in name:
            continue
        with pytest.raises(_lib.ScaError):
            call()


def _aligned(n):
    raw = C.create_string_buffer(n + 64)
    return raw, (C.addressof(raw) + 63) // 64 * 64


def _step(**fields):
    keep, at = _aligned(64)
    p, x = _lib.DecodeFwdParams(), _lib.PagedStep()
    p.q = p.k = p.v = p.out = p.page_table = p.seq_lens = at
    p.batch, p.num_heads, p.num_kv_heads, p.head_dim, p.scale, p.dtype = 4, 8, 2, 64, 0.1, _lib.DTYPE_BF16
    p.q_stride = p.o_stride = _lib.DecodeStrides(512, 64, 64)
    p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = 16, 8, 100
    x.scratch, x.scratch_floats = at, 1 << 40
    x.weights, x.weights_row = at, 128
    lists = {}
    for name, value in fields.items():
        if isinstance(value, list):
            lists[name] = value = np.array(value, np.int32)
            setattr(x, name, value.ctypes.data)
        elif hasattr(x, name):
            setattr(x, name, value)
        else:
            setattr(p, name, value)
    rc = _lib.lib().sca_launch_paged_step(C.byref(p), C.byref(x), None)
    return rc, _lib.lib().sca_last_error().decode()


@pytest.mark.parametrize("fields,what", [
    (dict(q=None), "null"), (dict(page_table=None), "null"), (dict(scratch=None), "null"), (dict(dtype=_lib.DTYPE_F32), "fp16 or bf16"), (dict(head_dim=48), "not instantiated"),
    (dict(num_heads=7), "geometry"), (dict(batch=0), "geometry"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(block_size=0), "positive"), (dict(max_blocks_per_seq=0), "positive"), (dict(weights_row=127), "rows of 127"), (dict(num_kv_blocks=1 << 30), "2^31"),
    (dict(scratch_floats=10), "too small"), (dict(num_groups=1), "null groups"), (dict(num_groups=-1), "null groups"),
    (dict(num_groups=1, cu_groups=[0, 3], prefix_lens=[16]), "start at 0 and end"), (dict(num_groups=1, cu_groups=[1, 4], prefix_lens=[16]), "start at 0 and end"),
    (dict(num_groups=2, cu_groups=[0, 5, 4], prefix_lens=[16, 16]), "must not fall"), (dict(num_groups=1, cu_groups=[0, 4], prefix_lens=[129]), "prefix of 129"),
    (dict(num_groups=1, cu_groups=[0, 4], prefix_lens=[-1]), "prefix of -1"), (dict(num_groups=1, cu_groups=[0, 4], prefix_lens=[16], block_size=24, weights_row=192), "block_size=24"),
    (dict(batch=300, num_groups=150, cu_groups=list(range(0, 301, 2)), prefix_lens=[16] * 150), "150 groups")])
def test_step_entry_refuses(fields, what):
    rc, message = _step(**fields)
    assert rc == 4 and what in message, message


def test_step_scratch_covers_rows_and_scores():
    p, x = _lib.DecodeFwdParams(), _lib.PagedStep()
    p.batch, p.num_heads, p.num_kv_heads, p.head_dim, p.scale, p.dtype = 4, 8, 2, 64, 0.1, _lib.DTYPE_BF16
    p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = 16, 8, 100
    without = _lib.lib().sca_paged_step_scratch_floats(C.byref(p), C.byref(x))
    x.weights, x.weights_row = 64, 128
    assert without >= 4 * 8 * 66 and _lib.lib().sca_paged_step_scratch_floats(C.byref(p), C.byref(x)) >= without + 4 * 8 * 128
    x.longest_len = 40
    assert _lib.lib().sca_paged_step_scratch_floats(C.byref(p), C.byref(x)) < without + 4 * 8 * 128
    p.head_dim = 1
    assert _lib.lib().sca_paged_step_scratch_floats(C.byref(p), C.byref(x)) < 0


def _evict(**fields):
    keep, at = _aligned(64)
    x, shape, elem = _lib.KvEvict(), _lib.KvCacheShape(10, 16, 2, 64), 2
    x.layer_k = x.layer_v = x.weights = x.page_table = x.seq_lens = x.scratch = at
    x.new_lens = at + 32
    x.weights_row, x.num_seqs, x.max_blocks_per_seq, x.keep, x.scratch_ints = 128, 3, 8, 20, 1 << 30
    for name, value in fields.items():
        if name == "elem":
            elem = value
        else:
            setattr(shape if hasattr(shape, name) else x, name, at if value == "lens" else value)
    rc = _lib.lib().sca_launch_kv_evict(C.byref(x), C.byref(shape), elem, None)
    return rc, _lib.lib().sca_last_error().decode()


@pytest.mark.parametrize("fields,what", [
    (dict(layer_k=None), "null"), (dict(weights=None), "null"), (dict(scratch=None), "null"), (dict(new_lens="lens"), "memory of their own"), (dict(num_seqs=0), "positive"),
    (dict(block_size=0), "positive"), (dict(elem=0), "positive"), (dict(keep=-1), "negative"), (dict(recent=-2), "negative"), (dict(first=-3), "negative"),
    (dict(weights_row=127), "rows of 127"), (dict(scratch_ints=3), "too small"), (dict(num_blocks=1 << 40), "out of range"), (dict(max_blocks_per_seq=1 << 40), "out of range")])
def test_evict_entry_refuses(fields, what):
    rc, message = _evict(**fields)
    assert rc == 4 and what in message, message


@pytest.mark.parametrize("fields,what", [(dict(lse=None), "null"), (dict(weights=None), "null"), (dict(weights_row=10), "rows of 10"), (dict(last=-1), "last"),
                                         (dict(scale=float("inf")), "scale"), (dict(block_size=24), "block_size=24")])
def test_chunk_entry_refuses(fields, what):
    keep, at = _aligned(64)
    p, w = _lib.FlashPagedParams(), _lib.ChunkWeights(at, at, 1 << 20, 0)
    cu, lens = np.array([0, 4], np.int32), np.array([20], np.int32)
    p.q = p.out = p.k_pool = p.v_pool = p.page_table = p.workspace = at
    p.total_q, p.num_heads, p.num_kv_heads, p.head_dim, p.num_seqs, p.num_blocks, p.block_size, p.max_blocks_per_seq = 4, 8, 2, 64, 1, 10, 16, 8
    p.cu_seqlens_q, p.seq_lens_kv, p.scale, p.causal, p.dtype_id, p.workspace_bytes = cu.ctypes.data, lens.ctypes.data, 0.1, 1, _lib.DTYPE_BF16, 1 << 20
    for name, value in fields.items():
        setattr(w if hasattr(w, name) else p, name, value)
    assert _lib.lib().sca_launch_flash_paged_weights(C.byref(p), C.byref(w), None) == 4
    assert what in _lib.lib().sca_last_error().decode()
