"""Calls over the 8-bit cache that cannot be served are refused before anything is launched: by the operators (on the CPU, with the launch
layer replaced) and by the C entries."""
import ctypes as C

import numpy as np
import pytest
import torch

from scicompute_attention_b200 import _lib, ops

BF, I32 = torch.bfloat16, torch.int32
B, HQ, HKV, D, BS, NB = 2, 4, 2, 64, 16, 6


def _calls(dev):
    t = lambda *shape, dtype=BF: torch.zeros(shape, dtype=dtype, device=dev)
    ints = lambda *shape: torch.zeros(shape, dtype=I32, device=dev)
    pool = ops.Fp8Pool(t(NB, BS, HKV, D, dtype=torch.uint8).view(torch.float8_e4m3fn), t(NB, HKV, 16, dtype=torch.uint8))
    other = ops.Fp8Pool(t(NB, BS, HKV, 2 * D, dtype=torch.uint8), t(NB, HKV, 16, dtype=torch.uint8))
    new, slots, table, lens = t(3, HKV, D), ints(3), ints(B, 4), ints(B)
    q, q1 = t(9, HQ, D), t(B, HQ, 1, D)
    cu, total = np.array([0, 9], np.int32), np.array([20], np.int32)
    codes, scales = pool
    append = lambda k=pool, v=pool, kn=new, vn=new, s=slots: lambda **w: ops.kv_append_fp8(k, v, kn, vn, s, **w)
    batched = lambda k=pool, kn=new[:B], vn=new[:B], tab=table, n=lens: lambda **w: ops.kv_append_batched_fp8(k, k, kn, vn, tab, n, **w)
    gather = lambda p=pool, ids=slots, dtype=BF: lambda **w: ops.kv_gather_fp8(p, ids, dtype, **w)
    paged = lambda q_=q1, k=pool, v=pool, tab=table, n=lens, bs=BS: lambda **w: ops.paged_attention_fp8(q_, k, v, tab, n, block_size=bs, **w)
    chunk = lambda q_=q, k=pool, v=pool, tab=ints(1, 4), c=cu, n=total: lambda **w: ops.flash_attention_paged_fp8(q_, k, v, tab, c, n, **w)
    return [
        ("append, 16-bit codes", append(k=(t(NB, BS, HKV, D), scales))),
        ("append, codes sliced", append(k=(t(NB, BS, 2 * HKV, D, dtype=torch.uint8)[:, :, :HKV], scales))),
        ("append, scales too few", append(k=(codes, scales[:, :, :8].contiguous()))),
        ("append, scales turned", append(k=(codes, t(NB, 16, HKV, dtype=torch.uint8).transpose(1, 2)))),
        ("append, scales of another type", append(k=(codes, scales.to(torch.int32)))),
        ("append, pools differ", append(v=other)),
        ("append, rows strided", append(kn=t(3, 2 * HKV, D)[:, ::2])),
        ("append, rows narrow", append(kn=t(3, HKV, 32), vn=t(3, HKV, 32))),
        ("append, few v rows", append(vn=new[:2])),
        ("append, k and v of two types", append(vn=new.half())),
        ("append, rows of integers", append(kn=t(3, HKV, D, dtype=torch.int16), vn=t(3, HKV, D, dtype=torch.int16))),
        ("append, few slots", append(s=slots[:2])),
        ("append, long slots", append(s=slots.long())),
        ("batched, long table", batched(tab=table.long())),
        ("batched, table sliced", batched(tab=ints(B, 9)[:, :4])),
        ("batched, few table rows", batched(tab=table[:1])),
        ("batched, few lengths", batched(n=lens[:1])),
        ("gather, long ids", gather(ids=slots.long())),
        ("gather, strided ids", gather(ids=ints(6)[::2])),
        ("gather, into integers", gather(dtype=torch.int16)),
        ("gather, scales missing", gather(p=(codes, scales[:2]))),
        ("paged, fp32 queries", paged(q_=q1.float())),
        ("paged, q strided", paged(q_=t(B, 2 * HQ, 1, D)[:, ::2])),
        ("paged, head dims", paged(k=other, v=other)),
        ("paged, pools differ", paged(v=other)),
        ("paged, block size", paged(bs=8)),
        ("paged, heads do not divide", paged(q_=t(B, 3, 1, D))),
        ("paged, table sliced", paged(tab=ints(B, 9)[:, :4])),
        ("paged, long lengths", paged(n=lens.long())),
        ("paged, few lengths", paged(n=lens[:1])),
        ("chunk, fp32 queries", chunk(q_=q.float())),
        ("chunk, q of four dims", chunk(q_=q1)),
        ("chunk, q strided", chunk(q_=t(9, 2 * HQ, D)[:, ::2])),
        ("chunk, head dims", chunk(k=other, v=other)),
        ("chunk, offsets too few", chunk(c=cu[:1])),
        ("chunk, table sliced", chunk(tab=ints(2, 9)[:, :4])),
        ("chunk, table rows too few", chunk(c=np.array([0, 4, 9], np.int32), n=np.array([20, 20], np.int32))),
    ]


NAMES = [name for name, _ in _calls("meta")]


class _NoLaunch:
    def __getattr__(self, name):
        raise AssertionError(f"{name} called")


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(ops, "_require_cuda", lambda *tensors: None)
    monkeypatch.setattr(ops, "_elsewhere", lambda t, stream: False)
    monkeypatch.setattr(ops, "lib", _NoLaunch)
    monkeypatch.setattr(ops, "_stream_ptr", lambda stream=None: 0)
    monkeypatch.setattr(ops, "sm_count", lambda device: 148)
    monkeypatch.setattr(ops, "acquire_scratch_fp32", lambda n, device, **w: torch.empty(n))


@pytest.mark.parametrize("i", range(len(NAMES)), ids=NAMES)
def test_operators(no_launch, i):
    with pytest.raises(_lib.ScaError) as e:
        _calls("cpu")[i][1]()
    assert e.value.code == 4


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(NAMES)), ids=NAMES)
def test_the_native_forms_refuse_the_same(i):
    said = []
    for w in ({}, {"stream": torch.cuda.current_stream()}):
        with pytest.raises(_lib.ScaError) as e:
            _calls("cuda")[i][1](**w)
        said.append((e.value.code, e.value.message))
    assert said[0] == said[1] and said[0][0] == 4


def test_tensors_on_the_cpu_or_on_two_devices(monkeypatch):
    pool, row, ints = ops.fp8_pool(2, 16, 1, 32, device="cpu"), torch.zeros(1, 1, 32, dtype=BF), torch.zeros(1, dtype=I32)
    for call in (lambda: ops.kv_append_fp8(pool, pool, row, row, ints), lambda: ops.kv_append_batched_fp8(pool, pool, row, row, ints[None], ints),
                 lambda: ops.kv_gather_fp8(pool, ints, BF), lambda: ops.paged_attention_fp8(row[None], pool, pool, ints[None], ints, block_size=16),
                 lambda: ops.flash_attention_paged_fp8(row, pool, pool, ints[None], [0, 1], [1])):
        with pytest.raises(_lib.ScaError) as e:
            call()
        assert e.value.code == 5 and "no CPU path" in str(e.value)
    monkeypatch.setattr(ops, "_require_cuda", lambda *tensors: None)
    far = torch.zeros(1, dtype=I32, device="meta")
    for call in (lambda: ops.kv_append_fp8(pool, pool, row, row, far), lambda: ops.kv_append_batched_fp8(pool, pool, row, row, far[None], ints),
                 lambda: ops.kv_gather_fp8(pool, far, BF), lambda: ops.paged_attention_fp8(row[None], pool, pool, far[None], ints, block_size=16),
                 lambda: ops.flash_attention_paged_fp8(row, pool, pool, far[None], [0, 1], [1])):
        with pytest.raises(_lib.ScaError) as e:
            call()
        assert e.value.code == 4 and "one device" in str(e.value)


def test_decode_of_several_tokens_is_another_operator(no_launch):
    pool = ops.fp8_pool(2, 16, 1, 32, device="cpu")
    with pytest.raises(_lib.ScaError) as e:
        ops.paged_attention_fp8(torch.zeros(1, 1, 2, 32, dtype=BF), pool, pool, torch.zeros(1, 1, dtype=I32), None, block_size=16)
    assert e.value.code == 5


def test_c_entries():
    lib = _lib.lib()
    at = 1 << 20  # an address that nothing reads: every call here is refused on the host
    layer, shape = _lib.Fp8Layer(at, at, at, at), lambda nb=4, bs=16, h=2, d=64: C.byref(_lib.KvCacheShape(nb, bs, h, d))
    assert lib.sca_launch_kv_append_fp8(None, at, at, at, 1, shape(), 2, None) == 4
    assert lib.sca_launch_kv_append_fp8(C.byref(_lib.Fp8Layer(at, at, at, None)), at, at, at, 1, shape(), 2, None) == 4
    assert lib.sca_launch_kv_append_fp8(C.byref(layer), at, None, at, 1, shape(), 2, None) == 4
    assert lib.sca_launch_kv_append_fp8(C.byref(layer), at, at, at, 0, shape(), 2, None) == 4
    for bad in (shape(nb=0), shape(bs=0), shape(h=0), shape(d=0), shape(d=24), shape(d=272), shape(nb=1 << 28), None):
        assert lib.sca_launch_kv_append_fp8(C.byref(layer), at, at, at, 1, bad, 2, None) == 4
        assert lib.sca_launch_kv_append_batched_fp8(C.byref(layer), at, at, at, at, 1, 4, bad, 2, None) == 4
        assert lib.sca_launch_kv_gather_fp8(at, at, at, 1, at, bad, 2, None) == 4
    assert lib.sca_launch_kv_append_fp8(C.byref(layer), at, at, at, 1, shape(), 7, None) == 4
    assert lib.sca_launch_kv_append_fp8(C.byref(_lib.Fp8Layer(at + 8, at, at, at)), at, at, at, 1, shape(), 2, None) == 4
    assert lib.sca_launch_kv_append_batched_fp8(C.byref(layer), at, at, at, at, 0, 4, shape(), 2, None) == 4
    assert lib.sca_launch_kv_append_batched_fp8(C.byref(layer), at, at, at, at, 1, 0, shape(), 2, None) == 4
    assert lib.sca_launch_kv_gather_fp8(at, at, at, 1, at + 8, shape(), 2, None) == 4
    assert lib.sca_launch_kv_gather_fp8(at, at, at, 1, at, shape(), 9, None) == 4

    def decode(**change):
        p = _lib.DecodeFwdParams()
        p.q = p.k = p.v = p.out = p.partial_m = p.partial_l = p.partial_o = p.page_table = at
        p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = 2, 4, 2, 100, 64, 2
        p.q_stride = p.o_stride = _lib.DecodeStrides(256, 64, 64)
        p.scale, p.dtype, p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = 0.1, 2, 16, 4, 8
        scales = change.pop("scales", at)
        for name, value in change.items():
            setattr(p, name, value)
        return lib.sca_launch_paged_attention_fp8(C.byref(p), scales, at, None, None)
    for change in (dict(q=None), dict(out=None), dict(partial_o=None), dict(page_table=None), dict(scales=None), dict(dtype=0), dict(num_splits=0),
                   dict(num_heads=3), dict(num_kv_heads=0), dict(batch=0), dict(block_size=0), dict(block_size=6), dict(max_blocks_per_seq=0),
                   dict(num_kv_blocks=0), dict(num_kv_blocks=1 << 28), dict(q=at + 8), dict(k=at + 4), dict(scales=at + 2), dict(out=at + 2),
                   dict(partial_o=at + 4), dict(head_dim=80), dict(q_stride=_lib.DecodeStrides(256, 60, 64)), dict(num_splits=1 << 20)):
        assert decode(**change) == 4, change
    assert lib.sca_launch_paged_attention_fp8(None, at, at, None, None) == 4

    def chunk(**change):
        p = _lib.FlashPagedParams()
        cu, lens = np.array(change.pop("cu", [0, 9]), np.int32), np.array(change.pop("lens", [20]), np.int32)
        p.q = p.out = p.k_pool = p.v_pool = p.page_table = p.workspace = at
        p.total_q, p.num_heads, p.num_kv_heads, p.head_dim, p.num_seqs = 9, 4, 2, 64, 1
        p.num_blocks, p.block_size, p.max_blocks_per_seq = 8, 16, 4
        p.cu_seqlens_q, p.seq_lens_kv, p.scale, p.causal, p.dtype_id, p.workspace_bytes = cu.ctypes.data, lens.ctypes.data, 0.1, 1, 2, 4096
        scales = change.pop("scales", at)
        for name, value in change.items():
            setattr(p, name, value)
        return lib.sca_launch_flash_paged_fp8(C.byref(p), scales, at, None)
    for change in (dict(scales=None), dict(scales=at + 8), dict(q=None), dict(page_table=None), dict(num_seqs=0), dict(cu=[0, 8]), dict(cu=[1, 9]),
                   dict(block_size=4), dict(block_size=128), dict(block_size=24), dict(num_blocks=0), dict(lens=[0]), dict(lens=[65]), dict(lens=[8]),
                   dict(dtype_id=0), dict(num_heads=3), dict(scale=0.0), dict(out=at + 8), dict(head_dim=80)):
        assert chunk(**change) == 4, change
    assert lib.sca_launch_flash_paged_fp8(None, at, at, None) == 4
