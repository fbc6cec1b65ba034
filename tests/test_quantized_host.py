"""8-bit pool and block tables on the host: the C ABI's refusals, which come before any CUDA call,
the bindings' refusal of CPU tensors, and the plain forms against themselves."""
import ctypes

import numpy as np
import pytest
import torch

import shardserve_b200 as sb
from oracle import quantized as oq
from shardserve_b200 import _native

S = _native.strides


def attend(**over):
    a = dict(q=1, qs=(0, 0, 1), kp=1, ks=(0, 0, 0, 1), vp=1, vs=(0, 0, 0, 1), fmt=0, sc=1, ss=(0, 0, 1),
             bt=1, bts=(1, 1), rows=1, cols=1, seq=1, pos=1, out=1, os=(0, 0, 1), T=1, H=8, KVH=1, D=128,
             N=1, scale=0.1, ws=1, wsb=1 << 30)
    a.update(over)
    return _native.lib().ss_ragged_paged_attention_q8(
        a["q"], S(a["qs"]), a["kp"], S(a["ks"]), a["vp"], S(a["vs"]), a["fmt"], a["sc"], S(a["ss"]),
        a["bt"], S(a["bts"]), a["rows"], a["cols"], 0, a["seq"], 0, a["pos"], 1, a["out"], S(a["os"]),
        a["T"], a["H"], a["KVH"], a["D"], a["N"], a["scale"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("over,needle", [
    (dict(D=96), "64 or 128"), (dict(fmt=2), "code_format"), (dict(T=0), "empty"),
    (dict(T=1 << 31), "2^31"), (dict(H=6, KVH=4), "divisible"), (dict(KVH=0), "positive"),
    (dict(N=0), "positive"), (dict(N=1 << 31), "2^31"), (dict(rows=0), "block_tables"),
    (dict(cols=1 << 27), "columns"), (dict(q=None), "null"), (dict(kp=None), "null"),
    (dict(sc=None), "null"), (dict(out=None), "null"), (dict(scale=float("inf")), "finite"),
    (dict(ks=(-1, 0, 0, 1)), "negative"), (dict(ss=(0, -1, 1)), "negative"), (dict(os=(0, -1, 1)), "negative")])
def test_attention_refusals(over, needle):
    assert attend(**over) == _native.SS_ERR_INVALID
    assert needle in _native.last_error()


def test_attention_wants_a_workspace():
    assert attend(ws=None) == _native.SS_ERR_WORKSPACE
    need = ctypes.c_size_t(0)
    lib = _native.lib()
    assert lib.ss_q8_workspace_bytes(0, 16, 2, 128, ctypes.byref(need)) == 0 and need.value > 1 << 20
    assert lib.ss_q8_workspace_bytes(0, 16, 2, 96, ctypes.byref(need)) == _native.SS_ERR_INVALID
    assert lib.ss_q8_workspace_bytes(0, 15, 2, 64, ctypes.byref(need)) == _native.SS_ERR_INVALID
    assert lib.ss_q8_workspace_bytes(0, 16, 2, 64, None) == _native.SS_ERR_INVALID


def test_append_and_read_refusals():
    lib = _native.lib()

    def append(k=1, fmt=0, T=4, N=2, KVH=1, D=64, ks=(0, 0, 1), slots=1, sc=1):
        return lib.ss_kv_append_q8(k, S(ks), 1, S((0, 0, 1)), 1, S((0, 0, 0, 1)), 1, S((0, 0, 0, 1)), fmt,
                                   sc, S((0, 0, 1)), slots, 1, T, N, KVH, D, None, None)

    def read(T=4, out=1, D=64, os=(0, 0, 1)):
        return lib.ss_kv_read_q8(1, S((0, 0, 0, 1)), 1, S((0, 0, 0, 1)), 0, 1, S((0, 0, 1)), 1, 1, out, S(os),
                                 1, S((0, 0, 1)), T, 2, 1, D, None, None)

    assert append(T=0) == 0 and read(T=0) == 0
    for bad in (dict(k=None), dict(fmt=-1), dict(T=-1), dict(N=0), dict(KVH=0), dict(D=32),
                dict(ks=(-1, 0, 1)), dict(slots=None), dict(sc=None)):
        assert append(**bad) == _native.SS_ERR_INVALID, bad
    for bad in (dict(T=-1), dict(out=None), dict(D=100), dict(os=(0, -2, 1))):
        assert read(**bad) == _native.SS_ERR_INVALID, bad


def test_block_tables_refusals():
    def tables(rows=2, cols=3, T=4, F=5, cached=1, bt=1, free=1, head=1, seqs=1, last=1, ws=1, bts=(3, 1)):
        return _native.lib().ss_build_block_tables(cached, 0, 1, 0, bt, S(bts), rows, cols, 0, free, 0, F, head,
                                                   T, seqs, 1, 1, last, 1, 1, ws, None)

    for bad in (dict(rows=-1), dict(T=-1), dict(F=-1), dict(rows=12289), dict(cols=0), dict(T=1 << 31),
                dict(cached=None), dict(bt=None), dict(free=None), dict(head=None), dict(seqs=None),
                dict(last=None), dict(ws=None), dict(bts=(-3, 1))):
        assert tables(**bad) == _native.SS_ERR_INVALID, bad


def test_cpu_tensors_are_refused():
    k = torch.zeros(2, 16, 1, 64, dtype=torch.int8)
    s = torch.zeros(2, 1, 2)
    i = torch.zeros(3, dtype=torch.int32)
    x = torch.zeros(3, 1, 64).bfloat16()
    for call in (lambda: sb.kv_append_q8(k, k, s, x, x, i), lambda: sb.kv_read_q8(k, k, s, i),
                 lambda: sb.ragged_attention_q8(x, k, k, s, i[None], i, i, 0.1),
                 lambda: sb.build_block_tables(i, i, i[:, None], i, i[:1], 3)):
        with pytest.raises(sb.KernelUnsupported):
            call()


def test_plain_forms():
    """The plain attention is softmax, and the plain tables hand out each page once."""
    rng = np.random.RandomState(0)
    k, v = rng.randint(-127, 128, (4, 16, 2, 8)).astype(float), rng.randint(-127, 128, (4, 16, 2, 8)).astype(float)
    s = rng.rand(4, 2, 2) / 50
    q = rng.randn(1, 4, 8)
    out, _ = oq.attention(q, k, v, s, np.array([[2, 0]]), [0], [19], 0.3)
    kk = np.concatenate([k[2] * s[2, :, 0][:, None], k[0] * s[0, :, 0][:, None]])[:20]
    vv = np.concatenate([v[2] * s[2, :, 1][:, None], v[0] * s[0, :, 1][:, None]])[:20]
    for h in range(4):
        x = np.exp(kk[:, h // 2] @ q[0, h] * 0.3)
        assert np.allclose(out[0, h], x @ vv[:, h // 2] / x.sum(), rtol=1e-12)
    got = oq.block_tables([0, 16, 31], [17, 1, 2], np.zeros((3, 3), int), np.arange(10, 20), 1, 20)
    assert got["tables"].tolist() == [[11, 12, 0], [0, 13, 0], [0, 0, 14]]
    assert got["slots"].tolist()[:17] == list(range(176, 192)) + [192]
    assert got["last"].tolist() == [16, 17, 19] and got["free_head"].tolist() == [5]
    new, written = oq.append_scales(np.array([[3.0], [1.0]]), np.array([[[254.0]], [[-127.0]]]), [5, 16], 127)
    assert new.tolist() == [[3.0], [1.0]] and written == {0: {5: 0}, 1: {0: 1}}
