"""CPU tests of the 4-bit cache and of shaped attention: sizes, refusals of a
handle without a device, the layout's inverse and the 64-bit restatement."""
import ctypes as C

import numpy as np
import pytest

import _attn64 as A
from langtrain_studio_b200 import _native as N
from langtrain_studio_b200.kv import KvCache, KvError, unswizzle_pool_q4


def test_pool_bytes():
    kv = KvCache(3, 2, 128, 16 * 10, max_seqs=2, device=-1, kv_format="q4_0")
    assert kv.bytes() == 3 * 10 * 2 * 18 * 128
    assert kv.capacity() == 160


def test_unknown_formats_are_refused(native):
    with pytest.raises(ValueError):
        KvCache(1, 1, 64, 16, device=-1, kv_format="q3_0")
    cfg = N.lt_kv_config(n_layers=1, n_kv_heads=1, head_dim=64, n_heads=1, n_tokens=16, max_seqs=1, max_batch=1,
                         device=-1, kv_format=3)
    h = C.c_void_p()
    assert native.lt_kv_create(C.byref(cfg), C.byref(h)) == N.LT_E_ARG


def test_calls_without_a_device_are_refused(native):
    kv = KvCache(1, 1, 64, 64, n_heads=4, max_seqs=2, device=-1, kv_format="q4_0")
    b, s = kv.append_batch([0, 0], [0, 1])
    buf = np.zeros(512, np.float32)
    p = buf.ctypes.data
    seq, pos = np.zeros(1, np.uint32), np.zeros(1, np.uint32)
    score = N.lt_kv_score(softcap=1.0)
    args = (kv._h, 0, p, N.LT_F32, seq.ctypes.data, pos.ctypes.data, 1)
    assert native.lt_kv_attend_shaped(*args, C.byref(score), p, N.LT_F32, 1.0, None) == N.LT_E_ARG
    assert native.lt_kv_attend_shaped(*args, None, p, N.LT_F32, 1.0, None) == N.LT_E_ARG
    assert native.lt_kv_attend_shaped(kv._h, 0, p, 7, *args[4:], C.byref(score), p, N.LT_F32, 1.0, None) == N.LT_E_ARG
    assert native.lt_kv_read(kv._h, 0, b.ctypes.data, s.ctypes.data, 2, p, p, N.LT_F32, None) == N.LT_E_ARG
    assert native.lt_kv_read(kv._h, 0, b.ctypes.data, s.ctypes.data, 2, p, p, 9, None) == N.LT_E_ARG
    assert native.lt_kv_write(kv._h, 0, b.ctypes.data, s.ctypes.data, 2, p, p, N.LT_F32, None) == N.LT_E_ARG
    assert native.lt_kv_attend_shaped(None, *args[1:], C.byref(score), p, N.LT_F32, 1.0, None) == N.LT_E_ARG
    assert native.lt_kv_read(None, 0, b.ctypes.data, s.ctypes.data, 2, p, p, N.LT_F32, None) == N.LT_E_ARG


def test_noalloc_refuses_the_format(native):
    buf = np.zeros(4096, np.uint8)
    p = buf.ctypes.data + (-buf.ctypes.data % 16)
    seq, pos = np.zeros(1, np.uint32), np.zeros(1, np.uint32)
    rc = native.lt_paged_attend_noalloc(p, N.LT_KV_Q4_0, 4, 1, 64, 1, p, 2, 4, seq.ctypes.data, pos.ctypes.data, 1, p,
                                        N.LT_F32, p, N.LT_F32, 1.0, None)
    assert rc == N.LT_E_UNSUPPORTED


@pytest.mark.parametrize("hd", [64, 128])
def test_layout_is_a_permutation(hd):
    """Every byte of a tile is one slot's pair of codes or half a scale: the
    inverse finds each nibble once."""
    rng = np.random.default_rng(0)
    raw = rng.integers(0, 256, (2, 3, 18 * hd), dtype=np.uint8)
    kc, vc, kd, vd = unswizzle_pool_q4(raw, hd)
    assert kc.shape == (2, 16, 3 * hd) and kd.shape == (2, 16, 3 * hd // 32)
    for codes, part in ((kc, raw[:, :, : 8 * hd]), (vc, raw[:, :, 8 * hd: 16 * hd])):
        both = np.concatenate([part & 15, part >> 4], -1)
        for b in range(2):
            for h in range(3):
                one = codes[b, :, h * hd:(h + 1) * hd].reshape(-1)
                assert np.array_equal(np.bincount(one, minlength=16), np.bincount(both[b, h], minlength=16))
    # each byte changes codes of one slot alone, two dims 8 apart
    flat = np.zeros((1, 1, 18 * hd), np.uint8)
    for byte in range(16 * hd):
        flat[:] = 0
        flat[0, 0, byte] = 0xFF
        k, v, _, _ = unswizzle_pool_q4(flat, hd)
        hit = np.argwhere((k if byte < 8 * hd else v)[0] == 15)
        assert len(hit) == 2 and hit[0, 0] == hit[1, 0] and hit[1, 1] - hit[0, 1] == 8
    scales = np.arange(2 * 16 * hd // 32, dtype=np.uint16)
    flat[:] = 0
    flat[0, 0, 16 * hd:] = scales.view(np.uint8)
    _, _, kd, vd = unswizzle_pool_q4(flat, hd)
    assert np.array_equal(np.sort(np.concatenate([kd.reshape(-1), vd.reshape(-1)])), scales)


def test_values_are_f16s():
    """(code - 8) * d never needs more than f16 holds, over every scale."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((4000, 32)) * np.exp2(rng.uniform(-26, 15, (4000, 1)))
    v = A.value4(*A.quant4(x))
    assert np.array_equal(v.astype(np.float16).astype(np.float64), v)
    ok = (np.abs(x).max(-1) > 2.0 ** -10) & (np.abs(x).max(-1) < 8 * A.MAX_SCALE)
    # Values are their own nearest values where f16 holds all 8 bits of the
    # scale, i.e. max|x| / 8 >= 2^-17.  Below, a scale is a few multiples of
    # 2^-24: max|x| = 4.4 * 2^-24 has d = 2^-24 and the largest value 4 d, whose
    # own scale is 2^-25, a tie that f16 rounds to 0.
    code, d = A.quant4(v[ok])
    assert np.array_equal(A.value4(code, d), v[ok])
    code, d = A.quant4(x)
    err, step = np.abs(v - x)[ok], np.abs(d)[ok]
    # half a step, or what is cut off beyond +7 steps
    assert (err <= np.maximum(step / 2, np.abs(x[ok]) - 7 * step) * (1 + 2 ** -8)).all()
