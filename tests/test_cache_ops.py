"""Cache-maintenance operators on CPU: refusals of the C entry points before any CUDA call, of the
tensor wrappers, the rotary scalings, and the 64-bit restatement against the quantizer."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from kvssd_b200 import CacheSpec, DeviceKVCache, RotaryEmbedding, _native, ops
from kvssd_b200.quant import dequantize_tensor, quantize_tensor
from oracle import cache_oracle as orc

DUMMY = ctypes.c_void_p(16)


def _refused(status, text, code=_native.ERR_INVALID_ARGUMENT):
    assert status == code
    assert text in _native.library().kvssd_b200_last_error()


def _rotary(**kw):
    a = dict(x=DUMMY, dtype=1, xt=128, xh=128, tokens=1, heads=1, d=128, pos=DUMMY, pos64=0,
             freq=DUMMY, pairs=64, inter=0, mag=1.0, out=DUMMY, ot=128, oh=128, stream=None) | kw
    return _native.library().kvssd_b200_rotary(*a.values())


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=3), b"element type"), (dict(tokens=-1), b"negative"), (dict(d=0), b"positive"),
    (dict(x=None), b"NULL"), (dict(out=None), b"NULL"), (dict(pos=None), b"NULL"),
    (dict(freq=None), b"NULL"), (dict(pairs=0), b"pairs"), (dict(pairs=65), b"pairs"),
])
def test_rotary_refusals(kw, text):
    _refused(_rotary(**kw), text)


def test_rotary_unsupported_and_empty():
    _refused(_rotary(d=258), b"head_dim", _native.ERR_UNSUPPORTED)
    _refused(_rotary(heads=1 << 18), b"2^24", _native.ERR_UNSUPPORTED)
    assert _rotary(tokens=0) == 0 and _rotary(heads=0, x=None) == 0


def _append(**kw):
    a = dict(k=DUMMY, v=DUMMY, dtype=1, kt=64, kh=64, vt=64, vh=64, tokens=1, slots=DUMMY, s64=0,
             pos=DUMMY, pos64=0, freq=DUMMY, pairs=32, inter=0, mag=1.0, pk=DUMMY, pv=DUMMY,
             sk=DUMMY, sv=DUMMY, valid=None, n_pool=1, bt=8, kvh=1, d=64, bits=4, group=32,
             kval=None, vval=None, status=None, stream=None) | kw
    return _native.library().kvssd_b200_append(*a.values())


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=3), b"element type"), (dict(tokens=-1), b"negative"), (dict(bits=3), b"bits"),
    (dict(n_pool=0), b"positive"), (dict(group=48), b"divide"), (dict(bits=2, group=2), b"pack-aligned"),
    (dict(k=None), b"NULL"), (dict(v=None), b"NULL"), (dict(slots=None), b"NULL"),
    (dict(pk=None), b"NULL"), (dict(sv=None), b"NULL"), (dict(pos=None), b"positions"),
    (dict(pairs=33), b"pairs"), (dict(kval=DUMMY), b"both"), (dict(vval=DUMMY), b"both"),
])
def test_append_refusals(kw, text):
    _refused(_append(**kw), text)


def test_append_unsupported_and_empty():
    _refused(_append(d=512, group=32), b"head_dim", _native.ERR_UNSUPPORTED)
    assert _append(tokens=0, k=None) == 0


def test_append_of_too_many_tokens():
    _refused(_append(tokens=2**31 - 1), b"2^31", _native.ERR_UNSUPPORTED)


def _weights(**kw):
    a = dict(q=DUMMY, dtype=1, queries=1, pk=DUMMY, sk=DUMMY, valid=DUMMY, table=None, visible=None,
             n_pool=2, n_sel=2, bt=8, qh=4, kvh=2, d=64, bits=4, group=32, scale=0.125, given=1,
             lse=DUMMY, prev=None, pstride=0, out=DUMMY, ostride=16, scratch=None, bytes=0,
             status=None, stream=None) | kw
    return _native.library().kvssd_b200_attention_weights(*a.values())


@pytest.mark.parametrize("kw, text", [
    (dict(bits=1), b"bits"), (dict(n_sel=0), b"at least one block"), (dict(n_sel=3), b"pool holds"),
    (dict(queries=0), b"positive"), (dict(qh=3), b"divisible"), (dict(dtype=4), b"dtype"),
    (dict(q=None), b"NULL"), (dict(lse=None), b"NULL"), (dict(out=None), b"NULL"),
    (dict(valid=None), b"NULL"), (dict(group=24), b"divide"),
])
def test_weights_refusals(kw, text):
    _refused(_weights(**kw), text)


def test_weights_workspace_and_limits():
    _refused(_weights(given=0), b"scratch", _native.ERR_WORKSPACE)
    _refused(_weights(d=512), b"head_dim", _native.ERR_UNSUPPORTED)
    _refused(_weights(n_sel=1 << 28, n_pool=1 << 28), b"2^31", _native.ERR_UNSUPPORTED)
    need = ctypes.c_size_t()
    lib = _native.library()
    assert lib.kvssd_b200_attention_weights_scratch_size(1, 2, 8, 4, 2, 64, 4, 32, None) == 1
    _refused(lib.kvssd_b200_attention_weights_scratch_size(0, 2, 8, 4, 2, 64, 4, 32,
                                                           ctypes.byref(need)), b"positive")


def _evict(**kw):
    a = dict(w=DUMMY, ws=16, pos=DUMMY, ps=16, n=16, keep=8, sink=0, recent=1 << 40, shared=0,
             nw=DUMMY, np=DUMMY, columns=16, pk=DUMMY, pv=DUMMY, sk=DUMMY, sv=DUMMY, valid=DUMMY,
             table=None, n_pool=2, n_sel=2, bt=8, kvh=2, pd=32, groups=2, scratch=DUMMY,
             bytes=1 << 20, status=None, stream=None) | kw
    return _native.library().kvssd_b200_evict(*a.values())


@pytest.mark.parametrize("kw, text", [
    (dict(n=0), b"n_tokens"), (dict(n=17), b"n_tokens"), (dict(keep=0), b"keep"),
    (dict(keep=17), b"keep"), (dict(columns=15), b"columns"), (dict(n_sel=3), b"pool holds"),
    (dict(pd=0), b"positive"), (dict(w=None), b"NULL"), (dict(nw=None), b"NULL"),
    (dict(valid=None), b"NULL"), (dict(sk=None), b"NULL"),
])
def test_evict_refusals(kw, text):
    _refused(_evict(**kw), text)


def test_evict_workspace():
    _refused(_evict(scratch=None), b"scratch", _native.ERR_WORKSPACE)
    _refused(_evict(bytes=4 * 2 * 17 - 1), b"scratch", _native.ERR_WORKSPACE)
    need = ctypes.c_size_t()
    assert _native.library().kvssd_b200_evict_scratch_size(16, 8, 2, 0, ctypes.byref(need)) == 0
    assert need.value == 4 * 2 * 17
    _refused(_native.library().kvssd_b200_evict_scratch_size(16, 17, 2, 0, ctypes.byref(need)), b"sizes")


def test_wrappers_have_no_cpu_path():
    x = torch.zeros(1, 1, 8)
    i = torch.zeros(1, dtype=torch.int64)
    f = torch.zeros(4, dtype=torch.float64)
    pool = [torch.zeros(1, 8, 1, 4, dtype=torch.uint8)] * 2 + [torch.zeros(1, 8, 1, 1).half()] * 2
    valid = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.rotary(x, i, f), lambda: ops.append(x, x, i, *pool, 4, 8),
                 lambda: ops.attention_weights(x, pool[0], pool[2], valid, 4, 8, 1.0),
                 lambda: ops.evict(torch.zeros(1, 8), torch.zeros(1, 8, dtype=torch.int32), 8, 4,
                                   *pool, valid)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="CUDA device"):
        DeviceKVCache(CacheSpec(1, 1, 8, 8, 4, 8), 1, "cpu")


def test_rotary_embedding_scalings():
    plain = RotaryEmbedding(128).frequencies()
    assert plain.dtype == torch.float64 and plain.shape == (64,)
    assert plain[0] == 1.0 and math.isclose(plain[-1], 10000.0 ** (-126 / 128))
    torch.testing.assert_close(RotaryEmbedding(128, scaling="linear", factor=4.0).frequencies(), plain / 4)
    ntk = RotaryEmbedding(128, scaling="ntk", factor=4.0).frequencies()
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 4, rel_tol=1e-12)
    smooth = RotaryEmbedding(128, scaling="smooth", factor=8.0, original_length=8192).frequencies()
    turns = 8192 * plain / (2 * math.pi)
    assert torch.equal(smooth[turns >= 4], plain[turns >= 4])
    torch.testing.assert_close(smooth[turns <= 1], plain[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and ((smooth < plain) & (smooth > plain / 8))[mid].all()
    yarn = RotaryEmbedding(128, scaling="yarn", factor=8.0, original_length=8192)
    f = yarn.frequencies()
    assert math.isclose(yarn.magnitude, 0.1 * math.log(8.0) + 1.0)
    assert torch.equal(f[turns > 40], plain[turns > 40])
    torch.testing.assert_close(f[turns < 0.8], plain[turns < 0.8] / 8)
    assert RotaryEmbedding(128, rotary_dim=64).frequencies().shape == (32,)


@pytest.mark.parametrize("kw, text", [
    (dict(rotary_dim=130), "rotary_dim"), (dict(rotary_dim=7), "rotary_dim"),
    (dict(rotary_dim=0), "rotary_dim"), (dict(scaling="other"), "unknown scaling"),
    (dict(base=1.0), "base"), (dict(scaling="linear", factor=0.5), "factor"),
    (dict(scaling="yarn"), "original_length"), (dict(scaling="ntk", rotary_dim=2), "above 2"),
    (dict(scaling="smooth", original_length=64, low=8.0), "ascending"),
])
def test_rotary_embedding_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        RotaryEmbedding(128, **kw)


@pytest.mark.parametrize("bits, group", [(2, 16), (4, 32), (4, 48)])
def test_oracle_quantizer_is_the_formats(bits, group):
    x = torch.randn(5, 3, 2 * group, generator=torch.Generator().manual_seed(group)) * 3
    q = quantize_tensor(x, bits, group)
    codes, scales = orc.quantize(x.numpy(), bits, group)
    np.testing.assert_array_equal(orc.pack(codes, bits), q.packed.numpy())
    np.testing.assert_array_equal(scales, q.scales.numpy())
    np.testing.assert_array_equal(orc.unpack(q.packed.numpy(), bits), codes)
    np.testing.assert_array_equal(orc.values(codes, scales, bits, group).astype(np.float32),
                                  dequantize_tensor(q).numpy())
