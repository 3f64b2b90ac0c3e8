"""The C ABI of the operators that norm and turn heads, on a host without a GPU: bad arguments are rejected before any launch."""

import ctypes

import pytest
import torch

from wavelet_amd import _lib
from wavelet_amd.plan import Heads

# fake device pointers: only where no GPU is visible, so that no call can reach a device
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device pointers: host-only test")

A = 1 << 12  # an aligned address


def _rotary(**kw):
    return _lib.WkvRotary(**{**dict(positions=A, axis_stride=0, axes=None, inv_freq=A, num_axes=1, rotary_dim=128,
                                    interleaved=0, inverse=0, scale=1.0, reserved=0), **kw})


def _norm(**kw):
    return _lib.WkvHeadNorm(**{**dict(q_weight=A, k_weight=A, q_weight_stride_h=0, k_weight_stride_h=0, weight_dtype=1,
                                      weight_offset=0.0, eps=1e-6, reserved=0), **kw})


def _rows_args(**kw):
    d = dict(dtype=1, q=A, qst=4096, qsh=128, qo=A, qot=4096, qoh=128, hq=32, k=A, kst=1024, ksh=128, ko=A, kot=1024,
             koh=128, hk=8, d=128, norm=_norm(), rotary=_rotary(), tokens=4, stream=None)
    assert not set(kw) - set(d)
    return list({**d, **kw}.values())


BAD_ROTARY = (dict(rotary_dim=0), dict(rotary_dim=130), dict(rotary_dim=7), dict(scale=float("inf")), dict(scale=float("nan")),
              dict(num_axes=0), dict(axis_stride=-1), dict(reserved=1), dict(positions=None), dict(positions=A + 4),
              dict(inv_freq=None), dict(inv_freq=A + 4), dict(axes=A + 2))
BAD_NORM = (dict(eps=0.0), dict(eps=-1.0), dict(eps=1e-40), dict(eps=float("nan")), dict(eps=float("inf")),
            dict(weight_offset=float("nan")), dict(weight_dtype=2), dict(weight_dtype=-1), dict(q_weight=A + 1),
            dict(k_weight_stride_h=-1), dict(reserved=1))
BAD_ROWS = (dict(dtype=3), dict(dtype=-1), dict(tokens=-1), dict(tokens=1 << 31), dict(hq=-1), dict(hk=65536), dict(d=0), dict(d=127),
            dict(d=514), dict(q=None), dict(qo=None), dict(k=None), dict(q=A + 1), dict(qst=-1), dict(koh=-1))


def test_rotary_axes():
    lib = _lib.load()

    def call(**kw):
        args = _rows_args(**kw)
        del args[16]  # the norm
        return lib.wkv_rotary_axes(*args)

    assert call(tokens=0) == _lib.WKV_OK
    for bad in BAD_ROWS:
        assert call(**bad) == _lib.WKV_ERR_INVALID, bad
    for bad in BAD_ROTARY:
        assert call(rotary=_rotary(**bad)) == _lib.WKV_ERR_INVALID, bad
    assert call(rotary=None) == _lib.WKV_ERR_INVALID


def test_norm_rotary():
    lib = _lib.load()
    assert lib.wkv_norm_rotary(*_rows_args(tokens=0)) == _lib.WKV_OK
    assert lib.wkv_norm_rotary(*_rows_args(tokens=0, rotary=None)) == _lib.WKV_OK
    assert lib.wkv_norm_rotary(*_rows_args(hq=0, hk=0)) == _lib.WKV_OK
    for bad in BAD_ROWS:
        assert lib.wkv_norm_rotary(*_rows_args(**bad)) == _lib.WKV_ERR_INVALID, bad
    for bad in BAD_ROTARY:
        assert lib.wkv_norm_rotary(*_rows_args(rotary=_rotary(**bad))) == _lib.WKV_ERR_INVALID, bad
    for bad in BAD_NORM:
        assert lib.wkv_norm_rotary(*_rows_args(norm=_norm(**bad))) == _lib.WKV_ERR_INVALID, bad
    assert lib.wkv_norm_rotary(*_rows_args(norm=None)) == _lib.WKV_ERR_INVALID
    # more workgroups than a launch can have
    assert lib.wkv_norm_rotary(*_rows_args(tokens=(1 << 31) - 1)) == _lib.WKV_ERR_INVALID
    assert "too many" in _lib.last_error()


def test_norm_rotary_backward():
    lib = _lib.load()
    size = lib.wkv_norm_rotary_workspace_size
    assert size(0, 4, 2, 64, 0, 0) == 0
    assert size(100, 4, 2, 64, 0, 0) > 0 and size(100, 4, 2, 64, 1, 1) >= size(100, 4, 2, 64, 0, 0)
    for bad in ((-1, 4, 2, 64, 0, 0), (1 << 31, 4, 2, 64, 0, 0), (1, -1, 2, 64, 0, 0), (1, 4, 65536, 64, 0, 0),
                (1, 4, 2, 0, 0, 0), (1, 4, 2, 514, 0, 0)):
        assert size(*bad) == -1, bad

    def call(**kw):
        d = dict(dtype=1, q=A, qst=4096, qsh=128, gq=A, gqt=4096, gqh=128, dq=A, dqt=4096, dqh=128, hq=32, k=A, kst=1024, ksh=128,
                 gk=A, gkt=1024, gkh=128, dk=A, dkt=1024, dkh=128, hk=8, d=128, norm=_norm(), rotary=_rotary(), dqw=A, dkw=A,
                 tokens=4, ws=A, bytes=1 << 20, stream=None)
        assert not set(kw) - set(d)
        return lib.wkv_norm_rotary_backward(*{**d, **kw}.values())

    for bad in (dict(dtype=5), dict(q=None), dict(gq=None), dict(gk=A + 1), dict(dq=A + 1), dict(gqt=-1), dict(dkh=-1), dict(norm=None),
                dict(d=126 + 1), dict(ws=None), dict(ws=A + 8), dict(bytes=16), dict(tokens=-1),
                dict(norm=_norm(q_weight=None)), dict(norm=_norm(k_weight=None)), dict(hq=0)):
        assert call(**bad) == _lib.WKV_ERR_INVALID, bad
    for bad in BAD_ROTARY:
        assert call(rotary=_rotary(**bad)) == _lib.WKV_ERR_INVALID, bad
    for bad in BAD_NORM:
        assert call(norm=_norm(**bad)) == _lib.WKV_ERR_INVALID, bad


def test_rotary_append():
    lib = _lib.load()

    def cache(**kw):
        return _lib.WkvCache(**{**dict(k=A, v=A, k_scale=None, v_scale=None, num_blocks=4, block_size=16, num_kv_heads=8,
                                       head_dim=128, kv_dtype=0, flags=0, reserved=0), **kw})

    def call(**kw):
        d = dict(cache=ctypes.byref(cache()), key=A, kst=1024, ksh=128, value=A, vst=1024, vsh=128, slots=A, q=A, qst=4096, qsh=128,
                 qo=A, qot=4096, qoh=128, hq=32, norm=_norm(), rotary=_rotary(), tokens=4, stream=None)
        assert not set(kw) - set(d)
        return lib.wkv_rotary_append(*{**d, **kw}.values())

    assert call(tokens=0) == _lib.WKV_OK
    for bad in (dict(cache=None), dict(cache=ctypes.byref(cache(k=None))), dict(cache=ctypes.byref(cache(block_size=24))),
                dict(cache=ctypes.byref(cache(kv_dtype=1))), dict(cache=ctypes.byref(cache(num_blocks=1 << 31))),
                dict(cache=ctypes.byref(cache(num_kv_heads=65536))),
                dict(key=None), dict(key=A + 8), dict(kst=1023), dict(vsh=-8), dict(value=A + 2), dict(slots=None),
                dict(slots=A + 4), dict(q=None), dict(q=A + 1), dict(qo=None), dict(qst=-1), dict(hq=-1), dict(hq=65536),
                dict(norm=None, rotary=None), dict(tokens=-1), dict(tokens=1 << 31), dict(tokens=(1 << 31) - 1)):
        assert call(**bad) == _lib.WKV_ERR_INVALID, bad
    assert call(cache=ctypes.byref(cache(head_dim=96))) == _lib.WKV_ERR_UNSUPPORTED
    for bad in BAD_ROTARY:
        assert call(rotary=_rotary(**bad)) == _lib.WKV_ERR_INVALID, bad
    for bad in BAD_NORM:
        assert call(norm=_norm(**bad)) == _lib.WKV_ERR_INVALID, bad


def test_mla_rotary_append():
    lib = _lib.load()

    def cache(**kw):
        return _lib.WkvMlaCache(**{**dict(latent=A, num_blocks=4, block_size=64, kv_lora_rank=512, rope_dim=64), **kw})

    def call(**kw):
        d = dict(cache=ctypes.byref(cache()), kvc=A, kvst=576, kpe=A, kpst=576, slots=A, q=A, qst=8192, qsh=64, qo=A, qot=8192,
                 qoh=64, heads=128, norm=_norm(q_weight=None), rotary=_rotary(rotary_dim=64), tokens=4, stream=None)
        assert not set(kw) - set(d)
        return lib.wkv_mla_rotary_append(*{**d, **kw}.values())

    assert call(tokens=0) == _lib.WKV_OK
    for bad in (dict(cache=None), dict(cache=ctypes.byref(cache(latent=None))), dict(cache=ctypes.byref(cache(rope_dim=0))),
                dict(cache=ctypes.byref(cache(rope_dim=520))), dict(kvc=None), dict(kvc=A + 8), dict(kvst=575), dict(kpe=A + 2),
                dict(kpst=-8), dict(slots=None), dict(q=None), dict(qo=A + 1), dict(qoh=-1), dict(heads=-1), dict(heads=65536),
                dict(rotary=None), dict(norm=_norm()), dict(norm=_norm(q_weight=None, k_weight=A + 8)), dict(tokens=-1)):
        assert call(**bad) == _lib.WKV_ERR_INVALID, bad
    for bad in BAD_NORM:
        if "q_weight" not in bad:
            assert call(norm=_norm(**{"q_weight": None, **bad})) == _lib.WKV_ERR_INVALID, bad
    # rows of 16-byte pieces only from rope_dim 136 on, where a lane would hold more than one unit
    assert call(cache=ctypes.byref(cache(rope_dim=256)), q=A + 2, rotary=_rotary(rotary_dim=256)) == _lib.WKV_ERR_UNSUPPORTED


def test_mla_norm_weight_is_one_row():
    """A weight for each head has no meaning for an entry: the kernel would take the first row for all."""
    lib = _lib.load()
    cache = _lib.WkvMlaCache(latent=A, num_blocks=4, block_size=64, kv_lora_rank=512, rope_dim=64)

    def call(**norm):
        return lib.wkv_mla_rotary_append(ctypes.byref(cache), A, 576, A, 576, A, A, 8192, 64, A, 8192, 64, 128,
                                         _norm(q_weight=None, **norm), _rotary(rotary_dim=64), 0, None)

    assert call() == _lib.WKV_OK
    assert call(k_weight_stride_h=512) == _lib.WKV_ERR_INVALID
    assert "one row" in _lib.last_error()


def test_a_plan_s_entry_weights():
    """What MLADecodeStep checks of a layer's norm when it is built (as mla_rotary_append does for a call)."""
    entries = torch.zeros((3, 512), dtype=torch.bfloat16)
    good = torch.ones(512, dtype=torch.bfloat16)
    off = torch.ones(520, dtype=torch.bfloat16)[1:513]
    norm = Heads(eps=1e-6, k_weight=[good]).entry_norm(0, 1, entries)
    assert norm.k_weight == good.data_ptr() and norm.k_weight_stride_h == 0
    assert Heads(eps=1e-6).entry_norm(0, 1, entries).k_weight is None
    assert Heads(eps=1e-6, k_weight=[None, good]).entry_norm(0, 2, entries).k_weight is None
    assert Heads().entry_norm(0, 1, entries) is None
    for bad in (torch.ones((512, 512), dtype=torch.bfloat16), torch.ones((1, 512), dtype=torch.bfloat16), off, good[:64],
                good.half()):
        with pytest.raises(ValueError):
            Heads(eps=1e-6, k_weight=[bad]).entry_norm(0, 1, entries)
    for bad in (Heads(k_weight=[good]), Heads(eps=1e-6, k_weight=[good, good]), Heads(eps=1e-6, q_weight=[good])):
        with pytest.raises(ValueError):
            bad.entry_norm(0, 1, entries)


def test_turn_heads():
    lib = _lib.load()

    def call(**kw):
        args = _rows_args(**kw)
        del args[16]  # the norm
        return lib.wkv_turn_heads(*args)

    assert call(tokens=0) == _lib.WKV_OK and call(hq=0, hk=0) == _lib.WKV_OK
    for bad in BAD_ROWS:
        assert call(**bad) == _lib.WKV_ERR_INVALID, bad
    for bad in BAD_ROTARY:
        assert call(rotary=_rotary(**bad)) == _lib.WKV_ERR_INVALID, bad
    assert call(rotary=None) == _lib.WKV_ERR_INVALID
