"""What the calls on a drafted cache refuse, without a device: every message comes before anything is launched."""
import ctypes

import pytest
import torch


def _f16(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _attention(**other):
    a = dict(q=_f16(2, 3, 4, 64), k_cache=_f16(2, 2, 20, 64), v_cache=_f16(2, 2, 20, 64), lengths=_i32(2))
    return {**a, **other}


@pytest.mark.parametrize("other,message", [
    (dict(), "must be CUDA"),
    (dict(q=_f16(2, 3, 4, 128)), "q must be"),
    (dict(q=_f16(1, 3, 4, 64)), "q must be"),
    (dict(q=_f16(2, 3, 4, 64).bfloat16()), "caches' type"),
    (dict(q=_f16(2, 65, 4, 64)), "1 .. 64 tokens"),
    (dict(q=_f16(2, 0, 4, 64)), "1 .. 64 tokens"),
    (dict(q=_f16(2, 3, 3, 64)), "multiple of the kv heads"),
    (dict(q=_f16(2, 3, 64, 4).transpose(2, 3)), "last dimension of q"),
    (dict(q=_f16(2, 3, 4, 68)[..., :64]), "multiples of 8"),
    (dict(k_cache=_f16(2, 2, 20, 96), v_cache=_f16(2, 2, 20, 96), q=_f16(2, 3, 4, 96)), "64 or 128"),
    (dict(v_cache=_f16(2, 2, 21, 64)), "same shape"),
    (dict(k_cache=_f16(2, 2, 20, 64).float(), v_cache=_f16(2, 2, 20, 64).float()), "float16 or bfloat16"),
    (dict(k_cache=_f16(2, 2, 40, 64)[:, :, :20]), "contiguous"),
    (dict(lengths=_i32(3)), "lengths"),
    (dict(lengths=_i32(2).long()), "lengths"),
    (dict(tree=_i32(3)), "tree"),
    (dict(tree=torch.zeros(4, dtype=torch.int64)), "tree"),
    (dict(tree=torch.zeros(3, 2, dtype=torch.int64).t()), "tree"),
    (dict(weights=_f16(2, 2, 20)), "weights"),
    (dict(weights=torch.zeros(2, 4, 20)), "weights"),
])
def test_tree_attention_refuses(other, message):
    from flh_b200 import _CUDA
    with pytest.raises(RuntimeError, match=message):
        _CUDA.tree_attention(**_attention(**other))


@pytest.mark.parametrize("other,message", [
    (dict(), "must be CUDA"),
    (dict(qkv=_f16(6, 7 * 64)), "qkv"),
    (dict(qkv=_f16(6, 8 * 64).bfloat16()), "qkv"),
    (dict(positions=_i32(2, 3).long()), "positions"),
    (dict(positions=_i32(6)), "positions"),
    (dict(cos=torch.zeros(9, 64)), "cos"),
    (dict(sin=torch.zeros(8, 32)), "sin"),
    (dict(lengths=_i32(1)), "lengths"),
    (dict(v_cache=_f16(2, 2, 20, 64).transpose(1, 2)), "same shape"),
])
def test_rope_kv_at_refuses(other, message):
    from flh_b200 import _CUDA
    a = dict(qkv=_f16(6, 8 * 64), cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), positions=_i32(2, 3), lengths=_i32(2), k_cache=_f16(2, 2, 20, 64), v_cache=_f16(2, 2, 20, 64), nh=4)
    with pytest.raises(RuntimeError, match=message):
        _CUDA.rope_kv_at(**{**a, **other})


@pytest.mark.parametrize("other,message", [
    (dict(), "must be CUDA"),
    (dict(k_caches=[], v_caches=[]), "layers"),
    (dict(v_caches=[_f16(2, 2, 20, 64)]), "layers"),
    (dict(k_caches=[_f16(2, 2, 20, 64)] * 129, v_caches=[_f16(2, 2, 20, 64)] * 129), "layers"),
    (dict(v_caches=[_f16(2, 2, 20, 64), _f16(2, 2, 19, 64)]), "alike"),
    (dict(k_caches=[_f16(2, 2, 20, 60)] * 2, v_caches=[_f16(2, 2, 20, 60)] * 2), "multiple of 8"),
    (dict(weights=[torch.zeros(2, 2, 19)] * 2), "weights"),
    (dict(weights=[torch.zeros(2, 2, 20)]), "layers"),
    (dict(drafted=65), "drafted"),
    (dict(drafted=2), "path"),
    (dict(path=_i32(2, 3).long()), "path"),
    (dict(accepted=_i32(3)), "accepted"),
])
def test_cache_accept_refuses(other, message):
    from flh_b200 import _CUDA
    a = dict(k_caches=[_f16(2, 2, 20, 64)] * 2, v_caches=[_f16(2, 2, 20, 64)] * 2, lengths=_i32(2), path=_i32(2, 3), accepted=_i32(2), drafted=5)
    with pytest.raises(RuntimeError, match=message):
        _CUDA.cache_accept(**{**a, **other})


@pytest.mark.parametrize("other,message", [
    (dict(), "must be CUDA"),
    (dict(keep=0), "keep"),
    (dict(keep=21), "keep"),
    (dict(recent=8), "recent"),
    (dict(recent=-1), "recent"),
    (dict(weights=None), "weights"),
    (dict(lengths=_i32(2, 1)), "lengths"),
])
def test_cache_evict_refuses(other, message):
    from flh_b200 import _CUDA
    a = dict(k_caches=[_f16(2, 2, 20, 64)], v_caches=[_f16(2, 2, 20, 64)], weights=[torch.zeros(2, 2, 20)], lengths=_i32(2), keep=7, recent=3)
    with pytest.raises(RuntimeError, match=message):
        _CUDA.cache_evict(**{**a, **other})


def test_the_c_entries_refuse_without_a_device():
    from flh_b200 import _lib
    lib = _lib.load()
    one, other = ctypes.c_void_p(16), ctypes.c_void_p(32)
    ptrs, few, off = ((ctypes.c_void_p * 2)(*p) for p in ((16, 16), (16, None), (16, 24)))

    def attend(q=one, ss=64, dtype=0, tree=None, stride=0, scale=1.0, B=2, S=3, nh=4, nkv=2, D=64, T=20, ws=one, ws_bytes=1 << 30, k=one):
        return lib.flh_b200_tree_attention(q, 768, ss, 64, dtype, k, one, one, tree, stride, scale, one, None, B, S, nh, nkv, D, T, ws, ws_bytes, None)

    assert attend(dtype=2) == 1 and attend(S=0) == 1 and attend(S=65) == 1 and attend(nh=3) == 1 and attend(D=96) == 1 and attend(T=0) == 1 and attend(T=(1 << 21) + 1) == 1
    assert attend(scale=0.0) == 1 and attend(scale=float("nan")) == 1 and attend(scale=float("inf")) == 1 and attend(scale=-1.0) == 1
    assert attend(ss=60) == 2 and attend(tree=one, stride=4) == 1 and attend(q=None) == 1 and attend(q=ctypes.c_void_p(8)) == 2 and attend(k=None) == 1
    assert attend(ws_bytes=100) == 1 and b"too small" in lib.flh_b200_last_error()
    assert attend(ws=None, ws_bytes=0) == 1 and attend(B=1 << 20, T=1 << 21) == 1
    assert attend(B=0) == 0
    assert lib.flh_b200_tree_attention_workspace_bytes(0, 3, 4, 2, 64, 20, 1) == 0
    assert lib.flh_b200_tree_attention_workspace_bytes(2, 3, 4, 2, 64, 20, 1) > lib.flh_b200_tree_attention_workspace_bytes(2, 3, 4, 2, 64, 20, 0) > 0

    def rope(dtype=0, D=64, q=one, B=2, S=3):
        return lib.flh_b200_rope_kv_at(q, dtype, one, one, 9, one, one, one, one, one, B, S, 4, 2, D, 20, None)

    assert rope(dtype=5) == 1 and rope(D=24) == 1 and rope(q=None) == 1 and rope(q=ctypes.c_void_p(2)) == 2 and rope(B=0) == 0 and rope(S=0) == 0

    def accept(k=ptrs, w=None, layers=2, lengths=one, now=other, A=3, drafted=5, D=64, path=one):
        return lib.flh_b200_cache_accept(k, ptrs, w, layers, 0, lengths, path, one, now, 2, 2, D, 20, A, drafted, None)

    assert accept(layers=0) == 1 and accept(layers=129) == 1 and accept(drafted=0) == 1 and accept(drafted=65) == 1 and accept(A=6) == 1 and accept(D=12) == 1
    assert accept(now=one) == 1 and accept(path=None) == 1 and accept(k=few) == 1 and accept(k=off) == 2 and accept(w=few) == 1

    def evict(k=ptrs, layers=2, keep=7, recent=3, now=other, D=64, T=20):
        return lib.flh_b200_cache_evict(k, ptrs, ptrs, layers, 1, one, keep, recent, one, one, now, 2, 2, D, T, None)

    assert evict(keep=0) == 1 and evict(keep=21) == 1 and evict(recent=8) == 1 and evict(recent=-1) == 1 and evict(now=one) == 1 and evict(k=few) == 1 and evict(k=off) == 2
    assert evict(D=264) == 1 and evict(T=0) == 1


def test_reference_eviction_order():
    import numpy as np
    import tree_reference as R
    w = np.array([1, np.nan, 2, 2, np.inf, -0.0, 0.0, 9], dtype=np.float32)
    assert R.evict(w, 8, 3, 1).tolist() == [1, 4, 7] and R.evict(w, 8, 4, 1).tolist() == [1, 2, 4, 7] and R.evict(w, 7, 6, 0).tolist() == [0, 1, 2, 3, 4, 5]
    assert R.evict(w, 3, 3, 1).tolist() == [0, 1, 2] and R.evict(w, 8, 2, 2).tolist() == [6, 7]


@pytest.mark.parametrize("other,message", [
    (dict(counted=_i32(2)), "counted goes with weights"),
    (dict(counted=_i32(3), weights=torch.zeros(2, 2, 20)), "counted"),
    (dict(counted=_i32(2).long(), weights=torch.zeros(2, 2, 20)), "counted"),
    (dict(counted=_i32(2), weights=torch.zeros(2, 2, 20)), "must be CUDA"),
])
def test_counted_is_refused(other, message):
    from flh_b200 import _CUDA
    with pytest.raises(RuntimeError, match=message):
        _CUDA.tree_attention(**_attention(**other))


def test_the_c_entry_refuses_counted_without_weights():
    from flh_b200 import _lib
    lib, one = _lib.load(), ctypes.c_void_p(16)
    assert lib.flh_b200_tree_attention_counted(one, 768, 256, 64, 0, one, one, one, None, 0, 1.0, one, None, one, 2, 3, 4, 2, 64, 20, one, 1 << 30, None) == 1
    assert b"counted" in lib.flh_b200_last_error()
