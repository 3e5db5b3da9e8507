"""Argument checks of the sliding-window operators: through Python and through the C ABI, without a device."""

import ctypes as C

import pytest
import torch

from kvm_paper_b200 import _lib, window


def _err():
    return _lib.load().kvm_last_error_string().decode()


def _cache(**kw):
    d = dict(batch=2, n_kv_heads=2, head_dim=64, window=32, sinks=1, bits=4, k=256, v=None)
    d.update(kw)
    return _lib.KvmWindowCache(*(d[n] for n in ("batch", "n_kv_heads", "head_dim", "window", "sinks", "bits", "k", "v")))


@pytest.mark.parametrize("kw,code,text", [
    (dict(head_dim=48), 5, "head_dim"), (dict(bits=8), 5, "4 or 16 bits"), (dict(batch=0), 1, "batch"), (dict(n_kv_heads=-1), 1, "n_kv_heads"),
    (dict(window=0), 1, "window"), (dict(sinks=-1), 1, "sinks"), (dict(window=(1 << 30) + 1), 1, "window"),
    (dict(batch=1 << 14, n_kv_heads=1 << 11), 2, "kv rows"), (dict(batch=64, window=1 << 26), 2, "cache rows"),
    (dict(k=None), 1, "NULL"), (dict(k=264), 1, "aligned"), (dict(bits=16), 1, "NULL")])
def test_cache_descriptions_are_checked(kw, code, text):
    lib, c = _lib.load(), _cache(**kw)
    assert lib.kvm_window_cache_read(C.addressof(c), None, 4, 256, 256, None) == code and text in _err()
    w = _lib.KvmWindowWriteArgs(C.addressof(c), 256, 64, 64, 64, 256, 64, 64, 64, None, None, 1, 0, 1)
    assert lib.kvm_window_cache_write(C.addressof(w), None) == code and text in _err()
    a = _lib.KvmWindowAttendArgs(C.addressof(c), 256, 64, 64, 64, None, 0, 0, 0, None, 0, 0, 0, None, 256, None, 0, 2, 4, 0.125)
    assert lib.kvm_window_attend(C.addressof(a), None) == code and text in _err()
    if "k" not in kw and kw != dict(bits=16):
        assert lib.kvm_window_cache_bytes(C.byref(c)) == 0 and lib.kvm_window_attend_workspace_bytes(C.addressof(c), 2) == 0


def test_cache_sizes():
    lib = _lib.load()
    assert lib.kvm_window_cache_bytes(C.byref(_cache(head_dim=128, window=33, sinks=5))) == 2 * 2 * (16 + 48) // 16 * 18 * 128
    assert lib.kvm_window_cache_bytes(C.byref(_cache(bits=16, window=16, sinks=0))) == 2 * 2 * 16 * 64 * 2


@pytest.mark.parametrize("change,code,text", [
    (dict(n_q_heads=3), 1, "multiple"), (dict(n_q_heads=0), 1, "multiple"), (dict(n_q_heads=34), 5, "at most 16"), (dict(q=None), 1, "q is NULL"),
    (dict(q=264), 1, "multiples of 16 bytes"), (dict(q_stride_h=4), 1, "multiples of 16 bytes"), (dict(k_new=256), 1, "together"),
    (dict(k_new=256, v_new=264), 1, "multiples"), (dict(scale=0.0), 1, "scale"), (dict(scale=float("nan")), 1, "scale"),
    (dict(scale=float("inf")), 1, "scale"), (dict(out=None), 1, "out"), (dict(out=8), 1, "out")])
def test_attend_arguments_are_checked(change, code, text):
    lib, c = _lib.load(), _cache()
    a = _lib.KvmWindowAttendArgs(C.addressof(c), 256, 128, 64, 64, None, 0, 0, 0, None, 0, 0, 0, None, 256, None, 0, 2, 4, 0.125)
    for n, x in change.items():
        setattr(a, n, x)
    assert lib.kvm_window_attend(C.addressof(a), None) == code and text in _err()


def test_attend_needs_its_workspace_where_rows_are_cut():
    lib, c = _lib.load(), _cache(batch=1, n_kv_heads=1, window=1 << 20)
    need = lib.kvm_window_attend_workspace_bytes(C.addressof(c), 4)
    assert need > 0
    a = _lib.KvmWindowAttendArgs(C.addressof(c), 256, 128, 64, 64, None, 0, 0, 0, None, 0, 0, 0, None, 256, 256, need - 1, 4, 4, 0.125)
    assert lib.kvm_window_attend(C.addressof(a), None) == 2 and "workspace" in _err()


@pytest.mark.parametrize("change,code,text", [
    (dict(head_dim=96), 5, "head_dim"), (dict(n_q_heads=3), 1, "multiple"), (dict(n_kv_heads=0), 1, "multiple"), (dict(batch=-1), 1, "negative"),
    (dict(n_queries=9), 1, "as many keys"), (dict(n_queries=-1), 1, "negative"), (dict(n_keys=1 << 30), 1, "2^30"), (dict(window=0), 1, "window"),
    (dict(sinks=-1), 1, "sinks"), (dict(scale=-1.0), 1, "scale"), (dict(q=None), 1, "q is NULL"), (dict(k=8), 1, "k: base"),
    (dict(v_stride_t=68), 1, "v: base"), (dict(k_stride_b=0), 1, "strides must be positive"), (dict(v_stride_h=-64), 1, "strides must be positive"),
    (dict(q_stride_t=0), 1, "strides must be positive"), (dict(out=None), 1, "out")])
def test_prompt_arguments_are_checked(change, code, text):
    lib = _lib.load()
    t = (256, 1024, 64, 128)
    a = _lib.KvmWindowPromptArgs(*t, *t, *t, None, 256, 8, 8, 4, 0, 2, 2, 2, 64, 0.125)
    for n, x in change.items():
        setattr(a, n, x)
    assert lib.kvm_window_attention(C.addressof(a), None) == code and text in _err()


def test_empty_calls_are_no_calls():
    lib, c = _lib.load(), _cache()
    assert lib.kvm_window_attention(C.addressof(_lib.KvmWindowPromptArgs(*[None, 0, 0, 0] * 3, None, None, 0, 8, 4, 0, 2, 2, 2, 64, 0.125)), None) == 0
    assert lib.kvm_window_cache_write(C.addressof(_lib.KvmWindowWriteArgs(C.addressof(c), *[None, 0, 0, 0] * 2, None, None, 0, 0, 0)), None) == 0
    assert lib.kvm_window_attend(None, None) == 1 and lib.kvm_window_attention(None, None) == 1 and lib.kvm_window_cache_write(None, None) == 1


def test_write_positions_are_checked():
    lib, c = _lib.load(), _cache()
    a = _lib.KvmWindowWriteArgs(C.addressof(c), 256, 64, 64, 64, 256, 64, 64, 64, None, None, 2, 2**31 - 2, 2)
    assert lib.kvm_window_cache_write(C.addressof(a), None) == 1 and "2^31" in _err()


def test_python_calls_refuse_the_cpu():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        window.window_attention(q, q, q, window=4)
    with pytest.raises(RuntimeError, match="CUDA"):
        window.WindowCache(1, 2, 64, window=4, device="cpu")
    with pytest.raises(ValueError, match="tensor"):
        window.window_attention(q[0], q, q, window=4)
    with pytest.raises(ValueError, match="tensor"):
        window.window_attention(None, q, q, window=4)


@pytest.mark.parametrize("kw", [dict(batch=2**32 + 1), dict(window=2**32 + 8), dict(sinks=-2**32 + 1), dict(head_dim=2**32 + 64), dict(bits=2**32 + 4)])
def test_numbers_beyond_32_bits_are_refused(kw):
    with pytest.raises(ValueError, match="32-bit"):
        window.WindowCache(**{**dict(batch=1, n_kv_heads=2, head_dim=64, window=8), **kw})


def test_scales_beyond_the_range_are_refused():
    lib, c = _lib.load(), _cache()
    a = _lib.KvmWindowAttendArgs(C.addressof(c), 256, 128, 64, 64, None, 0, 0, 0, None, 0, 0, 0, None, 256, None, 0, 2, 4, 2.9e38)
    assert lib.kvm_window_attend(C.addressof(a), None) == 1 and "scale" in _err()


@pytest.mark.parametrize("cls", [_lib.KvmWindowWriteArgs, _lib.KvmWindowAttendArgs, _lib.KvmWindowPromptArgs])
def test_packed_blocks_are_what_the_structures_hold(cls):
    values = [0.25 if t is C.c_float else 2**31 - 1 - i if t is C.c_int32 else 2**40 + i for i, (_, t) in enumerate(cls._fields_)]
    assert _lib.packer(cls)(*values) == bytes(cls(*values))


def test_outputs_over_inputs_are_refused():
    """The prompt call reads its inputs again behind its first outputs; the token call may write in place of the queries."""
    lib, c = _lib.load(), _cache(batch=2, n_kv_heads=1, window=1 << 10)
    at = 1 << 20
    q, k, v = (at, 8 * 128, 64, 128), (at + (1 << 16), 8 * 64, 512, 64), (at + (1 << 17), 8 * 64, 512, 64)  # [2,2,8,64], [2,1,8,64]
    size = 2 * 8 * 2 * 64 * 2
    for out in (at, at + size - 16, at - size + 16, k[0], k[0] + 2 * 8 * 64 * 2 - 16, v[0] - size + 16):
        a = _lib.KvmWindowPromptArgs(*q, *k, *v, None, out, 8, 8, 4, 0, 2, 2, 1, 64, 0.125)
        assert lib.kvm_window_attention(C.addressof(a), None) == 1 and "share memory" in _err(), out
    one = 2 * 2 * 64 * 2
    q1, k1, v1 = (at, 128, 64, 64), (at + 4096, 64, 64, 64), (at + 8192, -64, 64, 64)
    for q2, out in ((q1, at + 16), (q1, at - 16), (q1, k1[0]), (q1, v1[0] + 128 - 16), (q1, v1[0] - one - 128 + 16), ((at, 256, 64, 64), at), ((at, 128, 128, 64), at)):
        a = _lib.KvmWindowAttendArgs(C.addressof(c), *q2, *k1, *v1, None, out, 1 << 24, 1 << 30, 2, 4, 0.125)
        assert lib.kvm_window_attend(C.addressof(a), None) == 1 and "share memory" in _err(), (q2, out)
