"""Refusals of the head norm's and the 4-bit cache's operators without a GPU: the C entry points
check shapes, types, pointers and workspaces before any launch."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import kv_q4 as O
from siliconfer_amd import _lib
from siliconfer_amd._lib import SFError
from siliconfer_amd.kernels.kv_q4 import attention_q4kv, dequantize_kv_q4, kv_append_q4, rotary_kv_append_q4
from siliconfer_amd.kernels.rotary import qk_norm_rotary

P = 4096  # a pointer that is never followed: every call below is refused before its launch
F32, F16, BF16 = _lib.SF_F32, _lib.SF_F16, _lib.SF_BF16


def refused(rc, code, text):
    assert rc == code and text in _lib.last_error(), (rc, _lib.last_error())


def norm(**kw):
    a = dict(q=P, q_out=P, k=P, k_out=P, dtype=F32, q_weight=P, k_weight=P, wdt=F32, eps=1e-6, positions=P, pos_i64=0,
             pos_per_seq=1, inv_freq=P, pairs=32, scale=1.0, interleaved=0, B=1, T=1, H=14, KVH=2, D=64, strides=None,
             stream=None)
    a.update(kw)
    return _lib.load().sf_qk_norm_rotary(*a.values())


def back(**kw):
    a = dict(q=P, q_grad=P, dq=P, k=P, k_grad=P, dk=P, dtype=F32, q_weight=P, k_weight=P, wdt=F32, dqw=P, dkw=P, eps=1e-6,
             positions=P, pos_i64=0, pos_per_seq=1, inv_freq=P, pairs=32, scale=1.0, interleaved=0, B=1, T=1, H=14, KVH=2,
             D=64, strides=None, ws=P, ws_bytes=1 << 30, stream=None)
    a.update(kw)
    return _lib.load().sf_qk_norm_rotary_backward(*a.values())


SHARED = [(dict(dtype=3), -1, "bad dtype"), (dict(wdt=-1), -1, "bad dtype"), (dict(pairs=0), -1, "rotated pairs"),
          (dict(pairs=33), -1, "33 rotated pairs in a head of 64"), (dict(D=257, pairs=1), -2, "at most 256"),
          (dict(B=-1), -1, "invalid head norm shape"), (dict(H=0), -1, "invalid head norm shape"),
          (dict(B=1 << 15, T=1 << 13), -1, "exceed the grid"), (dict(positions=None), -1, "null"),
          (dict(inv_freq=None), -1, "null"), (dict(q_weight=None), -1, "null pointer"), (dict(k_weight=None), -1, "null")]


@pytest.mark.parametrize("kw,code,text", SHARED + [(dict(q=None), -1, "null pointer"), (dict(k_out=None), -1, "null")])
def test_norm_c(kw, code, text):
    refused(norm(**kw), code, text)


@pytest.mark.parametrize("kw,code,text", SHARED + [
    (dict(q_grad=None), -1, "null pointer"), (dict(dk=None), -1, "null"), (dict(dqw=None), -1, "null"), (dict(T=0), -1, "no rows"),
    (dict(ws=None), -1, "workspace"), (dict(ws_bytes=64), -1, "workspace"), (dict(ws=P + 8), -1, "workspace")])
def test_norm_backward_c(kw, code, text):
    refused(back(**kw), code, text)


def append(**kw):
    a = dict(q=P, k=P, v=P, in_dtype=F32, strides=(64,) * 9, q_weight=P, k_weight=P, wdt=F32, eps=1e-6, positions=P,
             pos_i64=0, pos_per_seq=1, inv_freq=P, pairs=32, scale=1.0, interleaved=0, q_out=P, q_dtype=F32, k_codes=P,
             k_params=P, v_codes=P, v_params=P, group=64, lengths=None, start=0, B=1, T=1, H=14, KVH=2, D=64, T_cap=128,
             stream=None)
    a.update(kw)
    a["strides"] = a["strides"] and (ctypes.c_longlong * 9)(*a["strides"])
    return _lib.load().sf_kv_q4_append(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(start=128), -1, "KV cache overflow: 128 + 1 > capacity 128"), (dict(start=-1), -1, "overflow"),
    (dict(T_cap=0, start=0), -1, "overflow"), (dict(group=48), -1, "divisible by group"), (dict(group=16), -2, "group=16"),
    (dict(D=72, group=72), -2, "multiple of 16"), (dict(D=512, group=64), -1, "compile-time max 256"), (dict(pairs=33), -1, "rotated pairs"),
    (dict(in_dtype=3), -1, "dtype"), (dict(q_dtype=9), -1, "dtype"), (dict(wdt=7), -1, "dtype"), (dict(KVH=0), -1, "invalid KV shape"),
    (dict(k=None), -1, "null pointer"), (dict(q=None), -1, "null"), (dict(v_params=None), -1, "null"), (dict(positions=None), -1, "null"),
    (dict(strides=None), -1, "null"), (dict(strides=(64,) * 8 + (60,)), -1, "whole 8"), (dict(v=P + 8), -1, "16 bytes"),
    (dict(k_codes=P + 8), -1, "16-byte"), (dict(B=1 << 14, T=1 << 14, lengths=P), -1, "exceed the grid"),
])
def test_append_c(kw, code, text):
    refused(append(**kw), code, text)


def read(**kw):
    a = dict(codes=P, params=P, out=P, dtype=F32, group=64, strides=(64,) * 6, B=1, KVH=2, T=3, D=64, stream=None)
    a.update(kw)
    a["strides"] = (ctypes.c_longlong * 6)(*a["strides"])
    return _lib.load().sf_kv_q4_dequant(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(codes=None), -1, "null"), (dict(codes=P + 2), -1, "4 bytes"), (dict(strides=(64, 62, 64, 64, 64, 64)), -1, "4 bytes"),
    (dict(strides=(64, 64, 64, 64, 63, 64)), -1, "4 bytes"), (dict(out=P + 4), -1, "16-byte"), (dict(dtype=5), -1, "dtype"),
    (dict(group=24), -1, "divisible"), (dict(T=-1), -1, "invalid KV shape"), (dict(B=1 << 20, KVH=1 << 10, T=1 << 20), -1, "grid")])
def test_read_c(kw, code, text):
    refused(read(**kw), code, text)


def attend(**kw):
    a = dict(q=P, q_dtype=F32, k_codes=P, k_params=P, v_codes=P, v_params=P, group=64, out=P, out_dtype=F32, ws=P,
             ws_bytes=1 << 40, B=1, Tq=1, H=14, KVH=2, lengths=None, T=100, T_max=100, T_cap=128, D=64, scale=0.1, n_splits=0,
             stream=None)
    a.update(kw)
    return _lib.load().sf_attn_q4kv(*a.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(T=101), -1, "invalid attention shape"), (dict(T=-1), -1, "invalid"), (dict(T_max=129, T=9), -1, "invalid"),
    (dict(Tq=0), -1, "invalid"), (dict(KVH=3), -1, "not a multiple"), (dict(group=48), -1, "divisible"), (dict(group=16), -2, "group=16"),
    (dict(D=40, group=40), -2, "multiple of 16"), (dict(q_dtype=4), -1, "dtype"), (dict(out_dtype=-1), -1, "dtype"),
    (dict(q=None), -1, "null"), (dict(q=P + 8), -1, "16-byte"), (dict(v_params=P + 4), -1, "16-byte"), (dict(ws=None, n_splits=2), -1, "workspace"),
    (dict(ws=P + 16, n_splits=2), -1, "workspace"), (dict(ws_bytes=100, n_splits=2), -1, "too small"), (dict(B=70000), -1, "grid"),
    (dict(T_max=0x7fffff01, T_cap=0x7fffffff, T=1), -2, "at most"), (dict(Tq=1 << 20, B=1 << 10, H=14), -1, "grid")])
def test_attend_c(kw, code, text):
    refused(attend(**kw), code, text)


def test_nothing_to_do_is_no_error():
    assert norm(T=0) == 0 and norm(B=0, q=None) == 0
    assert append(T=0) == 0 and read(T=0) == 0 and read(B=0, codes=None) == 0


def test_sizes():
    lib = _lib.load()
    assert lib.sf_attn_q4_workspace_bytes(1, 1, 14, 2, 64, 64, 64, F32, F32, 0) == 0  # one tile: no partials
    assert lib.sf_attn_q4_workspace_bytes(1, 1, 14, 2, 6400, 64, 64, F32, F32, 3) == 14 * 3 * 64 * 4 + 14 * 3 * 8
    assert lib.sf_attn_q4_workspace_bytes(1, 1, 14, 2, 1 << 20, 64, 64, F32, F32, 1000) == 14 * 128 * 64 * 4 + 14 * 128 * 8
    assert lib.sf_attn_q4_workspace_bytes(1, 1, 14, 3, 64, 64, 64, F32, F32, 0) == 0
    assert lib.sf_qk_norm_backward_workspace_bytes(1, 1, 14, 2, 64) > 0


def test_python_layer_without_device():
    q, w = torch.zeros(1, 2, 3, 64), torch.ones(64)
    codes, params = torch.zeros(1, 3, 8, 32, dtype=torch.uint8), torch.zeros(1, 3, 8, 1, 2, dtype=torch.float16)
    pos, inv = torch.arange(2), torch.ones(32, dtype=torch.float64)
    bufs = (codes, params, codes, params)
    for call in (lambda: qk_norm_rotary(q, None, pos, inv, w), lambda: kv_append_q4(q, q, *bufs, lengths=0),
                 lambda: rotary_kv_append_q4(torch.zeros(1, 2, 9 * 64), pos, inv, *bufs, n_heads=3, lengths=0),
                 lambda: dequantize_kv_q4(codes, params), lambda: attention_q4kv(q, *bufs, lengths=1)):
        with pytest.raises(SFError, match="device"):
            call()


def test_oracle_round_trip():
    """The oracle's own codes: packed and read back within half a step and the parameters' rounding."""
    x = np.random.default_rng(1).standard_normal((3, 5, 96))
    for group in (32, 96):
        c, s, m, _ = O.quantize(x, group)
        y, _ = O.values(O.pack(c), np.stack([s, m], -1))
        step = np.repeat(s.astype(np.float64), group, -1)
        assert (c >= 0).all() and (c <= 15).all() and (abs(y - x) <= 0.5 * step + 2.0 ** -10 * (15 * step + abs(x).max())).all()
