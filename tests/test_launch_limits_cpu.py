"""Launches of the 8-bit cache and the int8 projection count their work items in 32 bits per grid dimension: calls past that are refused
on the host, before anything touches a device."""
import ctypes

import pytest

from test_int8_refusals_cpu import C, cache, refused   # noqa: F401  (fixture)


def test_a_cache_of_too_many_blocks(C):   # noqa: F811
    c = cache(C, nblk=1 << 24)
    d = C.KV8StoreDesc(k=256, v=256, dtype=0, L=1 << 30, start=256)
    refused(C, C._kv8_store(ctypes.byref(c), ctypes.byref(d), None), 'shape')
    refused(C, C._kv8_load(ctypes.byref(c), 256, 1 << 30, 256, 256, 0, None), 'shape')


@pytest.mark.parametrize('rows,H,S', [(65535, 4096, 64), (65535, 256, 65), (64, 64, 1 << 18)])
def test_a_prompt_of_too_many_workgroups(C, rows, H, S):   # noqa: F811
    d = C.KV8AttnDesc(q=256, q_dtype=0, S=S, Hq=H, len=256, len_stride=1, causal=1, out=256, out_mode=0)
    refused(C, C._kv8_attn(ctypes.byref(cache(C, rows=rows, H=H)), ctypes.byref(d), None), 'workgroups')


def test_a_projection_of_too_many_channels(C):   # noqa: F811
    d = C.LinearI8Desc(a=256, a_scale=256, w=256, w_scale=256, out=256, out_dtype=0, ldo=1 << 26, act=0, M=2, N=(1 << 25) + 1, K=64)
    refused(C, C._linear_i8(ctypes.byref(d), None), '2^25')
