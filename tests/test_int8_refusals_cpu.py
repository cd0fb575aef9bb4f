"""Refusals of the 8-bit cache's and the int8 projection's C entries: decided on the host, before anything touches a device."""
import ctypes

import pytest


@pytest.fixture(scope='module')
def C():
    from audiocraft_amd import _C
    return _C


def cache(C, **kw):
    d = dict(k_codes=256, v_codes=256, k_scale=256, v_scale=256, k_tail=256, v_tail=256, tail_dtype=C.BF16, rows=2, H=2, hd=64, nblk=4)
    d.update(kw)
    return C.KV8CacheDesc(**d)


def refused(C, rc, word):
    msg = C._last_error().decode()
    assert rc == -1 and word in msg, (rc, msg)


BAD_CACHES = [(dict(hd=48), 'head dim'), (dict(rows=0), 'shape'), (dict(rows=65536), 'shape'), (dict(H=0), 'shape'), (dict(nblk=0), 'shape'),
              (dict(tail_dtype=7), 'tail_dtype'), (dict(k_codes=None), 'null cache'), (dict(v_scale=None), 'null cache')]


@pytest.mark.parametrize('kw,word', BAD_CACHES)
def test_bad_caches(C, kw, word):
    c = cache(C, **kw)
    sd, ad = C.KV8StoreDesc(k=256, v=256, dtype=0, L=1, start=256), C.KV8AttnDesc(q=256, S=1, Hq=2, len=256, len_stride=1, out=256, causal=1)
    refused(C, C._kv8_store(ctypes.byref(c), ctypes.byref(sd), None), word)
    refused(C, C._kv8_load(ctypes.byref(c), 256, 1, 256, 256, 0, None), word)
    refused(C, C._kv8_attn(ctypes.byref(c), ctypes.byref(ad), None), word)
    assert C._kv8_attn_work(ctypes.byref(c), 1, 2) == 0


def test_null_descriptors(C):
    c = cache(C)
    for rc in (C._kv8_store(None, None, None), C._kv8_store(ctypes.byref(c), None, None), C._kv8_load(None, None, 1, None, None, 0, None),
               C._kv8_attn(None, None, None), C._kv8_attn(ctypes.byref(c), None, None), C._linear_i8(None, None)):
        assert rc == -1


@pytest.mark.parametrize('kw,word', [(dict(L=-1), 'L=-1'), (dict(dtype=2), 'dtype'), (dict(k=None), 'null'), (dict(v=None), 'null'),
                                     (dict(k=260), 'aligned rows'), (dict(v_tok=2), 'aligned rows')])
def test_bad_stores(C, kw, word):
    d = C.KV8StoreDesc(**{**dict(k=256, v=256, dtype=0, L=1, start=256), **kw})
    refused(C, C._kv8_store(ctypes.byref(cache(C)), ctypes.byref(d), None), word)


@pytest.mark.parametrize('name', ['k_codes', 'v_codes', 'k_tail', 'v_tail'])
def test_misaligned_buffers(C, name):
    d = C.KV8StoreDesc(k=256, v=256, dtype=0, L=1, start=256)
    refused(C, C._kv8_store(ctypes.byref(cache(C, **{name: 264})), ctypes.byref(d), None), 'aligned')
    refused(C, C._kv8_load(ctypes.byref(cache(C)), 256, 1, 256 + 4 * (name[0] == 'k'), 256 + 4 * (name[0] == 'v'), 0, None), 'aligned')


def test_scratch_of_absurd_sizes(C):
    assert C._kv8_attn_work(ctypes.byref(cache(C, H=1)), 1 << 30, 1 << 16) == 0


@pytest.mark.parametrize('T,dt,k', [(257, 0, 256), (-1, 0, 256), (5, 3, 256), (5, 0, None)])
def test_bad_loads(C, T, dt, k):
    assert C._kv8_load(ctypes.byref(cache(C)), 256, T, k, 256, dt, None) == -1


@pytest.mark.parametrize('kw,word', [
    (dict(Hq=3), 'Hq'), (dict(Hq=0), 'Hq'), (dict(S=-1), 'S=-1'), (dict(q=None), 'null'), (dict(len=None), 'null'), (dict(len_stride=2), 'len_stride'),
    (dict(q_dtype=5), 'q_dtype'), (dict(out_mode=9), 'out_mode'), (dict(out_mode=2, S=2), 'out_mode'), (dict(out=264), 'aligned'),
    (dict(k_new=256), 'together'), (dict(k_new=256, v_new=256, S=2), 'S = 1'), (dict(k_new=256, v_new=256, causal=0), 'causal'),
    (dict(complete=1, S=3), 'S = 1'), (dict(k_new=256, v_new=256, new_dtype=4), 'new_dtype'), (dict(past_context=-1), 'past_context'),
    (dict(causal=0, past_context=3), 'past_context'), (dict(out_mode=2, out_dtype=1, out_col0=16), 'placement'),
    (dict(out_mode=2, out_dtype=1, out_rbs=1), 'placement'), (dict(q=260), 'aligned rows'), (dict(q_row=2), 'aligned rows'),
    (dict(k_new=256, v_new=256, kn_row=3), 'aligned rows'), (dict(k_new=256, v_new=264), 'aligned rows')])
def test_bad_attention(C, kw, word):
    d = C.KV8AttnDesc(**{**dict(q=256, q_dtype=0, S=1, Hq=2, len=256, len_stride=1, causal=1, out=256, out_mode=0), **kw})
    refused(C, C._kv8_attn(ctypes.byref(cache(C)), ctypes.byref(d), None), word)


def test_attention_scratch_is_required(C):
    c = cache(C, nblk=1000)
    d = C.KV8AttnDesc(q=256, S=1, Hq=2, len=256, len_stride=1, causal=1, out=256)
    n = C._kv8_attn_work(ctypes.byref(c), 1, 2)
    assert n > 0 and n % (16 * (64 + 4)) == 0
    refused(C, C._kv8_attn(ctypes.byref(c), ctypes.byref(d), None), 'work')


@pytest.mark.parametrize('kw,word', [(dict(K=0), 'K=0'), (dict(K=131073), 'K=131073'), (dict(dtype=2), 'dtype'), (dict(ldx=7), 'ldx'),
                                     (dict(codes=264), 'aligned'), (dict(x=None), 'null'), (dict(R=-1), 'R=-1'), (dict(R=2 ** 31 - 1), '2^30')])
def test_bad_quantisations(C, kw, word):
    a = {**dict(x=256, dtype=0, ldx=8, R=2, K=8, codes=256, scale=256), **kw}
    refused(C, C._quantize_rows_i8(a['x'], a['dtype'], a['ldx'], a['R'], a['K'], a['codes'], a['scale'], None), word)


@pytest.mark.parametrize('kw,word', [(dict(K=131073), 'K=131073'), (dict(N=0), 'N=0'), (dict(M=-1), 'M=-1'), (dict(out_dtype=3), 'out_dtype'),
                                     (dict(act=2), 'act'), (dict(ldo=3), 'ldo'), (dict(a=260), 'aligned'), (dict(w_scale=None), 'null'),
                                     (dict(M=1 << 30, N=1 << 20), '2^38'), (dict(M=2 ** 31 - 1), '2^30')])
def test_bad_projections(C, kw, word):
    d = C.LinearI8Desc(**{**dict(a=256, a_scale=256, w=256, w_scale=256, out=256, out_dtype=0, ldo=4, act=0, M=2, N=4, K=64), **kw})
    refused(C, C._linear_i8(ctypes.byref(d), None), word)


def test_nothing_to_do_is_no_error(C):
    d = C.LinearI8Desc(M=0, N=4, K=64)
    assert C._linear_i8(ctypes.byref(d), None) == 0
    assert C._quantize_rows_i8(None, 0, 0, 0, 8, None, None, None) == 0
    s = C.KV8StoreDesc(dtype=0, L=0, start=256)
    assert C._kv8_store(ctypes.byref(cache(C)), ctypes.byref(s), None) == 0
